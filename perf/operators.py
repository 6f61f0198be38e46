"""The decoder-layer operators of this package as measured cases: what each computes in plain torch operations, and the calls of
the package that compute the same.

  rms     residual addition, RMSNorm over the row and per-token 8-bit codes      dsaquant_b200.kernels.rms_norm.rms_norm_quant
  matvec  a few tokens times a 4-bit weight with group scales                    dsaquant_b200.kernels.w4_group.linear_w4_group
  rotary  rotary positions on q and k, half and interleaved, part of the head    dsaquant_b200.rotary.apply_rotary
  window  causal attention with a sliding window and always-visible first keys   dsaquant_b200.window_attention.window_attention
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}


def listed():
    return [
        # one token of a decoding sequence at the width of the 14B model, 8-bit float codes for a library product
        {"name": "rms_token", "op": "rms", "m": 1, "d": 5120, "dtype": "bf16", "residual": True, "codes": "e4m3"},
        # a whole prompt (the 32760 tokens of the benchmark's video) in front of the int8 GEMM
        {"name": "rms_prompt", "op": "rms", "m": 32760, "d": 5120, "dtype": "bf16", "residual": True, "codes": "int8"},
        # a ragged batch at the small model's width, residual stream kept in fp32
        {"name": "rms_fp32_odd", "op": "rms", "m": 517, "d": 1536, "dtype": "fp32", "residual": False, "codes": "e4m3"},
        # one token through the fused q/k/v projection of the 14B model
        {"name": "matvec_token", "op": "matvec", "m": 1, "n": 15360, "k": 5120, "group": 128, "dtype": "bf16", "bias": True},
        # eight sequences decoding together through the feed-forward's down projection
        {"name": "matvec_batch8", "op": "matvec", "m": 8, "n": 5120, "k": 13824, "group": 64, "dtype": "fp16", "bias": False},
        # the small model's up projection on 8-bit tokens, an odd batch
        {"name": "matvec_int8_odd", "op": "matvec", "m": 5, "n": 8960, "k": 1536, "group": 32, "dtype": "int8", "bias": True},
        # one token of 40 query heads that share 8 key heads
        {"name": "rotary_token", "op": "rotary", "t": 1, "hq": 40, "hkv": 8, "hd": 128, "rd": 128, "dtype": "bf16",
         "interleaved": False, "scaling": "none", "far": 32768},
        # a whole prompt, every head rotated in neighbouring pairs
        {"name": "rotary_prompt", "op": "rotary", "t": 32760, "hq": 40, "hkv": 40, "hd": 128, "rd": 128, "dtype": "fp16",
         "interleaved": True, "scaling": "none", "far": 32768},
        # positions far past the trained length, half of each head rotated
        {"name": "rotary_part_far", "op": "rotary", "t": 4097, "hq": 12, "hkv": 2, "hd": 128, "rd": 64, "dtype": "bf16",
         "interleaved": False, "scaling": "yarn", "far": 524288},
        # sixteen sequences decoding on one cache, lengths from nothing to full
        {"name": "window_token", "op": "window", "b": 16, "lq": 1, "lk": 8192, "hq": 40, "hkv": 8, "hd": 128, "dtype": "bf16",
         "window": 4096, "sinks": 4, "ragged": True},
        # a whole prompt of the 1.3B model's 12 heads
        {"name": "window_prompt", "op": "window", "b": 1, "lq": 32760, "lk": 32760, "hq": 12, "hkv": 12, "hd": 128, "dtype": "bf16",
         "window": 4096, "sinks": 64, "ragged": False},
        # a chunk of three prompts on a cache, some rows before the first key
        {"name": "window_chunk", "op": "window", "b": 3, "lq": 517, "lk": 2051, "hq": 8, "hkv": 2, "hd": 64, "dtype": "fp16",
         "window": 300, "sinks": 5, "ragged": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rms", "matvec", "rotary", "window"])
    if op == "rms":
        codes = rng.choice(["int8", "e4m3"])
        d = _log(rng, 64, 14000)
        if rng.random() < 0.7:
            d = d // 64 * 64
        return {"op": op, "m": _log(rng, 1, min(32760, 32760 * 5120 // d)), "d": d,
                "dtype": rng.choice(["bf16", "fp16"] + (["fp32"] if codes == "e4m3" else [])), "residual": rng.random() < 0.7,
                "codes": codes}
    if op == "matvec":
        group = rng.choice([32, 64, 128])
        k = max(2, _log(rng, 256, 14000) // group) * group
        return {"op": op, "m": _log(rng, 1, 64), "n": _log(rng, 100, 20000), "k": k, "group": group,
                "dtype": rng.choice(["bf16", "fp16", "int8"]), "bias": rng.random() < 0.5}
    if op == "rotary":
        hd = rng.choice([64, 128])
        hkv = rng.choice([1, 2, 8, 12])
        return {"op": op, "t": _log(rng, 1, 20000), "hq": hkv * rng.choice([1, 2, 3]), "hkv": hkv, "hd": hd,
                "rd": rng.choice([hd, hd // 2, hd // 4]), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
                "far": rng.choice([32768, 131072, 524288])}
    hkv, hd = rng.choice([1, 2, 4]), rng.choice([64, 128])
    case = {"op": op, "hq": hkv * rng.choice([1, 2, 4, 5]), "hkv": hkv, "hd": hd, "dtype": rng.choice(["bf16", "fp16"]),
            "sinks": rng.choice([0, 1, 4, 70]), "ragged": rng.random() < 0.7}
    if rng.random() < 0.5:
        lk = _log(rng, 2, 16000)
        return {**case, "b": _log(rng, 1, 32), "lq": min(lk, rng.choice([1, 1, 1, 2, 3])), "lk": lk, "window": _log(rng, 1, 8000)}
    lk = _log(rng, 130, 6000)
    return {**case, "b": rng.choice([1, 1, 2, 3]), "lq": _log(rng, 100, lk), "lk": lk, "window": _log(rng, 16, 4000)}


# ---------------------------------------------------------------------------------------------- inputs
def _inv_freq(case):
    """Angular frequency of each rotated pair in 64 bits, and the factor on the amplitudes."""
    rd, base, factor, trained = case["rd"], 10000.0, 8.0, 4096
    i = torch.arange(rd // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "linear":
        return base ** (-2 * i / rd) / factor, 1.0
    if case["scaling"] == "ntk":
        return (base * factor ** (rd / (rd - 2))) ** (-2 * i / rd), 1.0
    f = base ** (-2 * i / rd)
    if case["scaling"] == "yarn":
        low = math.floor(rd * math.log(trained / (32.0 * 2 * math.pi)) / (2 * math.log(base)))
        high = math.ceil(rd * math.log(trained / (1.0 * 2 * math.pi)) / (2 * math.log(base)))
        low, high = max(low, 0), min(high, rd - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)

    s = {"case": case}
    if case["op"] == "rms":
        dt = _DT[case["dtype"]]
        s["x"] = randn(case["m"], case["d"], dtype=dt)
        # a residual stream has a few channels far larger than the rest
        wide = torch.where(torch.rand(case["d"], generator=g, device="cuda") < 0.01, 20.0, 1.0)
        s["residual"] = (randn(case["m"], case["d"]) * wide).to(dt) if case["residual"] else None
        s["weight"] = (1 + randn(case["d"], by=0.1)).to(dt)
    elif case["op"] == "matvec":
        m, n, k = case["m"], case["n"], case["k"]
        s["packed"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(n, k // case["group"], generator=g, device="cuda")) * 0.01).half()
        s["bias"] = s["act_scale"] = None
        if case["dtype"] == "int8":
            s["x"] = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
            s["act_scale"] = (0.5 + torch.rand(m, generator=g, device="cuda")) / 40
            s["out"] = torch.float16
        else:
            s["x"] = randn(m, k, dtype=_DT[case["dtype"]])
            s["out"] = s["x"].dtype
        if case["bias"]:
            s["bias"] = randn(n, dtype=s["out"], by=0.1)
    elif case["op"] == "rotary":
        t, hq, hkv, hd = case["t"], case["hq"], case["hkv"], case["hd"]
        qkv = randn(t, hq + 2 * hkv, hd, dtype=_DT[case["dtype"]])  # one fused projection's output: q and k are views of it
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        start = torch.randint(0, case["far"] - t + 1, (1,), generator=g, device="cuda")
        s["positions"] = start + torch.arange(t, device="cuda")
        f, amplitude = _inv_freq(case)
        angle = torch.arange(case["far"], dtype=torch.float64, device="cuda")[:, None] * f
        s["cos_sin"] = (torch.stack([angle.cos(), angle.sin()], -1) * amplitude).float()
    else:
        b, lq, lk, hq, hkv, hd = (case[n] for n in ("b", "lq", "lk", "hq", "hkv", "hd"))
        dt = _DT[case["dtype"]]
        s["q"], s["k"], s["v"] = randn(b, lq, hq, hd, dtype=dt), randn(b, lk, hkv, hd, dtype=dt), randn(b, lk, hkv, hd, dtype=dt)
        s["lens"] = None
        if case["ragged"]:
            s["lens"] = torch.randint(0, lk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            s["lens"][0] = lk
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _rms_plain(s):
    case, x = s["case"], s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    top = 127.0 if case["codes"] == "int8" else 448.0
    scale = y.abs().amax(-1).clamp_min(1e-5) / top
    t = y / scale[:, None]
    codes = t.round().clamp(-128, 127).to(torch.int8) if case["codes"] == "int8" else t.clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, scale, x.to(s["x"].dtype) if s["residual"] is not None else None


def _matvec_plain(s):
    packed, group = s["packed"], s["case"]["group"]
    n, k = packed.shape[0], packed.shape[1] * 2
    codes = torch.stack([packed & 15, packed >> 4], -1).reshape(n, k // group, group).float()
    codes = codes - 16 * (codes > 7)
    w = (codes * s["scales"].float()[..., None]).reshape(n, k)
    y = s["x"].float() @ w.t()
    if s["act_scale"] is not None:
        y = y * s["act_scale"][:, None]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"])


def _rotate_plain(x, cos, sin, rd, interleaved):
    r, rest = x[..., :rd].float(), x[..., rd:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rd // 2], r[..., rd // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([r.to(x.dtype), rest], -1)


def _rotary_plain(s):
    cs = s["cos_sin"][s["positions"]][:, None]
    case = s["case"]
    return [_rotate_plain(x, cs[..., 0], cs[..., 1], case["rd"], case["interleaved"]) for x in (s["q"], s["k"])]


def _window_plain(s):
    """Queries in blocks; each block meets the first keys and the keys that its window can reach."""
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, lq, hq, hd = q.shape
    lk, hkv = k.shape[1], k.shape[2]
    w, sinks = min(s["case"]["window"], lk), min(s["case"]["sinks"], lk)
    lens = s["lens"].long() if s["lens"] is not None else torch.full((b,), lk, device=q.device)
    bs = min(lq, 256)
    nb = -(-lq // bs)
    q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, nb * bs - lq)).view(b, nb, bs, hkv, hq // hkv, hd)
    at = (lens[:, None] - lq + torch.arange(nb * bs, device=q.device)).view(b, nb, bs)
    first = torch.arange(sinks, device=q.device).expand(b, nb, sinks)
    near = at[..., :1] - w + 1 + torch.arange(w + bs - 1, device=q.device)
    j, p = torch.cat([first, near], -1)[:, :, None], at[..., None]
    inside = (j <= p) & (j > p - w) & (j >= 0)
    inside[..., :sinks] = (j <= p - w)[..., :sinks]  # a first key inside the window is met there
    rows = torch.cat([first, near], -1).clamp(0, lk - 1)
    which = torch.arange(b, device=q.device)[:, None, None]
    score = torch.einsum("bnihgd,bnthd->bnhgit", q, k[which, rows]) * (1 / math.sqrt(hd))
    score.masked_fill_(~inside[:, :, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    out = torch.einsum("bnhgit,bnthd->bnhgid", e, v[which, rows]) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 1, 4, 2, 3, 5).reshape(b, nb * bs, hq, hd)[:, :lq]
    lse = (top + total.log()).permute(0, 2, 3, 1, 4, 5).reshape(b, hq, nb * bs)[..., :lq]
    return out.to(s["q"].dtype), lse


def run(state):
    s, case = state, state["case"]
    if case["op"] == "rms":
        if own:
            from dsaquant_b200.kernels.rms_norm import rms_norm_quant

            dt = torch.int8 if case["codes"] == "int8" else torch.float8_e4m3fn
            codes, scale, *more = rms_norm_quant(s["x"], s["weight"], 1e-6, residual=s["residual"], out_dtype=dt)
            residual = more[0] if more else None
        else:
            codes, scale, residual = _rms_plain(s)
        if case["codes"] == "int8":  # as the values that the codes stand for
            codes = codes * scale.to(s["x"].dtype)[:, None]
        return {"codes": codes, "scale": scale, "residual": residual}
    if case["op"] == "matvec":
        if own:
            from dsaquant_b200.kernels.w4_group import linear_w4_group

            return linear_w4_group(s["x"], s["packed"], s["scales"], s["bias"], act_scale=s["act_scale"], out_dtype=s["out"])
        return _matvec_plain(s)
    if case["op"] == "rotary":
        if own:
            from dsaquant_b200.rotary import apply_rotary

            return apply_rotary(s["q"], s["k"], s["cos_sin"], s["positions"], interleaved=case["interleaved"])
        return _rotary_plain(s)
    if own:
        from dsaquant_b200.window_attention import window_attention

        return window_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"], kv_lens=s["lens"], return_lse=True)
    return _window_plain(s)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def _pairs(first, last, window, sinks):
    """(query, key) pairs of the queries at positions first..last, and the keys that any of them meets."""
    first = max(first, 0)
    if last < first:
        return 0, 0
    p = torch.arange(first, last + 1, dtype=torch.float64)
    near = (p + 1).clamp_max(window)
    pairs = float((near + (p + 1 - near).clamp_max(sinks)).sum())
    low = max(0, first - window + 1)
    return pairs, last - low + 1 + min(low, sinks)


def work(case):
    if case["op"] == "rms":
        each = case["m"] * case["d"]
        size = _SIZE[case["dtype"]]
        # x, the residual in and out, the codes, the weight, a scale a row
        return {"bytes": each * (size * (3 if case["residual"] else 1) + 1) + case["d"] * size + 4 * case["m"], "flops": 6 * each}
    if case["op"] == "matvec":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 2 * n * (k // case["group"]) + m * k * _SIZE[case["dtype"]] + 2 * m * n, "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        heads = case["t"] * (case["hq"] + case["hkv"])
        return {"bytes": 2 * heads * case["hd"] * _SIZE[case["dtype"]] + case["t"] * (8 + 4 * case["rd"]), "flops": 3 * heads * case["rd"]}
    b, lq, lk, hq, hkv, hd = (case[n] for n in ("b", "lq", "lk", "hq", "hkv", "hd"))
    # lengths are drawn evenly between nothing and full: the mean over a few of them
    ends = [lk] + ([int(lk * (i + 0.5) / 16) for i in range(16)] if case["ragged"] and b > 1 else [])
    got = [_pairs(e - lq, e - 1, case["window"], case["sinks"]) for e in ends]
    mean = [(got[0][i] + (b - 1) * (sum(x[i] for x in got[1:]) / max(1, len(got) - 1) if len(got) > 1 else got[0][i])) for i in (0, 1)]
    return {"bytes": 4 * b * lq * hq * hd + 4 * b * lq * hq + 4 * mean[1] * hkv * hd, "flops": 4 * mean[0] * hq * hd}


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rms":
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        y = x / (x.pow(2).sum(-1, keepdim=True) / case["d"] + 1e-6).sqrt() * s["weight"].double()
        top = {"int8": 127, "e4m3": 448}[case["codes"]]
        step = torch.clamp(y.abs().max(-1).values, min=1e-5) / top
        codes = y / step.unsqueeze(-1)
        if case["codes"] == "int8":
            codes = codes.round() * step.unsqueeze(-1)
        else:
            codes = codes.to(torch.float8_e4m3fn).double()
        return {"codes": codes, "scale": step, "residual": x if s["residual"] is not None else None}
    if case["op"] == "matvec":
        p = s["packed"].to(torch.int16)
        codes = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = (p % 16 + 8) % 16 - 8, (p // 16 + 8) % 16 - 8
        x = s["x"].double()
        if s["act_scale"] is not None:
            x = x * s["act_scale"].double().unsqueeze(1)
        y = x @ (codes * s["scales"].double().repeat_interleave(case["group"], 1)).T
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "rotary":
        f, amplitude = _inv_freq(case)
        turn = torch.polar(torch.full_like(f, amplitude).expand(case["t"], -1).contiguous(), s["positions"].double()[:, None] * f)
        rd, done = case["rd"], []
        for x in (s["q"].double(), s["k"].double()):
            pair = x[..., :rd].unflatten(-1, (rd // 2, 2)) if case["interleaved"] else x[..., :rd].unflatten(-1, (2, rd // 2)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:, None])
            done.append(torch.cat([z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2), x[..., rd:]], -1))
        return done
    q, k, v = s["q"], s["k"], s["v"]
    b, lq, hq, hd = q.shape
    lk, share = case["lk"], hq // case["hkv"]
    lens = s["lens"].tolist() if s["lens"] is not None else [lk] * b
    out = torch.zeros(b, lq, hq, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((b, hq, lq), -math.inf, dtype=torch.float64, device="cuda")
    key = torch.arange(lk, device="cuda")
    for i in range(b):
        for low in range(max(0, lq - lens[i]), lq, 512):
            at = lens[i] - lq + torch.arange(low, min(lq, low + 512), device="cuda")
            reach = (key <= at[-1]) & ((key > at[0] - case["window"]) | (key < case["sinks"]))
            j = key[reach]
            seen = (j[None] <= at[:, None]) & ((j[None] > at[:, None] - case["window"]) | (j[None] < case["sinks"]))
            kk, vv = (t[i][reach].double().repeat_interleave(share, 1).transpose(0, 1) for t in (k, v))
            score = q[i, low:low + 512].double().transpose(0, 1) @ kk.transpose(1, 2) / hd ** 0.5
            score = score.masked_fill(~seen, -math.inf)
            out[i, low:low + 512] = (score.softmax(-1) @ vv).transpose(0, 1)
            lse[i, :, low:low + 512] = score.logsumexp(-1)
    return out, lse
