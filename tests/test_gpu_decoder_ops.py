"""Decoder-layer operators against their definitions in 64 bits.

Tolerances count roundings: a value stored in type t is off by at most finfo(t).eps / 2 of itself (half a subnormal
step near zero); an fp32 sum of n terms by n * 2^-23 of the sum of their magnitudes (tensor cores may truncate, hence
twice half an eps); everything else is stated where it is used."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
HALF_SUB = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _within(got, want, bound):
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst excess {(err - bound).max().item():.3g}, error {err.max().item():.3g}"


# ------------------------------------------------------------------------------------------------ rms_norm_quant
def _check_rms(x, w, residual, out_dtype, eps=1e-6, clip=1.0):
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    got = rms_norm_quant(x, w, eps, residual=residual, out_dtype=out_dtype, clip_ratio=clip)
    d = x.shape[-1]
    s = x.double() + (residual.double() if residual is not None else 0)
    y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps) * w.double()
    top = 127.0 if out_dtype == torch.int8 else 448.0
    scale = y.abs().amax(-1).clamp_min(1e-5) / top * clip
    codes, got_scale = got[0], got[1]
    assert codes.dtype == out_dtype and codes.shape == x.shape and got_scale.shape == x.shape[:-1]
    # sum of squares: at most 64 + 10 additions one after another; then half of it, rsqrt, two products, a quotient
    rel = (74 / 2 + 8) * 2.0 ** -24
    _within(got_scale, scale, rel * scale + 1e-30)
    t = y / scale[..., None]
    if out_dtype == torch.int8:
        t = t.clamp(-128, 127)
        _within(codes, t, 0.5 + 2 * rel * t.abs() + 1e-9)
    else:
        t = t.clamp(-448, 448)
        _within(codes, t, 2.0 ** -4 * t.abs() + 2.0 ** -10 + 2 * rel * t.abs())
    if residual is not None:
        assert got[2].dtype == x.dtype
        _within(got[2], s, HALF_STEP[x.dtype] * s.abs() + HALF_SUB[x.dtype] + 2.0 ** -24 * s.abs())
    return got


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("out_dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("m, d", [(1, 1), (1, 5120), (3, 7), (2, 8), (5, 255), (5, 256), (9, 257), (4, 768), (33, 777), (17, 1536),
                                  (6, 2049), (3, 5120), (2, 6145), (2, 8960), (2, 13824), (3, 16384), (2, 16383), (1025, 64)])
def test_rms_norm_quant(m, d, dtype, out_dtype):
    g = _gen(m * 100003 + d)
    x, r = _randn(g, m, d, dtype=dtype), _randn(g, m, d, dtype=dtype)
    w = (1 + 0.1 * _randn(g, d)).to(dtype)
    _check_rms(x, w, None, out_dtype)
    _check_rms(x, w.float(), r, out_dtype)


def test_rms_norm_quant_strided_rows_clip_and_leading_dims():
    g = _gen(1)
    wide = _randn(g, 2, 50, 3 * 512, dtype=BF)
    w = _randn(g, 512, dtype=BF)
    part = wide[..., 512:1024]                                       # read in place: pitch 1536
    got = _check_rms(part, w, wide[..., :512], torch.int8, clip=0.9)
    again = _check_rms(part.contiguous(), w, wide[..., :512].contiguous(), torch.int8, clip=0.9)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    odd = _randn(g, 40, 130, dtype=FP)[:, 1:]                        # rows start off every alignment
    _check_rms(odd, _randn(g, 129, dtype=F32), odd, torch.float8_e4m3fn)
    _check_rms(_randn(g, 64, 128, dtype=BF).t(), _randn(g, 64, dtype=BF), None, torch.int8)   # column-major: copied


def test_rms_norm_quant_small_zero_and_not_finite_rows():
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    x = torch.randn(6, 512, device="cuda", generator=_gen(2))
    x[1] = 0
    x[2] *= 1e-12
    x[3, 100] = float("inf")
    x[4, 511] = float("nan")
    w = torch.ones(512, device="cuda")
    for dt in (torch.int8, torch.float8_e4m3fn):
        codes, scale = rms_norm_quant(x, w, out_dtype=dt)
        top = 127 if dt == torch.int8 else 448
        assert bool((codes[1].float() == 0).all()) and abs(scale[1].item() * top / 1e-5 - 1) < 1e-6
        assert bool(torch.isfinite(scale[[0, 1, 2, 5]]).all())
        assert bool(torch.isnan(scale[[3, 4]]).all()) and bool((codes[[3, 4]].float() == 0).all())
        keep = [0, 1, 2, 5]
        clean = rms_norm_quant(x[keep], w, out_dtype=dt)
        assert torch.equal(clean[0].view(torch.uint8), codes[keep].view(torch.uint8)) and torch.equal(clean[1], scale[keep])
    w[7] = float("nan")
    assert bool(torch.isnan(rms_norm_quant(x[:1], w)[1]).all())


@pytest.mark.parametrize("dtype, d, clip", [(F32, 1536, 1.0), (BF, 5120, 1.0), (FP, 777, 0.9), (F32, 96, 1.0)])
def test_rms_norm_quant_e4m3_codes_are_the_exact_ones(dtype, d, clip):
    """Millions of values, none on the wrong side of a midpoint: the definition in 64 bits, rounded to the nearest e4m3
    value with ties to even by a search over all of them."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(41 + d)
    m = 3_000_000 // d
    x, r = _randn(g, m, d, dtype=dtype), _randn(g, m, d, dtype=dtype)
    w = (1 + 0.1 * _randn(g, d)).to(dtype)
    codes, scale, _ = rms_norm_quant(x, w, residual=r, out_dtype=torch.float8_e4m3fn, clip_ratio=clip)
    y = (x.double() + r.double()) * w.double()                       # the rsqrt cancels in y / max|y|
    t = (y * 448 / (y.abs().amax(-1, keepdim=True) * clip)).clamp(-448, 448)
    table = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()   # 0 .. 448
    mid = (table[1:] + table[:-1]) / 2
    low = torch.searchsorted(mid, t.abs())                           # mid[low - 1] < |t| <= mid[low]
    tie = (low < 126) & (t.abs() == mid[low.clamp(max=125)]) & (low % 2 == 1)
    want = torch.where(t < 0, -1.0, 1.0) * table[low + tie.long()]
    normal = t.abs() >= 2.0 ** -6
    assert torch.equal(codes.double()[normal], want[normal])
    # below the normal range the steps are absolute (2^-9) and an fp32 quotient is off by 2^-6 * 8 * 2^-24 at most
    _within(codes.double()[~normal], t[~normal], 2.0 ** -10 + 2.0 ** -27)


def test_rms_norm_quant_refusals_and_empty():
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    codes, scale, stream = rms_norm_quant(x[:0], w, residual=x[:0])
    assert codes.shape == (0, 64) and scale.shape == (0,) and stream.shape == (0, 64)
    for bad in (dict(residual=x[:2]), dict(residual=x.half()), dict(out_dtype=torch.uint8), dict(clip_ratio=0.0), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            rms_norm_quant(x, w, **bad)
    with pytest.raises(ValueError):
        rms_norm_quant(x, w[:63])
    with pytest.raises(RuntimeError):
        rms_norm_quant(x.double(), w)
    with pytest.raises(ValueError):
        rms_norm_quant(torch.zeros(1, 16385, device="cuda"), torch.zeros(16385, device="cuda"))


def test_rms_norm_codes_feed_the_int8_gemm():
    """int8 codes times per-channel 4-bit weights in the existing GEMM: exact integer sums."""
    from dsaquant_b200.kernels import vdm_w4a4 as vdm
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(3)
    m, k, n = 70, 1536, 256
    packed, sp, ws = vdm.quantize_weight_per_channel(_randn(g, n, k, dtype=FP) * 0.02)
    codes, scale = rms_norm_quant(_randn(g, m, k, dtype=BF), torch.ones(k, device="cuda"))
    out, acc = vdm.linear_prequantized(codes, scale, packed, sp, return_acc=True)
    want = codes.cpu().long() @ vdm.unpack_codes(packed, n, k, 2).cpu().long().t()
    assert torch.equal(acc.cpu().long(), want)
    y = want.cuda().double() * scale.double()[:, None] * ws.double()
    _within(out, y, 2.0 ** -11 * y.abs() + 2.0 ** -25 + 2.0 ** -22 * y.abs())


# ------------------------------------------------------------------------------------------------ linear_w4_group
def _codes_of(packed):
    p = packed.to(torch.int16)
    c = torch.stack([p & 15, p >> 4], -1).flatten(-2)
    return torch.where(c > 7, c - 16, c).double()


def _check_w4(x, packed, scales, bias=None, act_scale=None, out_dtype=None):
    from dsaquant_b200.kernels.w4_group import linear_w4_group

    got = linear_w4_group(x, packed, scales, bias, act_scale=act_scale, out_dtype=out_dtype)
    n, k = packed.shape[0], packed.shape[1] * 2
    w = _codes_of(packed) * scales.double().repeat_interleave(k // scales.shape[1], 1)
    xd = x.reshape(-1, k).double()
    if act_scale is not None:
        xd = xd * act_scale.double().reshape(-1, 1)
    y, size = xd @ w.t(), xd.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    want_dtype = out_dtype or (FP if x.dtype == torch.int8 else x.dtype)
    assert got.dtype == want_dtype and got.shape == x.shape[:-1] + (n,)
    _within(got.reshape(-1, n), y, HALF_STEP[want_dtype] * y.abs() + HALF_SUB[want_dtype] + (k + 16) * 2.0 ** -23 * size)
    return got


def _w4_case(g, n, k, group):
    packed = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((0.5 + torch.rand(n, k // group, generator=g, device="cuda")) * 0.01).half()
    return packed, scales


@pytest.mark.parametrize("xdtype", [BF, FP, torch.int8])
@pytest.mark.parametrize("m, n, k, group", [
    (1, 1, 32, 32), (1, 17, 64, 32), (1, 128, 96, 32), (1, 100, 128, 128), (2, 33, 192, 64), (7, 1536, 1536, 32), (8, 250, 5120, 128),
    (9, 64, 1536, 64), (16, 129, 640, 32), (17, 40, 1536, 128), (33, 257, 2048, 64), (64, 48, 1024, 32), (100, 31, 256, 128),
    (3, 70, 1536, 1536), (1, 20, 13824, 64), (5, 24, 1120, 224), (1, 15360, 5120, 128)])
def test_linear_w4_group(m, n, k, group, xdtype):
    g = _gen(m * 7919 + n * 31 + k + group)
    packed, scales = _w4_case(g, n, k, group)
    if xdtype == torch.int8:
        x = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        act = torch.rand(m, generator=g, device="cuda") / 40
        _check_w4(x, packed, scales, None, act)
        _check_w4(x, packed, scales, _randn(g, n, dtype=BF), act, BF)
    else:
        x = _randn(g, m, k, dtype=xdtype)
        _check_w4(x, packed, scales)
        _check_w4(x, packed, scales, _randn(g, n, dtype=xdtype))
        _check_w4(x, packed, scales, None, None, FP if xdtype == BF else BF)


def test_linear_w4_group_every_code_and_column():
    """A one-hot token reads one column: every nibble of every word, exactly."""
    from dsaquant_b200.kernels.w4_group import linear_w4_group

    g = _gen(5)
    n, k = 48, 256
    for group in (32, 64, 128):
        packed, _ = _w4_case(g, n, k, group)
        scales = torch.full((n, k // group), 0.5, device="cuda", dtype=FP)
        want = (_codes_of(packed) * 0.5).t()
        for dt in (BF, FP):
            assert torch.equal(linear_w4_group(torch.eye(k, device="cuda", dtype=dt), packed, scales).double(), want)
        assert torch.equal(linear_w4_group(torch.eye(k, device="cuda", dtype=torch.int8), packed, scales,
                                           act_scale=torch.ones(k, device="cuda")).double(), want)


def test_linear_w4_group_tokens_do_not_mix():
    """A token that holds a NaN leaves the others as they were; a token's value does not depend on its batch."""
    from dsaquant_b200.kernels.w4_group import linear_w4_group

    g = _gen(6)
    packed, scales = _w4_case(g, 200, 1536, 64)
    x = _randn(g, 8, 1536, dtype=BF)
    clean = linear_w4_group(x, packed, scales)
    x[3, 77] = float("nan")
    got = linear_w4_group(x, packed, scales)
    keep = [0, 1, 2, 4, 5, 6, 7]
    assert torch.equal(got[keep], clean[keep]) and bool(torch.isnan(got[3]).all())
    assert torch.equal(linear_w4_group(x[5:6], packed, scales), clean[5:6])


def test_linear_w4_group_views_leading_dims_refusals():
    from dsaquant_b200.kernels.w4_group import linear_w4_group

    g = _gen(7)
    packed, scales = _w4_case(g, 64, 256, 64)
    wide = _randn(g, 2, 3, 520, dtype=FP)
    part = wide[..., 4:260]
    assert torch.equal(_check_w4(part, packed, scales), _check_w4(part.contiguous(), packed, scales))
    assert linear_w4_group(wide[:, :0, 4:260], packed, scales).shape == (2, 0, 64)
    x = part.contiguous()
    for bad in (lambda: linear_w4_group(x[..., :128], packed, scales), lambda: linear_w4_group(x, packed, scales[:, :3]),
                lambda: linear_w4_group(x, packed, scales, act_scale=torch.ones(6, device="cuda")),
                lambda: linear_w4_group(x.to(torch.int8), packed, scales),
                lambda: linear_w4_group(x.to(torch.int8), packed, scales, act_scale=torch.ones(5, device="cuda")),
                lambda: linear_w4_group(x, packed, scales, torch.ones(65, device="cuda")),
                lambda: linear_w4_group(x, packed, scales, out_dtype=F32),
                lambda: linear_w4_group(x, packed.t().contiguous().t(), scales),
                lambda: linear_w4_group(x, packed, scales.cpu())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        linear_w4_group(x.float(), packed, scales)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n, k, group", [(3, 64, 32), (70, 640, 64), (16, 1536, 128), (5, 1536, 1536)])
def test_quantize_weight_grouped(n, k, group, dtype):
    from dsaquant_b200.kernels.w4_group import quantize_weight_grouped

    w = (_randn(_gen(n + k), n, k) * 0.02).to(dtype)
    w[0, :group] = 0
    packed, scales = quantize_weight_grouped(w, group)
    assert packed.shape == (n, k // 2) and scales.shape == (n, k // group)
    grouped = w.double().reshape(n, k // group, group)
    want = grouped.abs().amax(-1).clamp_min(1e-5) / 7
    # fp32 quotient, then fp16 (its subnormals step by 2^-24)
    _within(scales, want, 2.0 ** -11 * want + 2.0 ** -25 + 2.0 ** -23 * want)
    ratio = grouped / scales.double()[..., None]
    codes = _codes_of(packed).reshape(grouped.shape)
    _within(codes, ratio.clamp(-8, 7), 0.5 + 2.0 ** -20)
    assert int(codes[0, 0].abs().sum()) == 0


# ------------------------------------------------------------------------------------------------ rotary
def _rotate64(x, cos_sin, positions, interleaved, inverse=False):
    rd = 2 * cos_sin.shape[1]
    cs = cos_sin.double()[positions.long().clamp(0, cos_sin.shape[0] - 1)][:, None]
    c, s = cs[..., 0], cs[..., 1] * (-1 if inverse else 1)
    r, rest = x[..., :rd].double(), x[..., rd:].double()
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rd // 2], r[..., rd // 2:])
    u, v = a * c - b * s, a * s + b * c
    size = (a.abs() + b.abs()) * cs.abs().amax()
    join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat([p, q], -1))
    keep = (positions < 0)[:, None, None]
    out = torch.cat([join(u, v), rest], -1)
    return torch.where(keep, x.double(), out), torch.cat([join(size, size), torch.zeros_like(rest)], -1)


def _check_rotary(q, k, table, positions, interleaved, inverse=False):
    from dsaquant_b200.rotary import apply_rotary

    got = apply_rotary(q, k, table, positions, interleaved=interleaved, inverse=inverse)
    for x, y in zip((q, k), got):
        if x is None:
            assert y is None
            continue
        want, size = _rotate64(x, table, positions, interleaved, inverse)
        # two products and a sum in fp32, one rounding to the type; what is not rotated is exact
        _within(y, want, torch.where(size > 0, HALF_STEP[x.dtype] * want.abs() + HALF_SUB[x.dtype] + 2.0 ** -22 * size, 0.0))
    return got


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("t, hq, hk, hd, rd", [
    (1, 40, 8, 128, 128), (1, 1, 0, 64, 64), (7, 3, 1, 128, 64), (33, 12, 2, 128, 32), (5, 4, 4, 96, 48), (300, 2, 1, 64, 16),
    (4, 5, 2, 80, 10), (3, 2, 2, 7, 2), (9, 1, 1, 512, 512), (2, 3, 1, 512, 2), (6, 130, 3, 16, 16), (11, 2, 2, 72, 40)])
def test_apply_rotary(t, hq, hk, hd, rd, dtype, interleaved):
    from dsaquant_b200.rotary import rotary_table

    g = _gen(t + hq * 7 + hd + rd)
    table = rotary_table(1000, rd, device="cuda")
    q, k = _randn(g, t, hq, hd, dtype=dtype), _randn(g, t, hk, hd, dtype=dtype) if hk else None
    positions = torch.randint(0, 1000, (t,), generator=g, device="cuda")
    _check_rotary(q, k, table, positions, interleaved)
    _check_rotary(q, k, table, positions.int(), interleaved, inverse=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 3])
def test_apply_rotary_reads_views_in_place_and_writes_in_place(interleaved, offset):
    from dsaquant_b200.rotary import apply_rotary, rotary_table

    g = _gen(11)
    t, hq, hk, hd = 50, 6, 2, 64
    table = rotary_table(400, 32, device="cuda")
    flat = _randn(g, t * (hq + 2 * hk) * hd + 8, dtype=BF)[offset:offset + t * (hq + 2 * hk) * hd]
    qkv = flat.view(t, hq + 2 * hk, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    positions = torch.arange(100, 100 + 2 * t, 2, device="cuda")
    want = _check_rotary(q, k, table, positions, interleaved)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)         # [T, heads, hd] whose memory is [heads, T, hd]
    assert torch.equal(apply_rotary(by_head, None, table, positions, interleaved=interleaved)[0], want[0])
    before = v.clone()
    got = apply_rotary(q, k, table, positions, interleaved=interleaved, inplace=True)
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, before)


def test_apply_rotary_padding_and_positions_behind_the_table():
    from dsaquant_b200.rotary import apply_rotary, rotary_table

    g = _gen(12)
    table = rotary_table(16, 64, device="cuda")
    q = _randn(g, 6, 3, 128, dtype=FP)
    q[4, 1, 5] = float("nan")                                        # garbage in a padding row stays what it is
    positions = torch.tensor([0, 15, 16, -1, -7, 1 << 40], device="cuda")
    for interleaved in (False, True):
        out, _ = apply_rotary(q, None, table, positions, interleaved=interleaved)
        assert torch.equal(out[[3, 4]].view(torch.int16), q[[3, 4]].view(torch.int16))
        assert bool(torch.isnan(out[[2, 5]][..., :64]).all()) and torch.equal(out[[2, 5]][..., 64:], q[[2, 5]][..., 64:])
        assert torch.equal(out[0], q[0]) and bool(torch.isfinite(out[1]).all())


def test_apply_rotary_round_trip_gradient_and_refusals():
    """The inverse is the transpose: <R q, y> = <q, R^T y>, which makes it the gradient; checked against differences."""
    from dsaquant_b200.rotary import apply_rotary, rotary_table

    g = _gen(13)
    table = rotary_table(64, 32, device="cuda")
    q, y = _randn(g, 5, 2, 32), _randn(g, 5, 2, 32)
    pos = torch.arange(5, device="cuda") * 9
    grad, _ = apply_rotary(y, None, table, pos, inverse=True)
    step = torch.zeros_like(q)
    step[2, 1, 7] = 0.5
    hi, lo = (apply_rotary(q + d, None, table, pos)[0].double() for d in (step, -step))
    # the map is linear, so a wide difference is exact up to the fp32 roundings of its 64 terms
    assert abs(((hi - lo) * y.double()).sum().item() - grad[2, 1, 7].item()) < 64 * 2.0 ** -23 * 10
    x = q.half()
    for bad in (lambda: apply_rotary(x, x[:4], table, pos), lambda: apply_rotary(x, None, table, pos[:4]),
                lambda: apply_rotary(x, None, table[:, :, :1], pos), lambda: apply_rotary(x, None, table.double(), pos),
                lambda: apply_rotary(x, None, rotary_table(4, 34, device="cuda"), pos),
                lambda: apply_rotary(x.transpose(1, 2), None, table, pos), lambda: apply_rotary(x, x.float(), table, pos),
                lambda: apply_rotary(x, None, table, pos.float()), lambda: apply_rotary(x, None, table.cpu(), pos),
                lambda: apply_rotary(x[:, :0], None, table, pos),
                lambda: apply_rotary(x[:, :1].expand(5, 3, 32), None, table, pos, inplace=True),
                lambda: apply_rotary(x, x[:1].expand(5, 2, 32), table, pos, inplace=True)):
        with pytest.raises(ValueError):
            bad()
    assert apply_rotary(x[:0], None, table, pos[:0])[0].shape == (0, 2, 32)


# ------------------------------------------------------------------------------------------------ window_attention
def _attention64(q, k, v, window, sinks, lens, scale):
    b, lq, hq, hd = q.shape
    lk, share = k.shape[1], hq // k.shape[2]
    kk, vv = (t.double().repeat_interleave(share, 2) for t in (k, v))
    at = (lens.long()[:, None] - lq + torch.arange(lq, device="cuda"))[:, None, :, None]
    j = torch.arange(lk, device="cuda")
    seen = (j <= at) & ((j > at - window) | (j < sinks))
    score = torch.einsum("bqhd,bkhd->bhqk", q.double(), kk) * scale
    size = torch.einsum("bqhd,bkhd->bhqk", q.double().abs(), kk.abs()) * scale
    score = score.masked_fill(~seen, -math.inf)
    lse = score.logsumexp(-1)
    p = torch.where(seen, (score - torch.where(lse.isinf(), 0.0, lse)[..., None]).exp(), 0.0)
    out = torch.einsum("bhqk,bkhd->bqhd", p, vv)
    spread = torch.einsum("bhqk,bkhd->bqhd", p, vv.abs())
    low = torch.einsum("bhqk,bkhd->bqhd", seen.double().expand_as(p), vv.abs())
    worst = torch.where(seen, size, 0.0).amax(-1)      # [b, h, q]
    return out, lse, spread, low, worst


def _check_attention(q, k, v, window, sinks=0, kv_lens=None, scale=None):
    from dsaquant_b200.window_attention import window_attention

    out, lse = window_attention(q, k, v, window, sinks, kv_lens=kv_lens, scale=scale, return_lse=True)
    b, lq, hq, hd = q.shape
    lk = k.shape[1]
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (b, hq, lq) and lse.dtype == F32
    lens = kv_lens if kv_lens is not None else torch.full((b,), lk, device="cuda")
    want, want_lse, spread, low, worst = _attention64(q, k, v, window, sinks, lens.clamp(0, lk), scale or hd ** -0.5)
    # a score: hd products summed, then scaled into log2 units; its error is relative in the weight, as is the one
    # of each exponential and of each step of the running maximum (2^-21 covers a thousandth of a percent per 20 tiles)
    ds = ((hd + 4) * 2.0 ** -23 * worst + 2.0 ** -21 * (1 + lk / 64 / 16))
    none = want_lse == -math.inf
    assert bool((lse[none] == -math.inf).all())
    _within(torch.where(none, 0.0, lse), torch.where(none, 0.0, want_lse), ds + 2.0 ** -22 * torch.where(none, 0.0, want_lse.abs()))
    ds = ds.transpose(1, 2)[..., None]
    half, sub = HALF_STEP[q.dtype], HALF_SUB[q.dtype]
    # weights rounded to the type (absolutely, once below its normal range), the sum in fp32, the result rounded
    _within(out, want, half * want.abs() + sub + (half + 2 * ds + lk * 2.0 ** -23) * spread + sub * low)
    assert bool((out.transpose(1, 2)[none] == 0).all())
    return out, lse


def _qkv(g, b, lq, lk, hq, hk, hd, dtype):
    return (_randn(g, b, lq, hq, hd, dtype=dtype), _randn(g, b, lk, hk, hd, dtype=dtype), _randn(g, b, lk, hk, hd, dtype=dtype))


@pytest.mark.parametrize("dtype, hd", [(BF, 128), (FP, 64), (FP, 128), (BF, 64)])
@pytest.mark.parametrize("b, lq, lk, hq, hk, window, sinks", [
    (1, 1, 1, 1, 1, 1, 0), (2, 1, 300, 8, 2, 64, 4), (1, 1, 2500, 40, 8, 1000, 4), (3, 1, 129, 5, 5, 1, 1), (1, 64, 64, 2, 2, 64, 0),
    (2, 65, 65, 4, 1, 17, 3), (1, 200, 200, 3, 3, 1000, 0), (2, 130, 517, 4, 2, 100, 70), (1, 3, 900, 12, 2, 333, 130),
    (1, 517, 517, 10, 2, 128, 0), (2, 700, 1100, 2, 1, 256, 5), (1, 1025, 1025, 1, 1, 1, 0), (1, 300, 1500, 6, 6, 1024, 64),
    (2, 256, 1024, 2, 2, 512, 1), (1, 129, 2000, 64, 1, 700, 9), (33, 2, 70, 4, 4, 40, 2)])
def test_window_attention(b, lq, lk, hq, hk, window, sinks, dtype, hd):
    g = _gen(b + lq * 3 + lk * 5 + hq)
    _check_attention(*_qkv(g, b, lq, lk, hq, hk, hd, dtype), window, sinks)


@pytest.mark.parametrize("dtype, hd", [(BF, 128), (FP, 64)])
@pytest.mark.parametrize("lq, lk, hq, hk, window, sinks", [
    (1, 600, 8, 2, 100, 4), (5, 600, 4, 4, 1, 0), (200, 600, 4, 2, 64, 3), (600, 600, 2, 1, 250, 80), (300, 300, 8, 1, 5000, 0)])
def test_window_attention_lengths_and_garbage_behind_them(lq, lk, hq, hk, window, sinks, dtype, hd):
    g = _gen(lq + lk + window)
    lens = torch.tensor([0, 1, 63, 64, 65, lk // 2, lk - 1, lk], dtype=torch.int32, device="cuda")
    q, k, v = _qkv(g, len(lens), lq, lk, hq, hk, hd, dtype)
    want = _check_attention(q, k, v, window, sinks, lens)
    for i, n in enumerate(lens.tolist()):
        k[i, n:], v[i, n:] = float("nan"), float("inf")              # unwritten cache
        low = n - lq - window + 1                                    # freed lines: before every window, behind the sinks
        if low > sinks:
            k[i, sinks:low], v[i, sinks:low] = float("inf"), float("nan")
    from dsaquant_b200.window_attention import window_attention

    got = window_attention(q, k, v, window, sinks, kv_lens=lens, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # lengths outside 0..Lk are clamped
    wide = lens.clone()
    wide[0], wide[-1] = -5, lk + 1000
    got = window_attention(q, k, v, window, sinks, kv_lens=wide, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_window_attention_large_scores_and_scale():
    g = _gen(21)
    q, k, v = _qkv(g, 1, 150, 400, 4, 2, 64, BF)
    _check_attention(q * 8, k * 8, v, 100, 4)
    _check_attention(q, k, v, 100, 4, scale=0.5)


@pytest.mark.parametrize("lq, dtype, hd", [(1, BF, 128), (3, FP, 64), (60, BF, 64), (400, BF, 128), (400, FP, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_window_attention_not_finite_scores_reach_the_rows_that_see_them(lq, dtype, hd, value):
    from dsaquant_b200.window_attention import window_attention

    lk, window, sinks = 400, 90, 2
    g = _gen(25)
    q, k, v = _qkv(g, 1, lq, lk, 2, 1, hd, dtype)
    q[..., 0] = 1.0
    clean, clean_lse = window_attention(q, k, v, window, sinks, return_lse=True)
    for key in (3, 130, 131, 192, 255, 333, 398, 399):               # every kind of place in a key tile
        bad = k.clone()
        bad[0, key, 0, 0] = value
        out, lse = window_attention(q, bad, v, window, sinks, return_lse=True)
        at = lk - lq + torch.arange(lq, device="cuda")
        sees = (at >= key) & (key > at - window)
        assert torch.equal(out[0, ~sees], clean[0, ~sees]) and torch.equal(lse[0][:, ~sees], clean_lse[0][:, ~sees])
        assert bool(torch.isnan(out[0, sees]).all()) and not bool(torch.isfinite(lse[0][:, sees]).any())


def test_window_attention_strided_views_and_head_major_cache():
    from dsaquant_b200.window_attention import window_attention

    g = _gen(22)
    for lq in (1, 130):
        qkv = _randn(g, 2, 200, 8 + 2 + 2, 128, dtype=BF)
        q, k, v = qkv[:, 200 - lq:, :8], qkv[:, :, 8:10], qkv[:, :, 10:]
        want = _check_attention(q, k, v, 50, 4)[0]
        assert torch.equal(want, window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 50, 4))
        major = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]   # memory [B, heads, L, hd]
        assert torch.equal(want, window_attention(q, *major, 50, 4))
        odd = torch.empty(2 * 200 * 2 * 128 + 1, device="cuda", dtype=BF)[1:].view(2, 200, 2, 128)
        odd.copy_(k)                                                               # two bytes off: copied first
        assert torch.equal(want, window_attention(q, odd, v, 50, 4))


def test_window_attention_shared_heads_and_sequences():
    """Keys that several heads or sequences share by a pitch of 0."""
    g = _gen(26)
    for lq in (1, 40, 300):
        q = _randn(g, 2, lq, 4, 64, dtype=BF)
        k = _randn(g, 1, 300, 1, 64, dtype=BF).expand(2, 300, 4, 64)
        _check_attention(q, k, k, 100, 3)
        one = k[:, :, :1]                                             # the prompt all sequences share
        _check_attention(q, one, one, 100, 3)


def test_window_attention_wide_window_is_causal_and_merges():
    """Two runs of keys joined by merge_attention are the attention over all of them."""
    from dsaquant_b200.attention_qkv import merge_attention
    from dsaquant_b200.window_attention import window_attention

    g = _gen(23)
    q, k, v = _qkv(g, 1, 1, 500, 4, 4, 128, BF)
    whole = window_attention(q, k, v, 500)
    o1, l1 = window_attention(q, k[:, :200], v[:, :200], 200, return_lse=True)
    o2, l2 = window_attention(q, k[:, 200:], v[:, 200:], 300, return_lse=True)
    both = merge_attention(o1.transpose(1, 2), l1, o2.transpose(1, 2), l2).view_as(whole)
    # each side and the whole carry a rounded result and rounded weights: four half steps of magnitudes below max |v|
    assert (both.double() - whole.double()).abs().max().item() <= 4 * 2.0 ** -8 * v.abs().max().item()


def test_window_attention_far_offsets():
    """A cache whose last sequence starts past 2^32 elements."""
    from dsaquant_b200.window_attention import window_attention

    b, lk, hd = 2, 300, 128
    pitch = (1 << 32) + 1024
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("not enough free memory")
    big = torch.empty(pitch + lk * hd, device="cuda", dtype=BF)
    k = big.as_strided((b, lk, 1, hd), (pitch, hd, hd, 1))
    g = _gen(24)
    k.copy_(_randn(g, b, lk, 1, hd, dtype=BF))
    for lq in (1, 200):
        q = _randn(g, b, lq, 2, hd, dtype=BF)
        got = window_attention(q, k, k, 100, 4)
        assert torch.equal(got, window_attention(q, k.contiguous(), k.contiguous(), 100, 4))
    del big, k


def test_window_attention_refusals_and_empty():
    from dsaquant_b200.window_attention import window_attention

    q, k = torch.zeros(2, 3, 4, 64, device="cuda", dtype=FP), torch.zeros(2, 5, 2, 64, device="cuda", dtype=FP)
    for bad in (dict(window=0), dict(window=4, sinks=-1), dict(window=4, scale=0.0), dict(window=4, kv_lens=torch.zeros(2, device="cuda")),
                dict(window=4, kv_lens=torch.zeros(3, device="cuda", dtype=torch.int32))):
        with pytest.raises(ValueError):
            window_attention(q, k, k, **bad)
    for a, b in ((q[..., :32], k[..., :32]), (q[:, :, :3], k), (q, k[:1]), (q, k.bfloat16()), (q[0], k[0])):
        with pytest.raises(ValueError):
            window_attention(a, b, b, 4)
    with pytest.raises(RuntimeError):
        window_attention(q.float(), k.float(), k.float(), 4)
    assert window_attention(q[:, :0], k, k, 4).shape == (2, 0, 4, 64)
    out, lse = window_attention(q + 1, k[:, :0], k[:, :0], 4, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


# ------------------------------------------------------------------------------------------------ together
class _Layer:
    """A decoder layer on 4-bit weights with a windowed cache, as a user writes it with these operators."""

    def __init__(self, g, d=512, hq=4, hk=2, hd=128, ff=1024, window=48, sinks=4):
        from dsaquant_b200.kernels.w4_group import quantize_weight_grouped
        from dsaquant_b200.rotary import rotary_table

        self.hq, self.hk, self.hd, self.window, self.sinks = hq, hk, hd, window, sinks
        mk = lambda n, k: quantize_weight_grouped(_randn(g, n, k) * k ** -0.5, 64)  # noqa: E731
        self.qkv, self.o, self.up, self.down = mk((hq + 2 * hk) * hd, d), mk(d, hq * hd), mk(ff, d), mk(d, ff)
        self.n1, self.n2 = (1 + 0.1 * _randn(g, d)).to(BF), (1 + 0.1 * _randn(g, d)).to(BF)
        self.table = rotary_table(512, 64, device="cuda")

    def __call__(self, x, stream, cache, pos, lens):
        """x, stream [B, T, d]: the last sublayer's output and the residual stream; cache (k, v) [B, L, hk, hd] is written
        at `pos` [T]."""
        from dsaquant_b200.kernels.rms_norm import rms_norm_quant
        from dsaquant_b200.kernels.w4_group import linear_w4_group
        from dsaquant_b200.rotary import apply_rotary
        from dsaquant_b200.window_attention import window_attention

        b, t, _ = x.shape
        codes, scale, stream = rms_norm_quant(x, self.n1, residual=stream)
        qkv = linear_w4_group(codes, *self.qkv, act_scale=scale, out_dtype=BF).view(b * t, -1, self.hd)
        q, k, v = qkv.split((self.hq, self.hk, self.hk), 1)
        q, k = apply_rotary(q, k, self.table, pos.repeat(b))
        cache[0].index_copy_(1, pos, k.view(b, t, self.hk, self.hd))
        cache[1].index_copy_(1, pos, v.reshape(b, t, self.hk, self.hd))
        o = window_attention(q.view(b, t, self.hq, self.hd), *cache, self.window, self.sinks, kv_lens=lens)
        x = linear_w4_group(o.flatten(2), *self.o)
        codes, scale, stream = rms_norm_quant(x, self.n2, residual=stream)
        h = torch.nn.functional.silu(linear_w4_group(codes, *self.up, act_scale=scale, out_dtype=BF))
        return linear_w4_group(h, *self.down), stream

    def exact(self, x, stream):
        """The whole sequence at once in 64 bits, without 8-bit codes."""
        w = lambda p: _codes_of(p[0]) * p[1].double().repeat_interleave(64, 1)  # noqa: E731
        norm = lambda s, n: s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-6) * n.double()  # noqa: E731
        stream = x.double() + stream.double()
        b, t, _ = x.shape
        q, k, v = (norm(stream, self.n1) @ w(self.qkv).t()).view(b, t, -1, self.hd).split((self.hq, self.hk, self.hk), 2)
        pos = torch.arange(t, device="cuda")
        q, k = (torch.stack([_rotate64(y[i], self.table, pos, False)[0] for i in range(b)]) for y in (q, k))
        lens = torch.full((b,), t, device="cuda")
        o = _attention64(q, k, v, self.window, self.sinks, lens, self.hd ** -0.5)[0]
        y = o.flatten(2) @ w(self.o).t()
        stream = stream + y
        h = torch.nn.functional.silu(norm(stream, self.n2) @ w(self.up).t())
        return h @ w(self.down).t(), stream


def test_decoder_layer_prompt_then_tokens():
    """A prompt and then single tokens on the cache give what the whole sequence gives at once."""
    g = _gen(31)
    layer = _Layer(g)
    b, prompt, total = 2, 70, 80
    x, s = _randn(g, b, total, 512, dtype=BF), _randn(g, b, total, 512, dtype=BF)
    cache = [torch.full((b, 128, 2, 128), float("nan"), device="cuda", dtype=BF) for _ in range(2)]
    outs = []
    for lo, hi in [(0, prompt)] + [(i, i + 1) for i in range(prompt, total)]:
        lens = torch.full((b,), hi, dtype=torch.int32, device="cuda")
        outs.append(layer(x[:, lo:hi], s[:, lo:hi], cache, torch.arange(lo, hi, device="cuda"), lens))
    y, stream = (torch.cat([o[i] for o in outs], 1).double() for i in (0, 1))
    want_y, want_stream = layer.exact(x, s)
    # 8-bit codes: steps of max / 127, about 4 / 127 of the row's root mean square, uniform errors of 1 / sqrt(12) of
    # one: 0.9 % of a value at each norm; bf16 adds 2^-8 / sqrt(3) = 0.2 % a tensor.  Attention and products keep relative
    # errors of independent terms, so a few percent in norm covers the chain with room for its gains.
    rel = lambda a, b: ((a - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(stream, want_stream) < 0.02 and rel(y, want_y) < 0.05


def test_decoder_step_captures_and_replays():
    """One token's step as a CUDA graph: positions, lengths and inputs are data, replays follow them bit for bit."""
    g = _gen(32)
    layer = _Layer(g)
    b = 2
    x, s = _randn(g, b, 1, 512, dtype=BF), _randn(g, b, 1, 512, dtype=BF)
    fill = [_randn(g, b, 128, 2, 128, dtype=BF) for _ in range(2)]
    cache = [c.clone() for c in fill]
    pos, lens = torch.tensor([60], device="cuda"), torch.full((b,), 61, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, s, cache, pos, lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, s, cache, pos, lens)
    for at in (60, 61, 100):
        x.copy_(_randn(g, b, 1, 512, dtype=BF))
        pos.fill_(at)
        lens.fill_(at + 1)
        for c, f in zip(cache, fill):
            c.copy_(f)
        graph.replay()
        got = [o.clone() for o in out] + [c.clone() for c in cache]
        for c, f in zip(cache, fill):
            c.copy_(f)
        want = list(layer(x, s, cache, pos, lens)) + cache
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_on_another_stream():
    """Work enqueued on a side stream stays on it: results equal those of the default stream."""
    from dsaquant_b200.window_attention import window_attention

    g = _gen(33)
    q, k, v = _qkv(g, 4, 1, 3000, 8, 2, 128, BF)
    want = window_attention(q, k, v, 2048, 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append([window_attention(q, k, v, 2048, 4) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for group in outs for o in group)


def test_prompts_on_two_streams_beside_the_gemm():
    """Prompt attention and the tcgen05 GEMM both want all of an SM's tensor memory: calls that overlap on two streams
    wait for one another and give what they give alone."""
    from dsaquant_b200.kernels import vdm_w4a4 as vdm
    from dsaquant_b200.window_attention import window_attention

    g = _gen(34)
    q, k, v = _qkv(g, 1, 700, 1500, 8, 2, 128, BF)
    packed, sp, _ = vdm.quantize_weight_per_channel(_randn(g, 1536, 1536, dtype=FP) * 0.02)
    codes = torch.randint(-8, 8, (3000, 1536), generator=g, device="cuda", dtype=torch.int8)
    scale = torch.rand(3000, generator=g, device="cuda")
    want, want_gemm = window_attention(q, k, v, 400, 4), vdm.linear_prequantized(codes, scale, packed, sp)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(3)]
    outs, gemms = [], []
    for _ in range(10):
        for st in side[:2]:
            with torch.cuda.stream(st):
                outs.append(window_attention(q, k, v, 400, 4))
        with torch.cuda.stream(side[2]):
            gemms.append(vdm.linear_prequantized(codes, scale, packed, sp))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs) and all(torch.equal(o, want_gemm) for o in gemms)
    assert vdm.last_device_status() == 0


def test_prompt_layer_captures_and_replays():
    """A chunk of a prompt as a CUDA graph: lengths and positions are data."""
    g = _gen(35)
    layer = _Layer(g)
    b, t = 2, 130
    x, s = _randn(g, b, t, 512, dtype=BF), _randn(g, b, t, 512, dtype=BF)
    fill = [_randn(g, b, 400, 2, 128, dtype=BF) for _ in range(2)]
    cache = [c.clone() for c in fill]
    pos, lens = torch.arange(t, device="cuda"), torch.full((b,), t, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, s, cache, pos, lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, s, cache, pos, lens)
    for start in (0, 7, 200):
        x.copy_(_randn(g, b, t, 512, dtype=BF))
        pos.copy_(torch.arange(start, start + t, device="cuda"))
        lens.copy_(torch.tensor([start + t, max(start - 50, 0)], device="cuda"))   # the second sequence ends before its rows
        for c, f in zip(cache, fill):
            c.copy_(f)
        graph.replay()
        got = [o.clone() for o in out] + [c.clone() for c in cache]
        for c, f in zip(cache, fill):
            c.copy_(f)
        want = list(layer(x, s, cache, pos, lens)) + cache
        assert all(torch.equal(a, b) for a, b in zip(got, want))
