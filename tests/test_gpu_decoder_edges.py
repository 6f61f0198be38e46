"""Decoder-layer operators where they can go wrong without a wrong formula: values beside a rounding border, values that are
not finite, memory that is shared, sizes that ask for much workspace.  Helpers and tolerances are those of
test_gpu_decoder_ops."""
import pytest
import torch

from test_gpu_decoder_ops import BF, F32, FP, HALF_STEP, HALF_SUB, _attention64, _check_w4, _codes_of, _gen, _qkv, _randn, _w4_case, _within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ rms_norm_quant
def _nearest_e4m3(t):
    """t (64 bits, |t| <= 448) rounded to the nearest e4m3 value with ties to even, by a search over all of them."""
    table = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()   # 0 .. 448
    mid = (table[1:] + table[:-1]) / 2
    low = torch.searchsorted(mid, t.abs())                           # mid[low - 1] < |t| <= mid[low]
    tie = (low < 126) & (t.abs() == mid[low.clamp(max=125)]) & (low % 2 == 1)
    return torch.where(t < 0, -1.0, 1.0) * table[low + tie.long()]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [64, 255, 256, 257, 768, 769])
def test_rms_norm_quant_e4m3_short_rows_share_a_block(d, dtype):
    """Up to 768 values a row has one warp and a block eight rows: each row's codes are the exact ones, whatever the warps beside
    it do, and the same in every run."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(51 + d)
    m = 6_000_000 // d
    x, w = _randn(g, m, d, dtype=dtype), (1 + 0.1 * _randn(g, d)).to(dtype)
    codes, scale = rms_norm_quant(x, w, out_dtype=torch.float8_e4m3fn)
    for _ in range(5):
        again = rms_norm_quant(x, w, out_dtype=torch.float8_e4m3fn)
        assert torch.equal(codes.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scale, again[1])
    y = x.double() * w.double()                                      # the rsqrt cancels in y / max|y|
    t = y * 448 / y.abs().amax(-1, keepdim=True)
    normal = t.abs() >= 2.0 ** -6
    assert torch.equal(codes.double()[normal], _nearest_e4m3(t)[normal])


@pytest.mark.parametrize("dtype, d", [(F32, 1536), (F32, 200), (F32, 777), (BF, 5120)])
def test_rms_norm_quant_e4m3_small_quotients_are_exact_too(dtype, d):
    """Rows with a few channels far larger than the rest have most of their quotients below 2^-6, where e4m3's steps are
    absolute: tens of millions of values, none on the wrong side of a border."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(52 + d)
    w = 0.5 + torch.rand(d, generator=g, device="cuda")
    w[::97] *= 50000.0
    w = w.to(dtype)
    small = 0
    for _ in range(10):
        x = _randn(g, 4_000_000 // d, d, dtype=dtype)
        codes, _ = rms_norm_quant(x, w, out_dtype=torch.float8_e4m3fn)
        y = x.double() * w.double()
        t = y * 448 / y.abs().amax(-1, keepdim=True)
        assert torch.equal(codes.double(), _nearest_e4m3(t))
        small += int((t.abs() < 2.0 ** -6).sum())
    assert small > 10_000_000


def test_rms_norm_quant_e4m3_largest_value_in_64_bits():
    """Two values so close that their fp32 products come out in the wrong order, and quotients that lie on one side of a
    border for one of them and on the other side for the other.  Rows of whole numbers, whose squares add up exactly."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(53)
    rows, d, found = 200_000, 32, 0
    x = torch.randint(129, 256, (rows, d), generator=g, device="cuda").float()
    w = 1 + torch.rand(rows, d, generator=g, device="cuda")
    w[:, 0] += 64                                                    # values 0 and 1 are the largest by far
    # torch's root may differ from the kernel's in the last bit; then a row is only not as hard as it was meant to be
    rstd = torch.rsqrt(x.square().mean(-1) + 1e-6)
    w[:, 1] = (x[:, 0].double() * w[:, 0].double() / x[:, 1].double()).float()
    w[:, 1] = (w[:, 1].view(torch.int32) + 1).view(F32)              # the true maximum is value 1
    top = x[:, 1].double() * w[:, 1].double()
    fp32 = x * rstd[:, None] * w
    wrong = (top > x[:, 0].double() * w[:, 0].double()) & (fp32[:, 1] < fp32[:, 0])
    for j in range(2, d):                                            # quotients as near to a border as fp32 weights allow
        border = 1.0625 * 2.0 ** (j % 6) + 0.125 * 2.0 ** (j % 6) * (j % 7)
        w[:, j] = (border * top / (448 * x[:, j].double())).float()
    for row in wrong.nonzero()[:, 0][:300].tolist():
        y = x[row].double() * w[row].double()
        t, t0 = y * 448 / y.abs().amax(), y * 448 / y[0].abs()
        want, with_other = _nearest_e4m3(t.clamp(max=448.0)), _nearest_e4m3(t0.clamp(max=448.0))
        if torch.equal(want, with_other):
            continue
        found += 1
        codes, _ = rms_norm_quant(x[row:row + 1], w[row], out_dtype=torch.float8_e4m3fn)
        assert torch.equal(codes[0].double(), want)
    assert found > 10


@pytest.mark.parametrize("d, eps", [(1536, 1.0), (200, 0.25), (777, 1.0), (64, 2.0 ** -10)])
def test_rms_norm_quant_e4m3_rows_with_the_least_scale_are_exact_too(d, eps):
    """Rows of max|y| up to and around 1e-5, whose scale does not follow them."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(54 + d)
    w = 1 + 0.1 * _randn(g, d)
    least = 0
    for _ in range(6):
        m = 3_000_000 // d
        x = (2 * torch.rand(m, d, generator=g, device="cuda") - 1) * eps ** 0.5 * 1e-5
        x[::3] *= torch.rand(len(x[::3]), 1, generator=g, device="cuda")
        codes, scale = rms_norm_quant(x, w, eps, out_dtype=torch.float8_e4m3fn)
        y = x.double() * w.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + eps)
        top = y.abs().amax(-1, keepdim=True)
        assert torch.equal(codes.double(), _nearest_e4m3(y * 448 / top.clamp_min(1e-5)))
        least += int((top < 1e-5).sum())
    assert least > 1000


@pytest.mark.parametrize("d, clip", [(512, 1.0), (5120, 1.0), (777, 0.9), (64, 0.5)])
def test_rms_norm_quant_int8_codes_are_those_of_the_division(d, clip):
    """codes = clamp(rint(y / scale)) with fp32's quotient, as the package's other quantiser rounds, at quotients beside the
    borders.  Squares far below eps = 1 leave rsqrt(1) = 1, so y is x."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(55 + d)
    m = 1_000_000 // d
    top = (1 + torch.rand(m, 1, generator=g, device="cuda")) * 2.0 ** -15
    scale = (top / torch.full_like(top, 127.0)) * torch.tensor(clip, device="cuda")   # (by a number torch multiplies with 1 / 127)
    half = torch.randint(-128, 128, (m, d), generator=g, device="cuda") + 0.5
    x = half * scale
    x = (x.view(torch.int32) + torch.randint(-1, 2, (m, d), generator=g, device="cuda", dtype=torch.int32)).view(F32)
    x = torch.minimum(torch.maximum(x, -top), top)
    x[:, d // 2] = top[:, 0]
    assert x.square().mean(-1).max().item() < 2.0 ** -25
    codes, got_scale = rms_norm_quant(x, torch.ones(d, device="cuda"), 1.0, clip_ratio=clip)
    assert torch.equal(got_scale, scale[:, 0])
    assert torch.equal(codes.float(), (x / scale).round().clamp(-128, 127))


@pytest.mark.parametrize("out_dtype", [torch.int8, torch.float8_e4m3fn])
def test_rms_norm_quant_rows_outside_the_range_of_fp32_are_marked(out_dtype):
    """Squares that leave fp32's normal range, and scales whose reciprocal does, give NaN and codes 0, not numbers that are off."""
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant

    g = _gen(57)
    x = _randn(g, 8, 300)
    x[1] *= 1e-17
    x[2] *= 1e-22
    x[3] *= 1e-30
    x[4] = 0
    w = 1 + 0.1 * _randn(g, 300)
    top = 127.0 if out_dtype == torch.int8 else 448.0
    y = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True)) * w.double()
    want = y.abs().amax(-1) / top
    codes, scale = rms_norm_quant(x, w, 0.0, out_dtype=out_dtype)
    fine = [0, 1, 5, 6, 7]
    # as in _check_rms: 300 squares in a row's 32 threads, then the root, two products and a quotient
    _within(scale[fine], want[fine], (74 / 2 + 8) * 2.0 ** -24 * want[fine])
    assert bool(torch.isnan(scale[[2, 3, 4]]).all()) and bool((codes[[2, 3, 4]].float() == 0).all())
    codes, scale = rms_norm_quant(x, w, 1e-30, out_dtype=out_dtype)   # an eps of any use keeps them
    assert bool(torch.isfinite(scale).all()) and bool((codes[4].float() == 0).all())
    for clip, marked in ((1e-34, True), (1e-25, False), (1e25, False)):
        codes, scale = rms_norm_quant(x[4:6], w, out_dtype=out_dtype, clip_ratio=clip)
        # of the row of zeros, whose scale is 1e-5 / top * clip
        assert bool(torch.isnan(scale[0])) == marked and bool((codes[0].float() == 0).all())
        assert bool(torch.isfinite(scale[1]))


# ------------------------------------------------------------------------------------------------ window_attention
def _attention_bound(q, k, v, window, sinks, lens):
    """The definition in 64 bits and how far a result may be off (the terms are explained at _check_attention)."""
    lk, hd = k.shape[1], q.shape[3]
    want, lse, spread, low, worst = _attention64(q, k, v, window, sinks, lens, hd ** -0.5)
    ds = ((hd + 4) * 2.0 ** -23 * worst + 2.0 ** -21 * (1 + lk / 64 / 16)).transpose(1, 2)[..., None]
    half, sub = HALF_STEP[q.dtype], HALF_SUB[q.dtype]
    return want, half * want.abs() + sub + (half + 2 * ds + lk * 2.0 ** -23) * spread + sub * low


@pytest.mark.parametrize("dtype, hd", [(BF, 128), (FP, 64)])
@pytest.mark.parametrize("lq, hq, hk, lens, window, sinks", [
    (3, 2, 2, (400, 1), 90, 2), (16, 4, 2, (400, 5), 5000, 0), (2, 8, 1, (1500, 700), 1000, 70), (60, 4, 2, (400, 30), 90, 2),
    (127, 2, 1, (1500, 64), 5000, 0), (400, 2, 1, (400, 100), 90, 70), (300, 2, 2, (1500, 200), 700, 5), (200, 4, 1, (500, 199), 5000, 0)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_window_attention_not_finite_values_reach_only_the_rows_that_see_them(lq, hq, hk, lens, window, sinks, dtype, hd, value):
    """A value of V that is not finite changes its own column of the rows that see its key, and nothing else: not the rows
    before the key, not those past the window, not those that see nothing."""
    from dsaquant_b200.window_attention import window_attention

    g = _gen(61 + lq + hq)
    lk = lens[0]
    q, k, v = _qkv(g, 2, lq, lk, hq, hk, hd, dtype)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean, clean_lse = window_attention(q, k, v, window, sinks, kv_lens=kv_lens, return_lse=True)
    want, bound = _attention_bound(q, k, v, window, sinks, kv_lens)
    for last in (0, 1, lq // 2, lq - 1):                              # keys that the query `last` and those behind it see
        for column in (0, hd - 1, slice(None)):
            bad = v.clone()
            hit = torch.zeros(want.shape, dtype=torch.bool, device="cuda")
            for i, n in enumerate(lens):
                at = n - lq + torch.arange(lq, device="cuda")
                key = max(n - lq + last, 0)
                bad[i, key, hk - 1, column] = value
                sees = (at >= key) & ((at < key + window) | (key < sinks))
                rows = torch.zeros(lq, hq, hd, dtype=torch.bool, device="cuda")
                rows[:, hq - hq // hk:, column] = True                # the heads that share the last key head
                hit[i] = rows & sees[:, None, None]
            out, lse = window_attention(q, k, bad, window, sinks, kv_lens=kv_lens, return_lse=True)
            assert torch.equal(lse, clean_lse)
            assert not bool(torch.isfinite(out[hit]).any())
            _within(torch.where(hit, 0.0, out), torch.where(hit, 0.0, want), bound)
            for i, n in enumerate(lens):
                none = n - lq + torch.arange(lq, device="cuda") < 0
                assert bool((out[i, none] == 0).all())
            again = window_attention(q, k, bad, window, sinks, kv_lens=kv_lens)
            assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    assert torch.equal(clean, window_attention(q, k, v, window, sinks, kv_lens=kv_lens))


@pytest.mark.parametrize("dtype, hd", [(FP, 64), (BF, 128)])
def test_window_attention_infinite_value_of_no_weight_in_the_blocks_edge(dtype, hd):
    """256 queries share a block, two tiles of 128.  Keys that every row of one tile sees and only some of the other are the block's
    edge for both: an infinite value there is added to the rows that see it, never multiplied with a weight that came out as 0,
    whichever tile gets to it first."""
    from dsaquant_b200.window_attention import window_attention

    g = _gen(64)
    b, lq, lk, heads, window = 4, 256, 1000, 24, 300
    q, k, v = _qkv(g, b, lq, lk, heads, heads, hd, dtype)
    at = lk - lq + torch.arange(lq, device="cuda")
    for key in (580, 639, 640, 703, 704, 767, 768, 831):              # 576 .. 703 the first tile sees whole, 704 .. 831 the second
        bad_q, bad_k, bad = q.clone(), k.clone(), v.clone()
        bad_q[..., 0], bad_k[:, key, :, 0], bad[:, key, :, 5] = 16.0, -200.0, float("inf")    # a score of -280 and less: a weight of 0 in fp32
        sees = (at >= key) & (at < key + window)
        first = window_attention(bad_q, bad_k, bad, window)
        assert bool((first[:, sees, :, 5] == float("inf")).all())
        assert bool(torch.isfinite(first[:, ~sees]).all()) and bool(torch.isfinite(first[..., :5]).all()) and bool(torch.isfinite(first[..., 6:]).all())
        for _ in range(5):
            assert torch.equal(first.view(torch.int16), window_attention(bad_q, bad_k, bad, window).view(torch.int16))


def test_window_attention_every_value_not_finite():
    """A whole prompt of NaN is slow at worst: it ends, rows that see nothing are 0, all others NaN."""
    from dsaquant_b200.kernels import vdm_w4a4 as vdm
    from dsaquant_b200.window_attention import window_attention

    g = _gen(62)
    for lq in (4, 100, 1000):
        q, k, v = _qkv(g, 2, lq, 1000, 4, 2, 128, BF)
        lens = torch.tensor([1000, lq // 2], dtype=torch.int32, device="cuda")
        out = window_attention(q, k, torch.full_like(v, float("nan")), 300, 4, kv_lens=lens)
        assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(out[1, lq - lq // 2:]).all())
        assert bool((out[1, :lq - lq // 2] == 0).all())
    assert vdm.last_device_status() == 0


@pytest.mark.parametrize("dtype, hd", [(BF, 128), (FP, 64)])
@pytest.mark.parametrize("lq, lk, window, sinks", [(400, 400, 90, 0), (300, 900, 200, 0), (256, 256, 64, 0), (500, 500, 90, 3), (300, 300, 5000, 0),
                                                   (60, 400, 90, 0), (3, 400, 90, 0)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_window_attention_not_finite_rows_and_keys_without_first_keys(lq, lk, window, sinks, dtype, hd, value):
    """Rows of a block whose windows begin in different key tiles, all with scores that are not finite - one bad key that they
    share, or queries that hold garbage - end, give NaN where the definition does, and leave the other rows as they are."""
    from dsaquant_b200.kernels import vdm_w4a4 as vdm
    from dsaquant_b200.window_attention import window_attention

    g = _gen(63 + lq + window)
    q, k, v = _qkv(g, 2, lq, lk, 2, 1, hd, dtype)
    q[..., 0] = q[..., 0].abs() + 1                                   # an infinite key scores with the sign it has
    lens = torch.tensor([lk, lk - 40], dtype=torch.int32, device="cuda")
    clean, clean_lse = window_attention(q, k, v, window, sinks, kv_lens=lens, return_lse=True)
    at = lens.long()[:, None] - lq + torch.arange(lq, device="cuda")
    for key in (lk - 41, lk - 100, lk - 129, lk - 200, max(lk - lq, 0)):
        bad = k.clone()
        bad[:, key, :, 0] = value
        out, lse = window_attention(q, bad, v, window, sinks, kv_lens=lens, return_lse=True)
        sees = (at >= key) & ((at < key + window) | (key < sinks))
        assert torch.equal(out[~sees], clean[~sees])
        assert torch.equal(lse.transpose(1, 2)[~sees], clean_lse.transpose(1, 2)[~sees])
        if value != float("-inf"):                                    # (a score of -inf is a weight of 0)
            assert bool(torch.isnan(out[sees]).all()) and not bool(torch.isfinite(lse.transpose(1, 2)[sees]).any())
    some = torch.zeros(2, lq, dtype=torch.bool, device="cuda")
    some[:, ::2] = some[:, lq // 2:lq // 2 + 40] = True
    bad = q.clone()
    bad[some] = value                                                 # whole queries: scores of both signs, or NaN
    out, lse = window_attention(bad, k, v, window, sinks, kv_lens=lens, return_lse=True)
    none = at < 0
    assert torch.equal(out[~some], clean[~some]) and bool((out[none] == 0).all())
    assert not bool(torch.isfinite(lse.transpose(1, 2)[some & ~none]).any())
    assert vdm.last_device_status() == 0


@pytest.mark.parametrize("b, lq, lk, hq, hk, hd", [
    (32, 127, 16000, 40, 8, 128), (32, 127, 65536, 40, 8, 128), (1, 127, 65536, 8, 8, 128), (4, 33, 8000, 4, 4, 64), (64, 64, 4000, 16, 1, 128),
    (16, 1, 8192, 40, 8, 128), (1, 1, 500000, 64, 1, 128), (64, 2, 100000, 16, 1, 64)])
def test_window_attention_workspace_stays_small(b, lq, lk, hq, hk, hd):
    """Partial outputs are a small part of the keys and values, or what four blocks an SM hold twice over."""
    from dsaquant_b200 import _lib

    need = _lib.load().b200w4a4_window_attention_workspace_bytes(b, lq, lk, hq, hk, hd, lk, 0)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    few = 2 * 4 * sms * 64 * (hd + 1) * 4
    assert need <= max(few, 4 * b * lk * hk * hd // 16)


def test_window_attention_prompts_need_no_workspace():
    """The wrapper asks for none from PROMPT_QUERIES queries on, and the library wants none from there on."""
    from dsaquant_b200 import _lib
    from dsaquant_b200.window_attention import PROMPT_QUERIES

    need = _lib.load().b200w4a4_window_attention_workspace_bytes
    assert need(1, PROMPT_QUERIES, 100000, 8, 8, 128, 100000, 0) == 0 and need(1, PROMPT_QUERIES - 1, 100000, 8, 8, 128, 100000, 0) > 0


# ------------------------------------------------------------------------------------------------ apply_rotary
def test_apply_rotary_inplace_refuses_shared_memory():
    """q and k that overlap each other, or tokens that overlap, would be rotated twice; out of place they are read only."""
    from dsaquant_b200.rotary import apply_rotary, rotary_table

    g = _gen(71)
    table, pos = rotary_table(64, 32, device="cuda"), torch.arange(5, device="cuda")
    x = _randn(g, 5, 6, 32, dtype=FP)
    sliding = _randn(g, 5 * 16 + 48, dtype=FP).as_strided((5, 2, 32), (16, 32, 1))
    keep = x.clone()
    for q, k in ((x, x), (x[:, :4], x[:, 3:]), (x[:, 2:], x[:, :3]), (x, x[:, 5:]), (sliding, None), (x, sliding)):
        with pytest.raises(ValueError):
            apply_rotary(q, k, table, pos, inplace=True)
        rq, rk = apply_rotary(q, k, table, pos)
        assert torch.equal(rq, apply_rotary(q.clone(), None, table, pos)[0])
        assert k is None or torch.equal(rk, apply_rotary(k.clone(), None, table, pos)[0])
    assert torch.equal(x, keep)
    want = [apply_rotary(part.clone(), None, table, pos)[0] for part in (x[:, 2:], x[:, :2])]
    got = apply_rotary(x[:, 2:], x[:, :2], table, pos, inplace=True)          # k in front of q
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(torch.cat([want[1], want[0]], 1), x)


# ------------------------------------------------------------------------------------------------ linear_w4_group
def test_linear_w4_group_refuses_the_gemms_weights_and_takes_them_regrouped():
    """A vdm_w4a4_packed_v1 weight has the shapes of a grouped one; regrouped it is the same weight, code by code."""
    from dsaquant_b200.kernels import vdm_w4a4 as vdm
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant
    from dsaquant_b200.kernels.w4_group import linear_w4_group, regroup_packed_weight
    from dsaquant_b200.quantization.quant_linear import QuantLinear

    g = _gen(81)
    m, n, k = 9, 256, 1536
    lin = torch.nn.Linear(k, n).half().cuda()
    layer = QuantLinear(lin, {"w": "lsq", "act": "dynamic"}, {"w": {}, "act": {}})
    layer.wquantizer.scale, layer.wquantizer.sym = (lin.weight.abs().amax(1) / 7).float(), True
    layer.prepare_vdm_kernel_weights()
    packed, wscales, channel = vdm.quantize_weight_per_channel(lin.weight)
    x = _randn(g, m, k, dtype=BF)
    codes, scale = rms_norm_quant(x, torch.ones(k, device="cuda"))
    plain = torch.ones(n, k // 64, device="cuda", dtype=FP)
    buffers = (layer.vdm_weight_packed, layer.vdm_weight_scale_packed)
    w_b200, _ = vdm.prepare_b200_weight(*buffers)
    for w, s in ((packed, wscales), (packed, plain), (torch.zeros_like(packed), wscales), buffers, (w_b200, plain)):
        with pytest.raises(ValueError):
            linear_w4_group(x, w, s)
    moved = layer.cpu().cuda()
    with pytest.raises(ValueError):
        linear_w4_group(x, moved.vdm_weight_packed, moved.vdm_weight_scale_packed)

    for qweight, ws, ch in ((packed, wscales, channel), (moved.vdm_weight_packed, moved.vdm_weight_scale_packed, moved.vdm_weight_scale)):
        grouped = regroup_packed_weight(qweight, ch)
        assert grouped[0].shape == (n, k // 2) and grouped[0].is_contiguous() and grouped[1].shape == (n, 1)
        want = vdm.unpack_codes(qweight, n, k, 2)
        assert torch.equal(_codes_of(grouped[0]), want.double())
        y = codes.double() @ want.double().t() * scale.double()[:, None] * ch.double()
        token = linear_w4_group(codes, *grouped, act_scale=scale)
        prompt = vdm.linear_prequantized(codes, scale, qweight, ws)
        # exact integer sums below 2^24 times two scales: two fp32 products (and for the matvec its sum over runs of 128,
        # 12 terms), one rounding to fp16
        size = codes.double().abs() @ want.double().abs().t() * scale.double()[:, None] * ch.double()
        for got in (token, prompt):
            _within(got, y, 2.0 ** -11 * y.abs() + 2.0 ** -25 + 28 * 2.0 ** -24 * size)
    for bad in (lambda: regroup_packed_weight(packed[:100], channel[:100]), lambda: regroup_packed_weight(packed, channel.float()),
                lambda: regroup_packed_weight(packed, channel[:128]), lambda: regroup_packed_weight(packed.to(torch.int8), channel)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), 1e6])
def test_quantize_weight_grouped_marks_groups_that_are_not_finite(dtype, value):
    """A weight that is not finite, or too large for an fp16 scale, shows in the scale and in every product, and leaves the other
    groups as they are."""
    from dsaquant_b200.kernels.w4_group import linear_w4_group, quantize_weight_grouped

    g = _gen(91)
    n, k, group = 40, 512, 64
    w = (_randn(g, n, k) * 0.02).to(dtype)
    packed, scales = quantize_weight_grouped(w, group)
    for row, col in ((0, 0), (17, 130), (39, 511)):
        w[row, col] = value                                          # 1e6 is an infinity in fp16
    got, got_scales = quantize_weight_grouped(w, group)
    hit = torch.zeros(n, k // group, dtype=torch.bool, device="cuda")
    hit[0, 0] = hit[17, 2] = hit[39, 7] = True
    assert bool(torch.isnan(got_scales[hit]).all()) and torch.equal(got_scales[~hit], scales[~hit])
    parts, want = got.view(n, k // group, -1), packed.view(n, k // group, -1)
    assert bool((parts[hit] == 0).all()) and torch.equal(parts[~hit], want[~hit])
    x = _randn(g, 3, k, dtype=BF)
    y, clean = linear_w4_group(x, got, got_scales), linear_w4_group(x, packed, scales)
    rows = hit.any(1)
    assert bool(torch.isnan(y[:, rows]).all()) and torch.equal(y[:, ~rows], clean[:, ~rows])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_weight_grouped_largest_scale(dtype):
    """The largest weight whose scale fp16 holds keeps its value; the next power of two marks the group."""
    from dsaquant_b200.kernels.w4_group import quantize_weight_grouped

    w = torch.zeros(2, 32, device="cuda", dtype=dtype)
    w[0, 3], w[1, 3] = 65504.0 * 7, 65536.0 * 7                      # 458752 = 7 * 2^16; bf16 rounds the first up to it
    packed, scales = quantize_weight_grouped(w, 32)
    assert bool(torch.isnan(scales[1]).all())
    if dtype == F32:
        assert scales[0].item() == 65504.0 and _codes_of(packed)[0, 3].item() == 7


@pytest.mark.parametrize("xdtype, out_dtype", [(BF, BF), (FP, FP), (torch.int8, FP), (torch.int8, BF)])
@pytest.mark.parametrize("bias_dtype", [BF, FP, F32, torch.float64])
def test_linear_w4_group_adds_the_bias_as_it_is(xdtype, out_dtype, bias_dtype):
    """A bias of another type than the output is not rounded to it before the addition."""
    g = _gen(95)
    packed, scales = _w4_case(g, 300, 256, 64)
    bias = (100 + _randn(g, 300)).to(bias_dtype)                     # its rounding to 16 bits would outweigh the sums
    act = None
    x = _randn(g, 5, 256, dtype=BF if xdtype == torch.int8 else xdtype) * 0.1
    if xdtype == torch.int8:
        x, act = (x * 100).round().clamp(-128, 127).to(torch.int8), torch.full((5,), 0.001, device="cuda")
    _check_w4(x, packed, scales, bias, act, out_dtype)
    _check_w4(x, packed, scales, bias.repeat_interleave(2)[::2], act, out_dtype)


def test_sizes_that_32_bits_do_not_hold_are_refused():
    """The foreign calls take 32-bit sizes and cut larger ones off."""
    from dsaquant_b200.kernels.w4_group import linear_w4_group, quantize_weight_grouped
    from dsaquant_b200.rotary import apply_rotary, rotary_table

    def big(dtype, *shape):
        return torch.zeros(1, device="cuda", dtype=dtype).expand(shape)

    k = (1 << 32) + 64
    with pytest.raises(ValueError, match="at most"):
        linear_w4_group(big(BF, 1, k), big(torch.uint8, 1, k // 2), big(FP, 1, k // 64))
    with pytest.raises(ValueError, match="at most"):
        linear_w4_group(big(BF, 1, 64), big(torch.uint8, (1 << 32) + 5, 32), big(FP, (1 << 32) + 5, 1))
    for n, width in ((1, k), ((1 << 32) + 5, 64)):
        with pytest.raises(ValueError, match="at most"):
            quantize_weight_grouped(big(BF, n, width), 64)
    table, pos = rotary_table(4, 2, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    few = torch.zeros(1, 2, 2, device="cuda", dtype=BF)
    many = few[:, :1].expand(1, (1 << 32) + 1, 2)
    for q, kk in ((many, None), (few, many)):
        with pytest.raises(ValueError, match="heads"):
            apply_rotary(q, kk, table, pos)
