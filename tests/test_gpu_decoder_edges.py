"""Decoder-layer operators where they can go wrong without a wrong formula: values beside a rounding border, values that are
not finite, memory that is shared, sizes that ask for much workspace.  Helpers and tolerances are those of
test_gpu_decoder_ops."""
import pytest
import torch

from test_gpu_decoder_ops import BF, F32, FP, _gen, _randn

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
