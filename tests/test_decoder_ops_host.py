"""CPU-only tests of the decoder-layer operators: header and binding agree, arguments are refused before anything
is launched, tables and packed forms are what their formulas say."""
import math
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
P = 1 << 12  # a 16-byte aligned address that no refused call may touch


@pytest.fixture(scope="module")
def lib():
    from dsaquant_b200 import _lib

    return _lib.load()


def test_header_and_binding_list_the_same_symbols(lib):
    from dsaquant_b200 import _lib

    header = (ROOT / "include" / "b200w4a4_decoder.h").read_text()
    declared = set(re.findall(r"^(?:int|size_t) (b200w4a4_[a-z0-9_]+)\(", header, re.M))
    assert declared == set(_lib.DECODER_SIGNATURES)
    for name in declared:
        assert hasattr(lib, name)


def _rms(lib, **over):
    a = dict(x=P, dt=1, ld=64, r=None, rld=64, w=P, wdt=1, eps=1e-6, codes=P, fmt=0, scale=P, ro=None, m=2, d=64, clip=1.0, s=None)
    a.update(over)
    return lib.b200w4a4_rms_norm_quant(*a.values())


@pytest.mark.parametrize("over, code", [
    (dict(dt=3), -1), (dict(wdt=-1), -1), (dict(fmt=2), -1), (dict(r=P), -1), (dict(ro=P), -1), (dict(clip=0.0), -1),
    (dict(clip=float("nan")), -1), (dict(eps=-1.0), -1), (dict(m=-1), -2), (dict(d=0), -2), (dict(d=16385, ld=16385), -2),
    (dict(x=None), -1), (dict(w=None), -1), (dict(codes=None), -1), (dict(scale=None), -1), (dict(ld=63), -2),
    (dict(r=P, ro=2 * P, rld=10), -2), (dict(r=P, ro=P), -1), (dict(r=2 * P, ro=P), -1), (dict(x=P + 1), -3), (dict(scale=P + 2), -3), (dict(m=0, x=None), 0),
])
def test_rms_norm_quant_refusals(lib, over, code):
    assert _rms(lib, **over) == code


def _w4(lib, **over):
    a = dict(x=P, dt=0, act=None, p=P, s=P, bias=None, out=P, odt=0, m=1, n=16, k=128, g=128, st=None)
    a.update(over)
    return lib.b200w4a4_linear_w4_group(*a.values())


@pytest.mark.parametrize("over, code", [
    (dict(dt=2), -1), (dict(odt=2), -1), (dict(act=P), -1), (dict(dt=3), -1), (dict(m=-1), -2), (dict(n=0), -2),
    (dict(k=100, g=100), -2), (dict(g=48), -2), (dict(g=0), -2), (dict(k=160, g=64), -2), (dict(x=P + 8), -3),
    (dict(p=P + 4), -3), (dict(x=None), -1), (dict(out=None), -1), (dict(m=65535 * 8 + 1), -2), (dict(m=0, x=None), 0),
])
def test_linear_w4_group_refusals(lib, over, code):
    assert _w4(lib, **over) == code


@pytest.mark.parametrize("args, code", [
    ((None, 0, P, P, 4, 64, 32, None), -1), ((P, 5, P, P, 4, 64, 32, None), -1), ((P, 0, P, P, 0, 64, 32, None), -2),
    ((P, 0, P, P, 4, 80, 32, None), -2), ((P, 0, P, P, 4, 64, 16, None), -2), ((P + 1, 0, P, P, 4, 64, 32, None), -3),
])
def test_quantize_weight_grouped_refusals(lib, args, code):
    assert lib.b200w4a4_quantize_weight_grouped(*args) == code


def _rot(lib, **over):
    a = dict(q=P, qt=256, qh=64, qo=P, qot=256, qoh=64, hq=4, k=P, kt=64, kh=64, ko=P, kot=64, koh=64, hk=1, dt=1, cs=P, mp=10,
             pos=P, p64=1, t=3, hd=64, rd=64, il=0, inv=0, st=None)
    a.update(over)
    return lib.b200w4a4_rotary(*a.values())


@pytest.mark.parametrize("over, code", [
    (dict(dt=3), -1), (dict(p64=2), -1), (dict(il=2), -1), (dict(inv=-1), -1), (dict(t=-1), -2), (dict(hq=0), -2),
    (dict(hk=-1), -2), (dict(mp=0), -2), (dict(hd=513), -2), (dict(rd=66), -2), (dict(rd=63), -2), (dict(rd=0), -2),
    (dict(q=None), -1), (dict(k=None), -1), (dict(cs=None), -1), (dict(pos=None), -1), (dict(pos=P + 4), -3),
    (dict(cs=P + 4), -3), (dict(ko=P + 1), -3), (dict(t=0, q=None), 0),
])
def test_rotary_refusals(lib, over, code):
    assert _rot(lib, **over) == code


def _attn(lib, **over):
    a = dict(q=P, qb=256, qt=128, qh=64, k=P, kb=256, kt=64, kh=64, v=P, vb=256, vt=64, vh=64, lens=None, out=P, lse=None, dt=1,
             b=1, lq=1, lk=4, hq=2, hk=1, hd=64, w=4, s=0, scale=0.125, ws=None, wb=0, st=None)
    a.update(over)
    return lib.b200w4a4_window_attention(*a.values())


@pytest.mark.parametrize("over, code", [
    (dict(dt=2), -1), (dict(hd=96), -2), (dict(hq=3, hk=2), -2), (dict(hq=65, hk=1), -2), (dict(hk=0), -2), (dict(b=-1), -2),
    (dict(b=65536), -2), (dict(lq=-1), -2), (dict(lk=-1), -2), (dict(w=0), -1), (dict(s=-1), -1), (dict(scale=0.0), -1),
    (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(out=None), -1),
    (dict(q=P + 8), -3), (dict(kt=68), -3), (dict(ws=P + 4), -3), (dict(lens=P + 2), -3), (dict(b=0, q=None), 0),
    (dict(lq=0, q=None), 0), (dict(lq=1 << 30, hq=64, hk=1), -2),
])
def test_window_attention_refusals(lib, over, code):
    assert _attn(lib, **over) == code


def test_python_wrappers_refuse_cpu_tensors_and_bad_tables(monkeypatch):
    from dsaquant_b200.kernels import vdm_w4a4

    monkeypatch.setattr(vdm_w4a4, "_EXT", None)  # the loaded library is not left behind for tests of its loading
    from dsaquant_b200.kernels.rms_norm import rms_norm_quant
    from dsaquant_b200.kernels.w4_group import linear_w4_group, quantize_weight_grouped
    from dsaquant_b200.rotary import apply_rotary, rotary_table
    from dsaquant_b200.window_attention import window_attention

    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        rms_norm_quant(x, torch.ones(64))
    with pytest.raises(RuntimeError):
        quantize_weight_grouped(x, 32)
    with pytest.raises(RuntimeError):
        linear_w4_group(x, torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.float16))
    with pytest.raises(RuntimeError):
        apply_rotary(x.view(2, 1, 64), None, rotary_table(4, 64), torch.arange(2))
    with pytest.raises(RuntimeError):
        window_attention(x.view(1, 2, 1, 64), x.view(1, 2, 1, 64), x.view(1, 2, 1, 64), 4)
    for bad in (dict(max_positions=0, rotary_dim=64), dict(max_positions=4, rotary_dim=63), dict(max_positions=4, rotary_dim=64, scaling="x"),
                dict(max_positions=4, rotary_dim=64, factor=0.5), dict(max_positions=4, rotary_dim=2, scaling="ntk")):
        with pytest.raises(ValueError):
            rotary_table(**bad)


def test_rotary_tables_follow_their_formulas():
    from dsaquant_b200.rotary import rotary_table

    rd, far = 64, 70000
    plain = rotary_table(far, rd, 10000.0)
    assert plain.shape == (far, rd // 2, 2) and plain.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (69999, 0), (69999, 31), (12345, 7)):
        angle = p * 10000.0 ** (-2 * i / rd)
        # one rounding to fp32 (half an eps) of a 64-bit cosine whose angle is exact to 2^-53 of itself
        for got, want in zip(plain[p, i].tolist(), (math.cos(angle), math.sin(angle))):
            assert abs(got - want) <= 2.0 ** -24 * max(abs(want), 1e-30) + far * 2.0 ** -50
    linear = rotary_table(1000, rd, scaling="linear", factor=4.0)
    assert torch.equal(linear[::4], plain[:250])
    ntk = rotary_table(1000, rd, scaling="ntk", factor=4.0)
    assert torch.equal(ntk[:, 0], plain[:1000, 0])                       # the fastest pair stays
    slow = 10000.0 ** (-2 * 31 / rd) / 4.0                               # the slowest is stretched by the factor
    assert abs(ntk[999, 31, 1].item() - math.sin(999 * slow)) < 1e-6
    yarn = rotary_table(1000, rd, scaling="yarn", factor=4.0, trained_positions=4096)
    amp = 0.1 * math.log(4.0) + 1
    assert torch.allclose(yarn[:, 0], plain[:1000, 0] * amp, rtol=3e-7, atol=1e-7)
    assert abs(yarn[999, 31, 1].item() - amp * math.sin(999 * slow)) < 1e-6
    assert abs(rotary_table(4, rd, scaling="yarn", factor=1.0) - rotary_table(4, rd)).max().item() == 0.0


def test_workspace_query_of_bad_or_empty_shapes_is_zero(lib):
    assert lib.b200w4a4_window_attention_workspace_bytes(0, 1, 4, 2, 1, 64, 4, 0) == 0
    assert lib.b200w4a4_window_attention_workspace_bytes(1, 1, 4, 3, 2, 64, 4, 0) == 0


def test_shared_memory_of_q_and_k_is_found():
    """`_distinct` and `_disjoint` against the addresses themselves: never true where two values share one, and true for the
    views that a fused projection or a head-major cache gives."""
    import random

    from dsaquant_b200.rotary import _disjoint, _distinct

    def addresses(x):
        at = torch.arange(int(x.untyped_storage().nbytes()) // x.element_size())
        return at.as_strided(x.shape, x.stride(), x.storage_offset()).flatten().tolist()

    rng = random.Random(5)
    flat = torch.zeros(4096)
    said = [0, 0]
    for _ in range(4000):
        def some():
            shape = [rng.choice([1, 2, 3]), rng.choice([1, 2, 3]), rng.choice([1, 2, 4])]
            return shape, [rng.choice([0, 1, 2, 4, 8, 12, 16, 24]), rng.choice([0, 1, 4, 8, 12, 16]), 1], rng.randrange(40)
        (n1, s1, o1), (n2, s2, o2) = some(), some()
        if rng.random() < 0.6:
            s2, n2 = s1, [n1[0], n2[1], n1[2]]
        q, k = flat.as_strided(n1, s1, o1), flat.as_strided(n2, s2, o2)
        a, b = addresses(q), addresses(k)
        if _distinct(q):
            assert len(set(a)) == len(a)
        if _distinct(q) and _distinct(k):
            said[_disjoint(q, k)] += 1
            if _disjoint(q, k):
                assert not set(a) & set(b) and _disjoint(k, q)
    assert min(said) > 200
    t, hq, hk, hd = 5, 6, 2, 8
    for views in (lambda x: (x[:, :hq], x[:, hq:hq + hk]), lambda x: (x[:, hk:hk + hq], x[:, :hk])):
        by_token = torch.zeros(t, hq + 2 * hk, hd)
        by_head = torch.zeros(hq + 2 * hk, t, hd).transpose(0, 1)
        for q, k in (views(by_token), views(by_head), views(by_token[2:3]), views(by_head[2:3])):
            assert _distinct(q) and _distinct(k) and _disjoint(q, k)
    each = torch.zeros(t, hq, 3, hd)                       # q, k and v of a head side by side
    assert _disjoint(each[:, :, 0], each[:, :, 1]) and _disjoint(each[:, :, 2], each[:, :, 0])
    assert not _disjoint(each[:, :, 0], each[:, :, 0]) and not _disjoint(by_token[:, :3], by_token[:, 2:4])
    assert _disjoint(torch.zeros(t, hq, hd), torch.zeros(t, hk, hd))


def test_weights_in_the_gemms_order_are_known_as_such(tmp_path):
    """The buffers of a layer read from a packed checkpoint carry their layout through moves, copies and fused projections;
    a saved state does not."""
    import copy

    from dsaquant_b200.attention_qkv import _cat_cached
    from dsaquant_b200.checkpoints import packed_checkpoint as pc
    from dsaquant_b200.kernels.vdm_w4a4 import in_gemm_layout
    from dsaquant_b200.quantization.quant_linear import QuantLinear

    def loaded():
        layer = QuantLinear(torch.nn.Linear(128, 128), {"w": "lsq", "act": "dynamic"}, {"w": {}, "act": {}})
        pc._switch_layer_to_packed(layer, {"vdm_weight_packed": torch.zeros(128, 64, dtype=torch.uint8),
                                           "vdm_weight_scale_packed": torch.ones(128, 2).half(), "vdm_weight_scale": torch.ones(128).half()})
        layer._bias_half = None
        return layer

    def known(layer):
        return in_gemm_layout(layer.vdm_weight_packed) and in_gemm_layout(layer.vdm_weight_scale_packed)

    layer = loaded()
    assert known(layer) and known(copy.deepcopy(layer)) and known(layer._apply(lambda t: t.clone()))
    assert not in_gemm_layout(layer.vdm_weight_scale) and in_gemm_layout(layer.vdm_weight_packed[:64])
    torch.save(layer.state_dict(), tmp_path / "layer.pt")
    state = torch.load(tmp_path / "layer.pt", weights_only=True)
    assert set(state) == {"bias", *pc.VDM_BUFFER_SUFFIXES} and not any(in_gemm_layout(t) for t in state.values())
    attn, layers = torch.nn.Module(), [loaded() for _ in range(3)]
    _cat_cached(attn, "_vdm_qkv", layers)
    assert in_gemm_layout(attn._vdm_qkv_weight_packed) and all(known(x) for x in layers)


@pytest.mark.parametrize("over, code", [(dict(odt=16, bias=P + 2), -3), (dict(odt=18), -1), (dict(odt=17, m=0), 0), (dict(odt=32), -1)])
def test_linear_w4_group_fp32_bias_refusals(lib, over, code):
    assert _w4(lib, **over) == code


@pytest.mark.parametrize("trained, base, rd", [(4, 10000.0, 64), (6, 10000.0, 64), (1, 10000.0, 32), (4096, 2.0, 16), (1 << 20, 1.5, 8), (4096, 10000.0, 128),
                                               (131072, 500000.0, 128)])
def test_yarn_tables_keep_fast_pairs_and_stretch_slow_ones(trained, base, rd):
    """Every pair against the two sentences of the definition, where the trained length or the base leaves no room for a ramp too;
    between them, the angles lie between the two."""
    from dsaquant_b200.rotary import rotary_table

    factor, positions = 8.0, 50
    table = rotary_table(positions, rd, base, scaling="yarn", factor=factor, trained_positions=trained).double() / (0.1 * math.log(factor) + 1)
    p = torch.arange(positions, dtype=torch.float64)
    for i in range(rd // 2):
        f = base ** (-2 * i / rd)
        turns = trained * f / (2 * math.pi)
        # two roundings to fp32, of the table and of what it was divided by
        same = lambda a: bool(((table[:, i, 0] - (p * a).cos()).abs() < 2.0 ** -22).all() and ((table[:, i, 1] - (p * a).sin()).abs() < 2.0 ** -22).all())  # noqa: E731
        if turns > 32:
            assert same(f)
        elif turns < 1:
            assert same(f / factor)
        else:
            angle = math.atan2(table[1, i, 1], table[1, i, 0])
            assert f / factor - 1e-6 <= angle <= f + 1e-6


def test_yarn_ramp_is_linear_in_the_pair():
    """The usual sizes: between the pair that turns 32 times over the trained length and the one that turns once."""
    from dsaquant_b200.rotary import rotary_table

    rd, base, factor, trained = 128, 10000.0, 8.0, 4096
    table = rotary_table(2, rd, base, scaling="yarn", factor=factor, trained_positions=trained).double()
    low = math.floor(rd * math.log(trained / (32 * 2 * math.pi)) / (2 * math.log(base)))
    high = math.ceil(rd * math.log(trained / (2 * math.pi)) / (2 * math.log(base)))
    assert (low, high) == (20, 46)
    for i in range(rd // 2):
        f, ramp = base ** (-2 * i / rd), min(max((i - low) / (high - low), 0.0), 1.0)
        want = f * (1 - ramp) + f / factor * ramp
        assert abs(math.atan2(table[1, i, 1], table[1, i, 0]) - want) < 2.0 ** -22


@pytest.mark.parametrize("over, code", [(dict(n=(1 << 31) - 1), -2), (dict(n=(1 << 31) - 511), -2), (dict(k=(1 << 20) + 128), -2)])
def test_linear_w4_group_refuses_sizes_past_its_row_numbers(lib, over, code):
    """A last block of rows past 2^31 would wrap."""
    assert _w4(lib, **over) == code
    assert lib.b200w4a4_quantize_weight_grouped(P, 0, P, P, 4, (1 << 20) + 32, 32, None) == -2
