"""Decoder-layer operators: refusals (no GPU needed, nothing is launched) and the 64-bit forms they are tested against."""
import ctypes as C

import numpy as np
import pytest

from layer_util import BF16, F16, F32, Paged, fp8_values, from_bits, to_bits
from oracle import layer as ol

INVALID, ALIGNMENT, WORKSPACE = -1, -2, -3
BUF = C.create_string_buffer(1 << 16)
P = (C.addressof(BUF) + 63) // 64 * 64  # never dereferenced: every call below is refused on the host


def norm(lib, **kw):
    a = dict(rows=2, cols=64, type=BF16, x=P, x_stride=64, residual=P, residual_out=P, weight=P, eps=1e-5, format=0, group=32, q=P, scales=P) | kw
    return lib.tb200_rmsnorm_quant(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=0), dict(type=3), dict(type=-1), dict(x_stride=63), dict(format=3), dict(format=-1), dict(group=16),
                                dict(group=-32), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None), dict(weight=None), dict(q=None), dict(scales=None)])
def test_norm_refuses(lib, kw):
    assert norm(lib, **kw) == INVALID


def test_norm_alignment_and_nothing_to_do(lib):
    for name, at in (("x", 1), ("residual", 1), ("residual_out", 3), ("weight", 2), ("scales", 2)):
        assert norm(lib, **{name: P + at}) == ALIGNMENT
    assert norm(lib, x=P + 2, type=F32) == ALIGNMENT
    assert norm(lib, rows=0, x=None, q=None) == 0


def plan(lib, **kw):
    a = dict(requests=2, page_size=16, max_pages=4, max_tokens=8, num_free=3, cached=P, new=P, free=P, table=P, cu=P, kv=P, positions=P, slots=P, counts=P) | kw
    return lib.tb200_paged_plan(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(requests=-1), dict(requests=16385), dict(page_size=0), dict(max_pages=-1), dict(max_tokens=-1), dict(max_tokens=(1 << 30) + 1),
                                dict(num_free=-1), dict(page_size=1 << 20, max_pages=1 << 11), dict(cached=None), dict(new=None), dict(free=None), dict(table=None),
                                dict(cu=None), dict(kv=None), dict(positions=None), dict(slots=None), dict(counts=None)])
def test_plan_refuses(lib, kw):
    assert plan(lib, **kw) == INVALID


def test_plan_alignment(lib):
    for name in ("cached", "new", "free", "table", "cu", "kv", "positions", "counts"):
        assert plan(lib, **{name: P + 2}) == ALIGNMENT
    assert plan(lib, slots=P + 4) == ALIGNMENT


def append(lib, **kw):
    a = dict(tokens=3, q_heads=4, kv_heads=2, head_dim=64, in_type=F32, q=P, k=P, v=P, q_stride=256, k_stride=128, v_stride=128, cos=P, sin=P, table_rows=10, rot_dim=64,
             interleaved=0, positions=P, cache_type=BF16, q_out=P, page_size=16, num_pages=4, slots=P, k_cache=P, v_cache=P) | kw
    return lib.tb200_rope_append(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(q_heads=-1), dict(kv_heads=0), dict(head_dim=0), dict(in_type=5), dict(cache_type=F32), dict(rot_dim=3), dict(rot_dim=66),
                                dict(rot_dim=-2), dict(table_rows=-1), dict(page_size=0), dict(num_pages=-1), dict(q_stride=255), dict(k_stride=127), dict(v_stride=0),
                                dict(q=None), dict(k=None), dict(v=None), dict(cos=None), dict(sin=None), dict(positions=None), dict(q_out=None), dict(slots=None),
                                dict(k_cache=None), dict(v_cache=None), dict(head_dim=65536, q_heads=65536, q_stride=1 << 40)])
def test_append_refuses(lib, kw):
    assert append(lib, **kw) == INVALID


def test_append_alignment_and_nothing_to_do(lib):
    for name, at in (("q", 2), ("k", 2), ("v", 1), ("q_out", 1), ("k_cache", 1), ("v_cache", 1), ("cos", 2), ("sin", 2), ("positions", 2), ("slots", 4)):
        assert append(lib, **{name: P + at}) == ALIGNMENT
    assert append(lib, tokens=0, q=None, k=None) == 0


def attention(lib, **kw):
    a = dict(tokens=3, requests=2, max_new=0, q_heads=4, kv_heads=2, head_dim=64, type=F16, q=P, q_stride=256, cu=P, kv=P, table=P, max_pages=4, page_size=16, num_pages=5,
             k=P, v=P, scale=0.125, window=0, out=P, out_stride=256, ws=P, ws_bytes=1 << 40) | kw
    return lib.tb200_paged_attention(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(requests=-1), dict(max_new=-1), dict(q_heads=3), dict(kv_heads=0), dict(q_heads=1), dict(head_dim=0), dict(head_dim=60),
                                dict(head_dim=264, q_stride=2000, out_stride=2000), dict(type=F32), dict(type=7), dict(q_stride=255), dict(out_stride=255), dict(max_pages=-1),
                                dict(page_size=0), dict(page_size=1 << 20, max_pages=1 << 11), dict(num_pages=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(window=-1), dict(q=None), dict(cu=None), dict(kv=None), dict(table=None), dict(k=None), dict(v=None), dict(out=None)])
def test_attention_refuses(lib, kw):
    assert attention(lib, **kw) == INVALID


def test_attention_workspace_alignment_and_nothing_to_do(lib):
    need = lib.tb200_paged_attention_workspace_bytes(3, 2, 4, 2, 64)
    assert need > 0
    assert attention(lib, ws=None) == WORKSPACE and attention(lib, ws_bytes=need - 1) == WORKSPACE
    for name, at in (("q", 1), ("out", 4), ("k", 4), ("v", 2), ("cu", 2), ("kv", 1), ("table", 2), ("ws", 8)):
        assert attention(lib, **{name: P + at}) == ALIGNMENT
    assert attention(lib, tokens=0, q=None, ws=None) == 0 and attention(lib, requests=0, ws=None) == 0
    for bad in ((-1, 2, 4, 2, 64), (3, -1, 4, 2, 64), (3, 2, 5, 2, 64), (3, 2, 4, 0, 64), (3, 2, 4, 2, 300), (3, 2, 4, 2, 12)):
        assert lib.tb200_paged_attention_workspace_bytes(*bad) == 0


# ---- the 64-bit forms ---------------------------------------------------------------------------------------------------
def test_fp8_rounding_of_the_oracle_meets_every_value_and_every_tie():
    for fmt, mantissa in (("e4m3", 3), ("e5m2", 2)):
        v = fp8_values(np.arange(128, dtype=np.uint8), fmt)
        v = v[np.isfinite(v)]
        assert v.max() == ol.TOP[fmt] and np.array_equal(ol.round_fp8(v, fmt), v) and np.array_equal(ol.round_fp8(-v, fmt), -v)
        mid = (v[1:] + v[:-1]) / 2
        even = np.where(np.arange(len(mid)) % 2 == 0, v[:-1], v[1:])  # codes are in order: an even code is the tie's side
        assert np.array_equal(ol.round_fp8(mid, fmt), even)
        assert ol.round_fp8(1e9, fmt) == ol.TOP[fmt]


def test_plan_of_the_oracle_by_hand():
    table = np.array([[9, 9, -1], [7, -1, -1]])
    t, cu, kv, pos, slots, counts = ol.paged_plan([5, 3], [4, 2], 4, 3, 7, [20, 21, 22], table)
    assert t.tolist() == [[9, 9, 20], [7, 21, -1]] and cu.tolist() == [0, 4, 6] and kv.tolist() == [9, 5]
    assert pos.tolist() == [5, 6, 7, 8, 3, 4, -1] and slots.tolist() == [37, 38, 39, 80, 31, 84, -1] and counts.tolist() == [6, 6, 2, 2]


def test_attention_of_the_oracle_ignores_bad_pages_and_masked_places():
    rng = np.random.default_rng(0)
    p = Paged(rng, [20, 5], [3, 2], 4, 2, 16, 4, F16, pad=2, garbage=np.nan)
    want, _ = p.expected()
    assert np.isfinite(want).all()
    # the same by one dense softmax
    k = np.concatenate([from_bits(p.k_bits, F16)[e, 1] for e in p.table[0, :6]])[:23]
    v = np.concatenate([from_bits(p.v_bits, F16)[e, 1] for e in p.table[0, :6]])[:23]
    s = k[:22] @ from_bits(p.q_bits, F16)[1, 3] * p.scale
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(want[1, 3], w @ v[:22], rtol=1e-12)
    assert np.array_equal(want[5:], from_bits(p.out_bits, F16)[5:])
    p.table[0, 2], p.table[1, :] = p.k_bits.shape[0], -1  # keys 8 .. 11 of request 0, all of request 1
    want, _ = p.expected()
    s = np.delete(k, np.s_[8:12], 0)[:18] @ from_bits(p.q_bits, F16)[1, 3] * p.scale
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(want[1, 3], w @ np.delete(v, np.s_[8:12], 0)[:18], rtol=1e-12) and np.all(want[3:5] == 0)


def test_rope_of_the_oracle_turns_pairs():
    cos, sin = np.array([[1.0], [0.0]], np.float32), np.array([[0.0], [1.0]], np.float32)
    x = np.arange(8.0).reshape(2, 1, 4)
    assert ol.rope(x, cos, sin, np.array([0, 1]), True)[:, 0].tolist() == [[0, 1, 2, 3], [-5, 4, 6, 7]]
    y = ol.rope(x, np.repeat(cos, 2, 1), np.repeat(sin, 2, 1), np.array([0, 1]), False)
    assert y[1, 0].tolist() == [-6, -7, 4, 5]


def test_bf16_patterns_round_to_even():
    assert to_bits(np.float32(1 + 2.0 ** -8), BF16) == 0x3F80 and to_bits(np.float32(1 + 3 * 2.0 ** -8), BF16) == 0x3F82
    assert np.isnan(from_bits(to_bits(np.array([np.nan], np.float32), BF16), BF16))[0]


# ---- task factories -----------------------------------------------------------------------------------------------------
def test_layer_factories_build_descriptors():
    from tornadovm_b200.arrays import BFloat16Array, ByteArray, FloatArray, HalfFloatArray, Int8Array, IntArray, LongArray
    from tornadovm_b200.b200 import B200
    from tornadovm_b200.descriptor import Access
    x, w, q, s = BFloat16Array(6 * 40), FloatArray(40), Int8Array(240), FloatArray(12)
    d = B200.addRmsnormQuant(6, 40, x, BFloat16Array(240), w, 1e-5, "int8", 32, q, s)
    assert d.getFunctionName() == "addRmsnormQuant" and d.getParameters()[2] == 2
    assert [i for i, a in enumerate(d.getAccess()) if a is not Access.READ_ONLY] == [4, 9, 10] and d.getAccess()[4] is Access.READ_WRITE
    d = B200.rmsnormQuant(6, 40, FloatArray(240), w, 0.0, "e4m3", 0, ByteArray(240), FloatArray(6))
    assert d.getParameters()[2] == 0 and d.getParameters()[6:8] == [1, 0]
    i = lambda n: IntArray(n)  # noqa: E731
    d = B200.pagedPlan(3, 16, 4, 20, i(3), i(3), i(7), i(12), i(4), i(3), i(20), LongArray(20), i(4))
    assert d.getParameters()[:5] == [3, 16, 4, 20, 7] and d.getAccess()[8] is Access.READ_WRITE and d.getAccess()[12] is Access.WRITE_ONLY
    k = HalfFloatArray(5 * 2 * 16 * 64)
    d = B200.ropeAppend(4, 8, 2, 64, FloatArray(4 * 12 * 64), FloatArray(100 * 32), FloatArray(100 * 32), 64, True, i(4), LongArray(4), 16, HalfFloatArray(4 * 512), k, k)
    assert d.getParameters()[8:11] == [100, 64, 1] and d.getParameters()[15] == 5
    d = B200.pagedAttention(4, 3, 2, 8, 2, 64, HalfFloatArray(2048), i(4), i(3), i(12), 16, k, k, 0.125, 0, HalfFloatArray(2048))
    assert d.getParameters()[11:14] == [4, 16, 5] and d.getAccess()[18] is Access.READ_WRITE


def test_layer_factories_refuse_early():
    from tornadovm_b200.arrays import BFloat16Array, FloatArray, HalfFloatArray, Int8Array, IntArray, LongArray
    from tornadovm_b200.b200 import B200
    f, h, i8, i, lo = FloatArray, HalfFloatArray, Int8Array, IntArray, LongArray
    norm = lambda **k: B200.rmsnormQuant(**(dict(rows=2, cols=64, x=f(128), weight=f(64), eps=1e-5, fmt="int8", group=32, q=i8(128), scales=f(4)) | k))  # noqa: E731
    norm()
    for k, text in ((dict(fmt="int4"), "formats"), (dict(group=16), "groups"), (dict(eps=-1.0), "eps"), (dict(scales=f(3)), "too small"), (dict(x=i8(128)), "take")):
        with pytest.raises(RuntimeError, match=text):
            norm(**k)
    with pytest.raises(RuntimeError, match="differ in type"):
        B200.addRmsnormQuant(2, 64, f(128), h(128), f(64), 1e-5, "int8", 32, i8(128), f(4))
    with pytest.raises(RuntimeError, match="requests"):
        B200.pagedPlan(16385, 16, 1, 1, i(1), i(1), i(1), i(1), i(1), i(1), i(1), lo(1), i(4))
    with pytest.raises(RuntimeError, match="too small"):
        B200.pagedPlan(2, 16, 1, 1, i(2), i(2), i(1), i(2), i(2), i(2), i(1), lo(1), i(4))
    k = h(2 * 16 * 64)
    rope = lambda **a: B200.ropeAppend(**(dict(tokens=1, qHeads=2, kvHeads=2, headDim=64, qkv=f(384), cosTable=f(64), sinTable=f(64), rotDim=64, interleaved=False,  # noqa: E731
                                               positions=i(1), slots=lo(1), pageSize=16, q=h(128), kCache=k, vCache=k) | a))
    rope()
    for a, text in ((dict(rotDim=63), "rotDim"), (dict(kCache=h(100), vCache=h(100)), "whole pages"), (dict(kCache=f(2048), vCache=f(2048)), "take"),
                    (dict(q=BFloat16Array(128)), "differ in type"), (dict(qkv=f(383)), "too small")):
        with pytest.raises(RuntimeError, match=text):
            rope(**a)
    att = lambda **a: B200.pagedAttention(**(dict(tokens=1, requests=1, maxNew=0, qHeads=4, kvHeads=2, headDim=64, q=h(256), cuNew=i(2), kvLens=i(1), blockTable=i(1),  # noqa: E731
                                                  pageSize=16, kCache=k, vCache=k, scale=0.1, window=0, out=h(256)) | a))
    att()
    for a, text in ((dict(qHeads=3), "multiple of kvHeads"), (dict(scale=0.0), "scale"), (dict(requests=0), "requests"), (dict(out=h(255)), "too small"),
                    (dict(q=BFloat16Array(256)), "differ in type"), (dict(window=-1), "window")):
        with pytest.raises(RuntimeError, match=text):
            att(**a)
