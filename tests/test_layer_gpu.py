"""Decoder-layer operators on the GPU against their 64-bit forms (oracle/layer.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

from harness import DevBuf, stream_ptr, sync_and_check
from layer_util import BF16, F16, F32, FORMATS, HALF_STEP, HALF_TINY, Paged, fp8_values, from_bits, to_bits
from oracle import layer as ol

pytestmark = pytest.mark.gpu


def ok(lib, st):
    assert st == 0, lib.tb200_status_string(st)


# ---- norm -----------------------------------------------------------------------------------------------------------
def run_norm(lib, x, residual, weight, kind, fmt, group, eps=1e-5, header=16, x_pad=0, place="own"):
    """place: residual_out is an array of its own, the residual, x, or left out."""
    rows, cols = x.shape
    groups = -(-cols // group) if group else 1
    xb = np.zeros((rows, cols + x_pad), to_bits(x, kind).dtype)
    xb[:, :cols] = to_bits(x, kind)
    dx, dw = DevBuf(xb, header), DevBuf(weight.astype(np.float32), header)
    dr = DevBuf(to_bits(residual, kind), header) if residual is not None else None
    dro = {"own": DevBuf(np.zeros((rows, cols), xb.dtype), header), "residual": dr, "x": dx, "none": None}[place]
    dq, ds = DevBuf(np.full((rows, cols), 0x55, np.uint8), header), DevBuf(np.full((rows, groups), np.nan, np.float32), header)
    ok(lib, lib.tb200_rmsnorm_quant(rows, cols, kind, dx.ptr, cols + x_pad, dr.ptr if dr else None, dro.ptr if dro else None, dw.ptr, eps, FORMATS[fmt],
                                    group, dq.ptr, ds.ptr, stream_ptr()))
    sync_and_check(lib)
    for b in (dx, dw, dr, dro, dq, ds):
        assert b is None or b.guard_intact()
    return dq.numpy(), ds.numpy(), dro.numpy()[:, :cols] if dro else None


def check_norm(x, residual, weight, kind, fmt, group, got, eps=1e-5):
    q, scales, stored = got
    rx, rr = from_bits(to_bits(x, kind), kind), None if residual is None else from_bits(to_bits(residual, kind), kind)
    ratio, want, h = ol.rmsnorm_quant(rx, rr, weight.astype(np.float32), eps, fmt, group)
    cols = x.shape[1]
    # fp32: the sum h (half a step), a sum of `cols` squares (its error halves under the root), the root, two products
    # and the two divisions of the scale
    rel = (0.5 * cols + 10) * 2.0 ** -24
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(scales), np.isnan(want)) and np.array_equal(np.isinf(scales), np.isinf(want))
    assert np.all(np.abs(scales[fin] - want[fin]) <= rel * want[fin] + 2.0 ** -149)
    val = q.view(np.int8).astype(np.float64) if fmt == "int8" else fp8_values(q, fmt)
    off = np.abs(val - ratio)
    moved = np.abs(ratio) * (2 * rel + 2.0 ** -23)
    if fmt == "int8":
        bound = 0.5 + moved + 2.0 ** -17  # the sum with 1/2 is rounded too: half a step at 127
    else:
        m, low = (3, -9) if fmt == "e4m3" else (2, -16)
        _, e = np.frexp(np.maximum(np.abs(ratio) + moved, 1e-300))
        bound = 0.5 * np.exp2(np.maximum(e - 1 - m, low).astype(np.float64)) + moved
    assert np.all(off <= bound), (off - bound).max()
    if stored is not None:
        s = from_bits(stored, kind)
        f = np.isfinite(h)
        assert np.all(np.abs(s[f] - h[f]) <= (HALF_STEP[kind] + 2.0 ** -24) * np.abs(h[f]) + HALF_TINY[kind])


NORM_SHAPES = [(1, 4096), (3, 8), (2, 1), (7, 33), (130, 256), (5, 1032), (2, 8200), (3, 14336), (2, 16400), (2, 32776), (1, 40001)]


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("fmt,group", [("int8", 32), ("int8", 0), ("e4m3", 128), ("e4m3", 0), ("e5m2", 64)])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm_against_64_bits(lib, rows, cols, kind, fmt, group):
    rng = np.random.default_rng(rows * 100003 + cols)
    x, r, w = rng.standard_normal((rows, cols)), 4 * rng.standard_normal((rows, cols)), 1 + 0.3 * rng.standard_normal(cols)
    check_norm(x, r, w, kind, fmt, group, run_norm(lib, x, r, w, kind, fmt, group))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("header", [16, 24])
@pytest.mark.parametrize("cols,x_pad", [(512, 0), (512, 8), (512, 3), (36, 4), (16640, 8), (33008, 0)])
@pytest.mark.parametrize("place", ["own", "residual", "none"])
def test_norm_places_strides_and_headers(lib, cols, x_pad, header, kind, place):
    rng = np.random.default_rng(cols + x_pad)
    x, r, w = rng.standard_normal((5, cols)), rng.standard_normal((5, cols)), rng.standard_normal(cols)
    check_norm(x, r, w, kind, "int8", 32, run_norm(lib, x, r, w, kind, "int8", 32, header=header, x_pad=x_pad, place=place))


@pytest.mark.parametrize("cols", [640, 40000])
def test_norm_without_residual_and_in_place_of_x(lib, cols):
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((4, cols)), rng.standard_normal(cols)
    check_norm(x, None, w, F16, "e4m3", 0, run_norm(lib, x, None, w, F16, "e4m3", 0, place="none"))
    r = rng.standard_normal((4, cols))
    check_norm(x, r, w, F16, "e4m3", 0, run_norm(lib, x, r, w, F16, "e4m3", 0, place="x"))


@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "e5m2"])
def test_norm_zeros_tiny_huge_and_not_finite(lib, fmt, group):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((6, 96)).astype(np.float32)
    x[0] = 0                       # with eps > 0: zeros, scale 1
    x[1] *= np.float32(1e-22)      # far below eps: y near 1e-19
    x[2] *= np.float32(1e17)
    x[3, 40] = np.inf
    x[4, 70] = np.nan
    w = np.ones(96)
    w[5] = 0
    got = run_norm(lib, x, None, w, F32, fmt, group)
    check_norm(x, None, w, F32, fmt, group, got)
    assert np.all(got[0][0] == 0) and np.all(got[1][0] == 1)
    # an infinite norm: every finite value over it is 0 (of either sign), the infinity over it a NaN; a NaN's norm makes all of them NaN
    assert np.all(got[0][3:5] & 0x7F == 0) and np.isnan(got[1][3, 40 // group if group else 0]) and np.isnan(got[1][4]).all()
    # a weight that is not finite spoils its own group alone
    w[40] = np.nan
    q, s, _ = run_norm(lib, x[5:], None, w, F32, fmt, 32)
    assert np.isnan(s[0, 1]) and np.isfinite(s[0, [0, 2]]).all() and np.all(q[0, 32:64] == 0) and q[0, :32].any()


def test_norm_subnormal_scale_stays_invertible(lib):
    x = np.full((1, 64), 3e-39, np.float32)
    x[0, 3] = 0
    q, s, _ = run_norm(lib, x, None, np.full(64, 1e-2), F32, "int8", 32, eps=1.0)
    assert np.all(s == np.float32(2.0 ** -126)) and np.all(q.view(np.int8) == 0)


def test_norm_matches_the_mat_vec_quantiser_bit_for_bit(lib):
    """Groups of 32 in int8 follow the rule of tb200_quantize_x: on values that the norm leaves as they are (mean square
    1, weight 1, eps 0) both give the same bytes."""
    rng = np.random.default_rng(3)
    x = rng.choice([-1.0, 1.0], (2, 256)).astype(np.float32)  # mean square exactly 1
    w = rng.standard_normal(256).astype(np.float32)
    q, s, _ = run_norm(lib, x, None, w, F32, "int8", 32, eps=0.0)
    dy = DevBuf((x * w).astype(np.float32))
    n = lib.tb200_qx_workspace_bytes(256, 2)
    ws = DevBuf(np.zeros(n, np.uint8))
    ok(lib, lib.tb200_quantize_x(256, 2, dy.ptr, ws.ptr, n, stream_ptr()))
    sync_and_check(lib)
    raw = ws.numpy()
    assert np.array_equal(raw[:512].reshape(2, 256), q)
    assert np.array_equal(raw[512:].view(np.float32).reshape(2, 8), s)


# ---- plan -----------------------------------------------------------------------------------------------------------
def run_plan(lib, cached, new, page, width, rows, free, table, header=16):
    n = len(cached)
    d = {k: DevBuf(v, header) for k, v in dict(
        cached=np.array(cached, np.int32), new=np.array(new, np.int32), free=np.array(free, np.int32), table=np.array(table, np.int32),
        cu=np.full(n + 1, -7, np.int32), kv=np.full(n, -7, np.int32), positions=np.full(rows, -7, np.int32), slots=np.full(rows, -7, np.int64),
        counts=np.full(4, -7, np.int32)).items()}
    ok(lib, lib.tb200_paged_plan(n, page, width, rows, len(free), d["cached"].ptr, d["new"].ptr, d["free"].ptr, d["table"].ptr, d["cu"].ptr, d["kv"].ptr,
                                 d["positions"].ptr, d["slots"].ptr, d["counts"].ptr, stream_ptr()))
    sync_and_check(lib)
    assert all(b.guard_intact() for b in d.values())
    return [d[k].numpy() for k in ("table", "cu", "kv", "positions", "slots", "counts")]


def check_plan(lib, cached, new, page, width, rows, free, rng, header=16):
    table = rng.integers(0, 1000, (len(cached), width)).astype(np.int32)
    got = run_plan(lib, cached, new, page, width, rows, free, table, header)
    want = ol.paged_plan(cached, new, page, width, rows, free, table)
    for g, w, name in zip(got, want, ("table", "cu", "kv", "positions", "slots", "counts")):
        assert np.array_equal(g, w), name
    return got


@pytest.mark.parametrize("requests", [1, 2, 33, 300, 1025, 5000])
@pytest.mark.parametrize("page,longest", [(16, 1), (1, 5), (7, 40), (64, 300)])
@pytest.mark.parametrize("header", [16, 24])
def test_plan_against_the_loop(lib, requests, page, longest, header):
    rng = np.random.default_rng(requests * 31 + page)
    cached, new = rng.integers(0, 200, requests), rng.integers(0, longest + 1, requests)
    width = -(-(200 + longest) // page)
    total = int(new.sum())
    free = rng.permutation(total + requests + 5)
    check_plan(lib, cached, new, page, width, total + int(rng.integers(0, 70)), free, rng, header)


def test_plan_limits(lib):
    rng = np.random.default_rng(1)
    c, n = [0, 5, 0, 63, 64, 70, -3, 9], [0, 3, 100, 4, 1, 2, 5, -8]
    free = rng.permutation(40)
    for rows in (0, 1, 5, 50, 200):            # rows run out inside a request
        for have in (0, 1, 6, 40):             # pages run out
            check_plan(lib, c, n, 8, 8, rows, free[:have], rng)
    check_plan(lib, [], [], 16, 4, 9, free, rng)                       # no requests: every row is padding
    check_plan(lib, [3, 0], [1, 2], 4, 0, 5, free, rng)                # no room in the table at all
    check_plan(lib, [2 ** 31 - 1, 1], [2 ** 31 - 1, 2 ** 31 - 1], 16, 4, 100, free, rng)  # lengths that overflow sums


def test_plan_one_long_prompt(lib):
    rng = np.random.default_rng(2)
    check_plan(lib, [13], [70001], 16, 4400, 70100, rng.permutation(4500), rng)


# ---- rotary positions and cache write ---------------------------------------------------------------------------------
def tables(length, rot):
    inv = 10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1))
    a = np.arange(length)[:, None] * inv
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def run_append(lib, rng, tokens, heads, kv_heads, dim, in_kind, kind, rot, inter, page, header=16, fused=True, pad=0, edit=None, q_place="own", status=0):
    pages, length = -(-tokens // page) + 2, 4096
    per = heads + 2 * kv_heads
    cos, sin = tables(length, rot)
    positions = rng.integers(0, length, tokens).astype(np.int32)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if edit:
        edit(positions, slots, pages * page, length)
    shape = (pages, kv_heads, page, dim)
    kc, vc, qo = (to_bits(rng.standard_normal(s), kind) for s in (shape, shape, (tokens, heads, dim)))
    size = 4 if in_kind == F32 else 2
    if fused:
        row = per * dim + pad
        x = to_bits(rng.standard_normal((tokens, row)), in_kind)
        dx = DevBuf(x, header)
        q, k, v = (dx.t.data_ptr() + header + o * dim * size for o in (0, heads, heads + kv_heads))
        strides = (row,) * 3
        xq = x[:, :heads * dim].reshape(tokens, heads, dim)
        xk = x[:, heads * dim:(heads + kv_heads) * dim].reshape(tokens, kv_heads, dim)
        xv = x[:, (heads + kv_heads) * dim:per * dim].reshape(tokens, kv_heads, dim)
        bufs = [dx]
    else:
        xq, xk, xv = (to_bits(rng.standard_normal((tokens, h, dim)), in_kind) for h in (heads, kv_heads, kv_heads))
        bufs = [DevBuf(b, header) for b in (xq, xk, xv)]
        q, k, v = (b.ptr for b in bufs)
        strides = (heads * dim, kv_heads * dim, kv_heads * dim)
    dk, dv, dq = DevBuf(kc, header), DevBuf(vc, header), DevBuf(qo, header)
    if q_place == "q":
        dq, qo = bufs[0], xq
    dc, dsn, dp, dsl = DevBuf(cos, header), DevBuf(sin, header), DevBuf(positions, header), DevBuf(slots, header)
    ok(lib, lib.tb200_rope_append(tokens, heads, kv_heads, dim, in_kind, q if heads else None, k, v, *strides, dc.ptr if rot else None, dsn.ptr if rot else None,
                                  length, rot, int(inter), dp.ptr, kind, dq.ptr if heads else None, page, pages, dsl.ptr, dk.ptr, dv.ptr, stream_ptr()))
    torch.cuda.synchronize()
    st = C.c_int(0)
    assert lib.tb200_device_status(C.byref(st)) == 0 and st.value == status
    assert all(b.guard_intact() for b in bufs + [dk, dv, dq, dc, dsn, dp, dsl])
    f = lambda b, t: from_bits(b, t)  # noqa: E731
    ref_slots = np.where((positions < 0) | ((positions >= length) & (rot > 0)), -1, slots)
    want = ol.rope_append(f(xq, in_kind), f(xk, in_kind), f(xv, in_kind), cos, sin, positions, inter, ref_slots, f(qo, kind), f(kc, kind), f(vc, kind))
    got = [f(dq.numpy().reshape(qo.shape), kind), f(dk.numpy(), kind), f(dv.numpy(), kind)]
    for g, w in zip(got, want):
        # two fp32 products and a sum of values below 6, then one rounding to the type
        assert np.all(np.abs(g - w) <= HALF_STEP[kind] * np.abs(w) + 3 * 2.0 ** -24 * 12 + HALF_TINY[kind])


@pytest.mark.parametrize("in_kind", [F32, F16, BF16])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(4, 1, 128, 128), (7, 7, 64, 32), (6, 2, 80, 80), (5, 1, 20, 10), (0, 3, 16, 16), (2, 2, 256, 0), (3, 1, 7, 6)])
def test_append_against_64_bits(lib, in_kind, kind, inter, heads, kv_heads, dim, rot):
    rng = np.random.default_rng(dim * 7 + rot)
    for tokens, page in ((1, 16), (37, 8), (50, 7)):
        run_append(lib, rng, tokens, heads, kv_heads, dim, in_kind, kind, rot, inter, page)


@pytest.mark.parametrize("header", [16, 24])
@pytest.mark.parametrize("fused,pad", [(True, 0), (True, 4), (True, 3), (False, 0)])
def test_append_layouts(lib, header, fused, pad):
    rng = np.random.default_rng(pad)
    for in_kind in (F32, BF16):
        run_append(lib, rng, 19, 4, 2, 64, in_kind, BF16, 64, False, 16, header=header, fused=fused, pad=pad)


def test_append_in_place_of_q(lib):
    rng = np.random.default_rng(8)
    for dim, rot in ((64, 64), (20, 20)):
        run_append(lib, rng, 33, 4, 2, dim, F16, F16, rot, True, 16, fused=False, q_place="q")


@pytest.mark.parametrize("dim", [64, 20])
def test_append_leaves_out_rows_and_places(lib, dim):
    rng = np.random.default_rng(4)

    def edit(positions, slots, places, length):
        positions[3] = positions[17] = -1            # padding rows: nothing is written
        slots[5], slots[6], slots[7] = -1, places, 2 ** 40  # no place: q only
    run_append(lib, rng, 20, 4, 2, dim, F32, BF16, dim, False, 16, edit=edit)

    def beyond(positions, slots, places, length):
        positions[2] = length                        # beyond the tables: recorded, row left out
    run_append(lib, rng, 20, 4, 2, dim, F32, BF16, dim, False, 16, edit=beyond, status=-1)


def test_append_far_slots(lib):
    """Places whose element offset passes 2**32: a cache of 8.7 GB."""
    kv_heads, dim, page = 8, 128, 16
    pages = (1 << 32) // (kv_heads * dim * page) + 3000
    kc = torch.zeros(pages, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    slots = torch.tensor([pages * page - 1, (pages - 2) * page + 3, 5], device="cuda")
    positions = torch.zeros(3, dtype=torch.int32, device="cuda")
    x = torch.randn(3, 2 * kv_heads, dim, device="cuda").bfloat16()
    cos, sin = torch.ones(1, dim // 2, device="cuda"), torch.zeros(1, dim // 2, device="cuda")
    P = lambda t, o=0: C.c_void_p(t.data_ptr() + o)  # noqa: E731
    row = 2 * kv_heads * dim
    ok(lib, lib.tb200_rope_append(3, 0, kv_heads, dim, BF16, None, P(x), P(x, kv_heads * dim * 2), 0, row, row, P(cos), P(sin), 1, dim, 0, P(positions), BF16, None,
                                  page, pages, P(slots), P(kc), P(vc), stream_ptr()))
    sync_and_check(lib)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(kc[s // page, :, s % page], x[i, :kv_heads]) and torch.equal(vc[s // page, :, s % page], x[i, kv_heads:])
    assert int((kc != 0).any(-1).any(1).sum()) == 3


# ---- attention --------------------------------------------------------------------------------------------------------
def run_attention(lib, p, window=0, max_new=None, header=16, q_pad=0, out_pad=0, workspace=None):
    row = p.heads * p.dim
    qb = np.zeros((p.tokens, row + q_pad), np.uint16)
    qb[:, :row] = p.q_bits.reshape(p.tokens, row)
    ob = np.full((p.tokens, row + out_pad), 0x1234, np.uint16)
    ob[:, :row] = p.out_bits.reshape(p.tokens, row)
    dq, do, dk, dv = DevBuf(qb, header), DevBuf(ob, header), DevBuf(p.k_bits, header), DevBuf(p.v_bits, header)
    dcu, dkv, dt = DevBuf(p.cu, header), DevBuf(p.kv, header), DevBuf(p.table, header)
    n = lib.tb200_paged_attention_workspace_bytes(p.tokens, len(p.kv), p.heads, p.kv_heads, p.dim)
    assert n > 0
    ws = torch.full((n + 512,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN everywhere: nothing may be read before it is written
    if max_new is None:
        max_new = int(p.new.max(initial=0))
    ok(lib, lib.tb200_paged_attention(p.tokens, len(p.kv), max_new, p.heads, p.kv_heads, p.dim, p.kind, dq.ptr, row + q_pad, dcu.ptr, dkv.ptr, dt.ptr, p.width, p.page,
                                      p.k_bits.shape[0], dk.ptr, dv.ptr, p.scale, window, do.ptr, row + out_pad, C.c_void_p(ws.data_ptr()), n, stream_ptr()))
    sync_and_check(lib)
    assert all(b.guard_intact() for b in (dq, do, dk, dv, dcu, dkv, dt)) and bool((ws[n:] == 0xFF).all())
    got = do.numpy()
    assert np.all(got[:, row:] == 0x1234)
    return got[:, :row].reshape(p.out_bits.shape)


def check_attention(lib, p, window=0, **kw):
    got = run_attention(lib, p, window, **kw)
    want, spread = p.expected(window)
    tol = p.tolerance(want, spread)
    g = from_bits(got, p.kind)
    bad = ~np.isfinite(want)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert np.array_equal(g[bad & ~np.isnan(want)], want[bad & ~np.isnan(want)])
    off = np.abs(g[~bad] - want[~bad]) - tol[~bad]
    assert off.max(initial=-1.0) <= 0, off.max()
    used = int(p.cu[-1])
    assert np.array_equal(got[used:], p.out_bits[used:])  # rows behind the last request
    return got


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 80, 8, 104, 256, 200])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (8, 8), (14, 2), (32, 1)])
def test_attention_of_single_tokens(lib, kind, dim, heads, kv_heads):
    rng = np.random.default_rng(dim + heads)
    for cached, page in (([0, 62, 63, 64, 500], 16), ([300, 5], 7), ([1000], 128)):
        check_attention(lib, Paged(rng, cached, [1] * len(cached), heads, kv_heads, dim, page, kind))


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 96, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (3, 3), (14, 2)])
@pytest.mark.parametrize("window", [0, 1, 50, 129])
def test_attention_of_chunks(lib, kind, dim, heads, kv_heads, window):
    rng = np.random.default_rng(dim + heads + window)
    for cached, new, page in (([0, 131, 64], [70, 5, 129], 16), ([300, 0], [2, 17], 64), ([40, 7, 200], [0, 33, 0], 20)):
        check_attention(lib, Paged(rng, cached, new, heads, kv_heads, dim, page, kind, pad=3), window)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 32, 64, 128, 256, 512])
def test_attention_page_sizes(lib, page):
    rng = np.random.default_rng(page)
    check_attention(lib, Paged(rng, [515, 1, 256], [1, 1, 1], 8, 2, 128, page, BF16))
    check_attention(lib, Paged(rng, [515, 1, 256], [40, 150, 64], 8, 2, 128, page, BF16))


def test_attention_without_a_bound_on_new_tokens(lib):
    rng = np.random.default_rng(77)
    p = Paged(rng, [100, 3, 700, 0], [1, 90, 1, 20], 8, 2, 128, 16, F16)
    for max_new in (0, 1, 90, 10 ** 6):  # a hint that is too small chooses slower kernels, nothing else
        check_attention(lib, p, max_new=max_new)


@pytest.mark.parametrize("garbage", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_attention_never_reads_what_is_masked(lib, garbage, kind, dim):
    """Unused places of pages hold infinities and NaN; keys in front of the window and keys of later tokens too."""
    rng = np.random.default_rng(3)
    check_attention(lib, Paged(rng, [100, 17, 0], [1, 1, 1], 4, 1, dim, 16, kind, garbage=garbage))
    for new in ([70, 5, 30], [1, 1, 1], [150, 140, 2]):
        for window in (0, 20):
            p = Paged(rng, [300, 17, 40], new, 4, 1, dim, 16, kind, garbage=garbage)
            bad = to_bits(np.float32(garbage), kind)
            if window:  # what has slid out of every row's window
                for r in range(3):
                    for j in range(max(0, int(p.cached[r]) - window + 1)):
                        p.k_bits[p.table[r, j // 16], :, j % 16] = bad
                        p.v_bits[p.table[r, j // 16], :, j % 16] = bad
            # the last token's value, seen by the last row only
            last = int(p.kv[0]) - 1
            p.v_bits[p.table[0, last // 16], :, last % 16, ::3] = bad
            got = check_attention(lib, p, window)
            if new[0] > 1:
                assert np.isfinite(from_bits(got[:new[0] - 1], kind)).all()


def test_attention_rows_that_see_nothing(lib):
    rng = np.random.default_rng(6)
    for new, heads in (([1, 1, 1, 1], 4), ([40, 20, 33, 70], 8)):
        p = Paged(rng, [90, 0, 30, 64], new, heads, 2, 64, 16, BF16)
        p.table[0] = -1                       # no page at all
        p.table[2, 0] = p.k_bits.shape[0]     # pages outside the cache
        p.table[2, 1] = 2 ** 31 - 1
        p.table[3, 1] = -2 ** 31
        p.kv[1] = max(0, new[1] - 3)          # shorter than its new tokens: the first rows stand in front of key 0
        got = check_attention(lib, p)
        assert np.all(got[:new[0]] == 0)
        check_attention(lib, p, window=16)
    p = Paged(rng, [90, 3], [1, 2], 4, 4, 64, 16, F16)
    p.kv[:] = 0
    assert np.all(check_attention(lib, p) == 0)
    p.kv[:] = -5
    assert np.all(run_attention(lib, p) == 0)


def test_attention_scores_of_minus_infinity(lib):
    """A key of the type's lowest values, or of infinities, at visible places."""
    rng = np.random.default_rng(12)
    p = Paged(rng, [40], [3], 2, 1, 64, 16, F16)
    p.q_bits[:] = to_bits(np.abs(from_bits(p.q_bits, F16)) + 0.1, F16)
    low = to_bits(np.float32(-65504), F16)
    for j in (0, 5, 39, 41):
        p.k_bits[p.table[0, j // 16], :, j % 16] = low
    check_attention(lib, p)
    for j in range(43):
        p.k_bits[p.table[0, j // 16], :, j % 16] = to_bits(np.float32(-np.inf), F16)
    assert np.all(check_attention(lib, p) == 0)  # only scores of -infinity: zeros


def test_attention_lengths_beyond_their_table(lib):
    rng = np.random.default_rng(2)
    p = Paged(rng, [60, 20], [4, 40], 4, 2, 64, 16, F16)
    p.kv[0] += 1000                           # keys past the table row have no place
    p.cu[2] = p.tokens + 50                   # rows past the arrays are not touched
    check_attention(lib, p, max_new=0)


@pytest.mark.parametrize("header,q_pad,out_pad", [(24, 0, 0), (16, 8, 4), (24, 3, 1), (16, 2, 6)])
@pytest.mark.parametrize("new", [1, 45])
def test_attention_strides_and_headers(lib, header, q_pad, out_pad, new):
    rng = np.random.default_rng(header + q_pad)
    for dim in (64, 128, 40):
        check_attention(lib, Paged(rng, [200, 33], [new, new], 8, 2, dim, 16, BF16, pad=2), header=header, q_pad=q_pad, out_pad=out_pad)


@pytest.mark.parametrize("new", [1, 3, 100])
def test_attention_of_many_ragged_requests(lib, new):
    rng = np.random.default_rng(new)
    n = 200 if new < 100 else 9
    cached, fresh = rng.integers(0, 150, n), rng.integers(0, new + 1, n)
    check_attention(lib, Paged(rng, cached, fresh, 4, 2, 64, 16, F16, pad=5))


def test_attention_of_a_long_context_split_over_the_gpu(lib):
    rng = np.random.default_rng(21)
    p = Paged(rng, [20011], [1], 4, 1, 128, 16, BF16)
    a = check_attention(lib, p)
    assert np.array_equal(a, run_attention(lib, p))  # the parts are joined in a fixed order
    p = Paged(rng, [9000, 11], [37, 37], 8, 2, 64, 32, F16)
    assert np.array_equal(check_attention(lib, p), run_attention(lib, p))


def test_attention_far_pages(lib):
    """Pages whose element offset passes 2**32."""
    kv_heads, dim, page = 8, 128, 64
    pages = (1 << 32) // (kv_heads * dim * page) + 300
    kc = torch.empty(pages, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    rng = np.random.default_rng(0)
    for new in (1, 80):
        small = Paged(rng, [200], [new], 32, kv_heads, dim, page, BF16)
        used = [int(e) for e in small.table[0]]
        far = [pages - 1 - 7 * i for i in range(len(used))]
        for s, f in zip(used, far):
            kc[f] = torch.from_numpy(small.k_bits[s].view(np.int16)).cuda().view(torch.bfloat16)
            vc[f] = torch.from_numpy(small.v_bits[s].view(np.int16)).cuda().view(torch.bfloat16)
        table, cu, kv = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (far, [0, new], small.kv.tolist()))
        q = torch.from_numpy(small.q_bits.view(np.int16)).cuda()
        out = torch.zeros_like(q)
        n = lib.tb200_paged_attention_workspace_bytes(new, 1, 32, kv_heads, dim)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        P = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        ok(lib, lib.tb200_paged_attention(new, 1, new, 32, kv_heads, dim, BF16, P(q), 32 * dim, P(cu), P(kv), P(table), len(far), page, pages, P(kc), P(vc), small.scale, 0,
                                          P(out), 32 * dim, P(ws), n, stream_ptr()))
        sync_and_check(lib)
        want, spread = small.expected()
        got = from_bits(out.cpu().numpy().view(np.uint16), BF16)
        assert np.all(np.abs(got - want) <= small.tolerance(want, spread))


def attention_args(p, bufs, ws, n, window=0, max_new=0):
    P = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    return [p.tokens, len(p.kv), max_new, p.heads, p.kv_heads, p.dim, p.kind, P(bufs["q"]), p.heads * p.dim, P(bufs["cu"]), P(bufs["kv"]), P(bufs["table"]), p.width, p.page,
            p.k_bits.shape[0], P(bufs["k"]), P(bufs["v"]), p.scale, window, P(bufs["out"]), p.heads * p.dim, P(ws), n]


def attention_bufs(p):
    t = lambda a: torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()  # noqa: E731
    return {"q": t(p.q_bits), "cu": t(p.cu), "kv": t(p.kv), "table": t(p.table), "k": t(p.k_bits), "v": t(p.v_bits), "out": t(p.out_bits)}


@pytest.mark.parametrize("new", [1, 60])
def test_attention_captured_once_and_replayed_with_other_lengths(lib, new):
    """Lengths, offsets and tables are read on the device: a captured step is replayed as the context grows."""
    rng = np.random.default_rng(14)
    p = Paged(rng, [400, 90], [new, new], 8, 2, 128, 16, BF16)
    bufs, n = attention_bufs(p), lib.tb200_paged_attention_workspace_bytes(p.tokens, 2, 8, 2, 128)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert lib.tb200_prepare(32) == 0
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        ok(lib, lib.tb200_paged_attention(*attention_args(p, bufs, ws, n, max_new=new), C.c_void_p(side.cuda_stream)))
    for cached in ([400, 90], [7, 300], [0, 0], [399, 1]):
        p.kv[:] = np.array(cached, np.int32) + p.new
        bufs["kv"].copy_(torch.from_numpy(p.kv))
        torch.cuda.synchronize()
        g.replay()
        sync_and_check(lib)
        want, spread = p.expected()
        got = from_bits(bufs["out"].cpu().numpy().view(np.uint16), BF16)
        assert np.all(np.abs(got - want) <= p.tolerance(want, spread))


def test_attention_on_two_streams_with_a_workspace_each(lib):
    rng = np.random.default_rng(15)
    ps = [Paged(rng, [3000, 900], [1, 1], 8, 2, 128, 16, F16), Paged(rng, [700], [130], 8, 2, 64, 16, BF16)]
    streams, bufs = [torch.cuda.Stream() for _ in ps], [attention_bufs(p) for p in ps]
    ns = [lib.tb200_paged_attention_workspace_bytes(p.tokens, len(p.kv), p.heads, p.kv_heads, p.dim) for p in ps]
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in ns]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s, b, w, n in zip(ps, streams, bufs, ws, ns):
            ok(lib, lib.tb200_paged_attention(*attention_args(p, b, w, n), C.c_void_p(s.cuda_stream)))
    sync_and_check(lib)
    for p, b in zip(ps, bufs):
        want, spread = p.expected()
        assert np.all(np.abs(from_bits(b["out"].cpu().numpy().view(np.uint16), p.kind) - want) <= p.tolerance(want, spread))
