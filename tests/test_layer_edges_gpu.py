"""Ends of the decoder-layer operators' ranges on the GPU: hints that are too small, windows without an end, values near
the ends of fp32, scores whose step is more than one, probabilities far below the largest one."""
import ctypes as C

import numpy as np
import pytest
import torch

from harness import stream_ptr, sync_and_check
from layer_util import BF16, F16, F32, HALF_STEP, HALF_TINY, Paged, fp8_values, from_bits, to_bits
from oracle import layer as ol
from test_layer_gpu import attention_args, attention_bufs, check_attention, run_attention, run_norm

pytestmark = pytest.mark.gpu


# ---- attention: a bound on the new tokens that is too small -------------------------------------------------------------
@pytest.mark.parametrize("dim,heads,kv_heads,max_new", [(128, 8, 2, 5), (128, 8, 2, 12), (64, 8, 2, 6), (256, 4, 2, 1), (200, 4, 2, 3), (128, 32, 1, 1)])
def test_attention_stores_every_row_whatever_the_bound_on_new_tokens_says(lib, dim, heads, kv_heads, max_new):
    """The context is long enough for every tile of rows to be split over several blocks and joined."""
    rng = np.random.default_rng(dim + max_new)
    p = Paged(rng, [2000], [90], heads, kv_heads, dim, 16, BF16, pad=2)
    check_attention(lib, p, max_new=max_new)
    check_attention(lib, p, max_new=90)


# ---- attention: windows that end nowhere --------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30 + 1, 2 ** 30])
@pytest.mark.parametrize("new,header", [(10, 16), (40, 16), (40, 24)])
def test_attention_window_without_an_end(lib, window, new, header):
    """kv_len below the new tokens, so that the first rows stand in front of key 0: none of the others loses its keys."""
    rng = np.random.default_rng(new)
    p = Paged(rng, [0, 70], [new, new], 4, 4, 64, 16, F16)
    p.kv[0] = new - 5
    a = check_attention(lib, p, window, header=header)
    assert np.array_equal(a, run_attention(lib, p, 0, header=header))


# ---- norm: values near the ends of fp32 ---------------------------------------------------------------------------------
def check_far_norm(lib, x, weight, kind, fmt, group, eps, residual=None, **kw):
    """Codes and scales against 64 bits.  As for values near 1: the sum of `cols` squares, the root, products and
    quotients move y by `rel` of itself.  Beside that h * weight is rounded to half of the smallest subnormal at worst,
    2**-150, which the norm's factor multiplies; a factor above 2**15 meets no such products (values of rows that small
    are taken nearer to 1 first)."""
    q, scales, stored = run_norm(lib, x, residual, weight, kind, fmt, group, eps=eps, **kw)
    rx, rr = from_bits(to_bits(x, kind), kind), None if residual is None else from_bits(to_bits(residual, kind), kind)
    w32 = weight.astype(np.float32)
    ratio, want, h = ol.rmsnorm_quant(rx, rr, w32, float(np.float32(eps)), fmt, group)
    cols = x.shape[1]
    rel = (0.5 * cols + 12) * 2.0 ** -24
    with np.errstate(all="ignore"):
        factor = 1 / np.sqrt((h * h).mean(1) + float(np.float32(eps)))
    lost = np.minimum(factor, 2.0 ** 15)[:, None] * 2.0 ** -150
    assert np.isfinite(want).all()
    assert np.all(np.abs(scales - want) <= rel * want + lost + 2.0 ** -149)
    g = group or cols
    scale_of = np.repeat(want, g, 1)[:, :cols]
    val = q.view(np.int8).astype(np.float64) if fmt == "int8" else fp8_values(q, fmt)
    assert np.isfinite(val).all()
    moved = np.abs(ratio) * (2 * rel + 2.0 ** -23) + lost / scale_of
    if fmt == "int8":
        bound = 0.5 + moved + 2.0 ** -17
    else:
        m, low = (3, -9) if fmt == "e4m3" else (2, -16)
        _, e = np.frexp(np.maximum(np.abs(ratio) + moved, 1e-300))
        bound = 0.5 * np.exp2(np.maximum(e - 1 - m, low).astype(np.float64)) + moved
    off = np.abs(val - ratio)
    assert np.all(off <= bound), (off - bound).max()
    if stored is not None:
        s = from_bits(stored, kind)
        assert np.all(np.abs(s - h) <= (HALF_STEP[kind] + 2.0 ** -24) * np.abs(h) + HALF_TINY[kind])
    return q, scales


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("fmt,group", [("int8", 32), ("int8", 0), ("e4m3", 128), ("e4m3", 0), ("e5m2", 64), ("e5m2", 32)])
@pytest.mark.parametrize("rows,cols", [(9, 256), (400, 512), (9, 33024)])
def test_norm_groups_down_to_subnormals(lib, kind, fmt, group, rows, cols):
    """Dead groups in an ordinary row, and rows that are tiny altogether (the factor of the norm is 316 there), with zeros
    among them: no code is a NaN, and none is off."""
    rng = np.random.default_rng(cols)
    w = 1 + 0.3 * rng.standard_normal(cols)
    x = rng.standard_normal((rows, cols))
    for i, tiny in enumerate((1e-30, 1e-34, 1e-36, 1e-37, 1e-38, 1e-39, 1e-41, 0.0)):
        x[i] *= 0.01
        x[i, 128:256] *= tiny * 100
        x[i, 130:140] = 0
    check_far_norm(lib, x, w, kind, fmt, group, 1e-5)
    for i, tiny in enumerate((1e-20, 1e-30, 1e-34, 1e-36, 1e-37, 1e-38, 1e-39, 1e-41)):
        x[i] = rng.standard_normal(cols) * tiny
        x[i, 3:200:7] = 0
    check_far_norm(lib, x, w, kind, fmt, group, 1e-5)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("fmt,group", [("int8", 32), ("e4m3", 0), ("e5m2", 128)])
@pytest.mark.parametrize("rows,cols", [(12, 96), (12, 4096), (500, 512), (12, 8200), (12, 16400), (320, 16400), (12, 33024), (12, 33001)])
@pytest.mark.parametrize("eps", [0.0, 1e-35, 1e-5])
def test_norm_of_rows_whose_squares_leave_fp32(lib, kind, fmt, group, rows, cols, eps):
    """The norm does not depend on a row's magnitude, so long as the sum h and the products h * weight are finite."""
    rng = np.random.default_rng(cols + int(eps * 1e6))
    w = 1 + 0.3 * rng.standard_normal(cols)
    x = rng.standard_normal((rows, cols))
    for i, size in enumerate((1e18, 1e25, 3e37, 1e-15, 1e-21, 1e-30, 1e-37, 1e-40)):
        x[i] *= size
    x[8, :40] *= 1e30            # huge values beside ordinary ones
    x[9, 50] = 3e38              # one huge value alone
    x[9, 0:32] *= 1e-3
    x[10, 20:96] *= 1e-25        # tiny groups in an ordinary row
    x[11, 1] = 1e21              # a huge channel that the weights leave out, for the row with it
    check_far_norm(lib, x, w, kind, fmt, group, eps, residual=np.zeros_like(x), place="residual")
    w[1] = 0
    check_far_norm(lib, x[11:12], w, kind, fmt, group, eps)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("place", ["own", "residual", "x", "none"])
@pytest.mark.parametrize("rows,cols", [(12, 512), (500, 512), (12, 9000), (400, 18000), (12, 33000), (400, 61)])
@pytest.mark.parametrize("header", [16, 24])
def test_norm_of_far_rows_wherever_the_sum_goes(lib, kind, place, rows, cols, header):
    """Rows far from 1 are read again when the others are done: the sum may stand in their inputs' place by then."""
    rng = np.random.default_rng(cols + header)
    x, r, w = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols)), 1 + 0.3 * rng.standard_normal(cols)
    far = np.arange(rows) % 5 == 1
    size = 1e3 if kind == F16 else 1e25
    x[far] *= size
    r[far] *= size * 0.01
    r[np.arange(rows) % 5 == 3] *= 1e-3 if kind == F16 else 1e-30
    x[np.arange(rows) % 5 == 3] *= 1e-3 if kind == F16 else 1e-30
    check_far_norm(lib, x, w, kind, "int8", 32, 0.0, residual=r, place=place, header=header)
    check_far_norm(lib, x, w, kind, "e4m3", 0, 1e-5, residual=r, place=place, header=header)


@pytest.mark.parametrize("kind,place", [(BF16, "residual"), (BF16, "own"), (F32, "x")])
def test_norm_of_far_rows_among_more_rows_than_a_block_remembers(lib, kind, place):
    rng = np.random.default_rng(11)
    rows, cols = 148 * 28 * 32 + 8001, 64
    x, r, w = rng.standard_normal((rows, cols), np.float32), rng.standard_normal((rows, cols), np.float32), 1 + 0.3 * rng.standard_normal(cols)
    far = rng.random(rows) < 0.01
    far[[0, rows - 1]] = True
    x[far] *= 1e25
    check_far_norm(lib, x.astype(np.float64), w, kind, "int8", 32, 1e-5, residual=r.astype(np.float64), place=place)


# ---- attention: scores whose fp32 step is more than one ------------------------------------------------------------------
def far_scores(rng, kind, new, cached, heads, dim, q, k, requests=1):
    p = Paged(rng, [cached] * requests, [new] * requests, heads, 1 if requests == 1 else heads, dim, 16, kind)
    p.q_bits[:] = to_bits(np.full(p.q_bits.shape, q, np.float32), kind)
    p.k_bits[:] = to_bits(np.full(p.k_bits.shape, k, np.float32), kind)
    return p


@pytest.mark.parametrize("kind,q,k", [(F16, 1000.0, 60000.0), (F16, 30000.0, 65504.0), (F16, -30000.0, 65504.0), (BF16, 2.0 ** 30, 2.0 ** 31), (BF16, 3 * 2.0 ** 29, 5 * 2.0 ** 28), (BF16, -3 * 2.0 ** 29, 5 * 2.0 ** 28)])
@pytest.mark.parametrize("new,header", [(1, 16), (40, 16), (40, 24)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_huge_equal_scores_is_the_mean(lib, kind, q, k, new, header, dim):
    """Every product is the same number, so every fp32 sum of them is too, whatever its rounding: equal weights."""
    p = far_scores(np.random.default_rng(dim), kind, new, 300, 4, dim, q, k)
    want, spread = p.expected()
    u, n = HALF_STEP[kind], int(p.kv[0])
    got = from_bits(run_attention(lib, p, header=header), kind)
    assert np.all(np.abs(got - want) <= u * np.abs(want) + (u + (n + 8) * 2.0 ** -23) * spread + HALF_TINY[kind])


@pytest.mark.parametrize("new,header", [(1, 16), (20, 16), (20, 24)])
def test_attention_of_huge_scores_a_step_apart(lib, new, header):
    """Scores of 2**27 + 16 in one key tile and 2**27 + 32 in the next one, in powers of two: a step of fp32 apart, and
    2**-16 the weight."""
    scale = next(float(s) for s in (np.float32(np.log(2)), np.nextafter(np.float32(np.log(2)), np.float32(1)), np.nextafter(np.float32(np.log(2)), np.float32(0)))
                 if np.float32(s) * np.float32(1.4426950408889634) == 1.0)
    p = far_scores(np.random.default_rng(4), F16, new, 128, 8, 64, 0.0, 0.0, requests=60)  # items that no block shares, most of them
    p.scale = scale
    q, k = np.zeros(64, np.float32), np.zeros(64, np.float32)
    q[:2], k[:2] = (2.0 ** 13, 4.0), (2.0 ** 14, 4.0)
    p.q_bits[:], p.k_bits[:] = to_bits(q, F16), to_bits(k, F16)
    k[1] = 8.0
    for r in range(60):
        p.k_bits[p.table[r, 4:8]] = to_bits(k, F16)
    got = from_bits(run_attention(lib, p, header=header), F16)
    want, spread = p.expected()
    u = HALF_STEP[F16]
    # the 64-bit form's scale is ln 2 to half a step of fp32: scores of 2**27 move by 8, but alike; their difference of 16 by 2**-20
    assert np.all(np.abs(got - want) <= u * np.abs(want) + (u + 200 * 2.0 ** -23 + 2.0 ** -19) * spread + HALF_TINY[F16])


# ---- attention: a long flat tail far below one large score ---------------------------------------------------------------
@pytest.mark.parametrize("requests,new,header", [(60, 1, 16), (20, 20, 16), (20, 20, 24)])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("gap", [12.0, 16.9, 17.6])
def test_attention_keeps_a_tail_of_small_probabilities(lib, requests, new, header, kind, gap):
    """One key takes nearly all of the weight and has V = 0; the result is what thousands of keys at e**-gap of it have.
    An fp16 probability is held to half a step of the type down to 2**-14 of the largest one at least, and below that to
    2**-25 times what the probabilities are raised by before the rounding (2**7 at least)."""
    rng = np.random.default_rng(requests)
    cached, heads, dim = 2000, 8, 64
    p = Paged(rng, [cached] * requests, [new] * requests, heads, heads, dim, 16, kind)
    p.scale = 0.125
    p.q_bits[:] = to_bits(np.full(p.q_bits.shape, 1.0, np.float32), kind)
    low = to_bits(np.full(p.k_bits.shape, 1.0, np.float32), kind)
    p.k_bits[:] = low
    p.v_bits[:] = to_bits(1 + 0.25 * rng.random(p.v_bits.shape), kind)
    first = np.full(dim, 1.0, np.float32)
    first[:8] += gap  # 8 * gap / 8: exact in both types where gap + 1 is
    for r in range(requests):
        p.k_bits[p.table[r, 0], :, 0], p.v_bits[p.table[r, 0], :, 0] = to_bits(first, kind), 0
    got = from_bits(run_attention(lib, p, header=header), kind)
    want, spread = p.expected()
    u, n = HALF_STEP[kind], cached + new
    ds = (dim + 2) * 2.0 ** -23 * 8.0 * np.sqrt((from_bits(to_bits(first, kind), kind) ** 2).sum()) * p.scale
    tail = n * HALF_TINY[kind] * 2.0 ** -7 * 1.25
    tol = u * np.abs(want) + (1 + u) * (u + 2 * ds + (n + 8) * 2.0 ** -23) * spread + tail + HALF_TINY[kind]
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) - tol)


# ---- attention: nothing but scores of minus infinity ---------------------------------------------------------------------
@pytest.mark.parametrize("value", [np.inf, np.nan])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("cached,new,header", [(40, 1, 16), (40, 3, 16), (100, 40, 16), (100, 40, 24), (5000, 1, 16), (5000, 40, 16)])
def test_attention_rows_of_minus_infinity_are_zeros_whatever_their_values(lib, value, kind, cached, new, header):
    rng = np.random.default_rng(cached + new)
    p = Paged(rng, [cached], [new], 4, 2, 64, 16, kind)
    p.q_bits[:] = to_bits(np.abs(from_bits(p.q_bits, kind)) + 0.1, kind)
    p.k_bits[:] = to_bits(np.float32(-np.inf), kind)
    p.v_bits[:, :, ::3] = to_bits(np.float32(value), kind)
    assert np.all(run_attention(lib, p, header=header)[:new] == 0)


# ---- plan: arrays that lie next to one another ----------------------------------------------------------------------------
def test_plan_of_neighbouring_arrays_and_shared_lengths(lib):
    """Only an output over another array is refused: kv_lens may begin where cached_lens ends, and both lengths may be one
    array."""
    n, page, width, rows = 3, 4, 5, 16
    lens, free = np.array([3, 0, 6], np.int32), np.arange(10, 16, dtype=np.int32)
    table = np.arange(n * width, dtype=np.int32).reshape(n, width)
    want = ol.paged_plan(lens, lens, page, width, rows, free, table)
    b = torch.zeros(512, dtype=torch.int32, device="cuda")
    places, at = {}, 0
    for name, size in (("slots", 2 * rows), ("cached", n), ("kv", n), ("cu", n + 1), ("counts", 4), ("positions", rows), ("free", len(free)), ("table", n * width)):
        places[name], at = (at, size), at + size
    host = b.cpu().numpy()
    host[places["cached"][0]:][:n], host[places["free"][0]:][:len(free)], host[places["table"][0]:][:n * width] = lens, free, table.ravel()
    b.copy_(torch.from_numpy(host))
    P = lambda k: C.c_void_p(b.data_ptr() + 4 * places[k][0])  # noqa: E731
    assert lib.tb200_paged_plan(n, page, width, rows, len(free), P("cached"), P("cached"), P("free"), P("table"), P("cu"), P("kv"), P("positions"), P("slots"), P("counts"),
                                stream_ptr()) == 0
    sync_and_check(lib)
    got = b.cpu().numpy()
    take = lambda k: got[places[k][0]:][:places[k][1]]  # noqa: E731
    assert np.array_equal(take("table").reshape(n, width), want[0]) and np.array_equal(take("slots").view(np.int64), want[4])
    for k, w in (("cu", want[1]), ("kv", want[2]), ("positions", want[3]), ("counts", want[5])):
        assert np.array_equal(take(k), w), k


# ---- attention: the result in the place of the queries --------------------------------------------------------------------
@pytest.mark.parametrize("cached,new,page", [([3000, 40], [1, 1], 16), ([100, 30], [1, 1], 16), ([700, 20], [90, 150], 16), ([700, 20], [90, 150], 20), ([0, 0], [300, 5], 64)])
@pytest.mark.parametrize("dim", [64, 256])
def test_attention_in_place_of_its_queries(lib, cached, new, page, dim):
    p = Paged(np.random.default_rng(dim), cached, new, 8, 2, dim, page, BF16, pad=2)
    bufs = attention_bufs(p)
    n = lib.tb200_paged_attention_workspace_bytes(p.tokens, 2, 8, 2, dim)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    q, used = bufs["q"].clone(), int(p.cu[-1])
    for b in (bufs, bufs | {"q": q, "out": q}):
        assert lib.tb200_paged_attention(*attention_args(p, b, ws, n, max_new=max(new)), stream_ptr()) == 0
    sync_and_check(lib)
    assert torch.equal(q[:used], bufs["out"][:used]) and torch.equal(q[used:], bufs["q"][used:])
