"""The decoder-layer operators together, as a model's step uses them: through the C ABI with the library's 8-bit product
between, and as a task graph that is captured once and replayed while its requests grow."""
import ctypes as C

import numpy as np
import pytest
import torch

from layer_util import BF16, F16, HALF_STEP, fp8_values, from_bits, to_bits
from oracle import layer as ol
from tornadovm_b200 import B200Native
from tornadovm_b200.arrays import BFloat16Array, FloatArray, HalfFloatArray, Int8Array, IntArray, LongArray
from tornadovm_b200.b200 import B200
from tornadovm_b200.taskgraph import DataTransferMode, TaskGraph, TornadoExecutionPlan

pytestmark = pytest.mark.gpu


def angles(length, rot):
    inv = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    a = np.arange(length)[:, None] * inv
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


class History:
    """Every request's keys and values in one piece, in 64 bits."""

    def __init__(self, requests, kv_heads, dim):
        self.k = [np.zeros((0, kv_heads, dim)) for _ in range(requests)]
        self.v = [np.zeros((0, kv_heads, dim)) for _ in range(requests)]

    def add(self, r, k, v):
        self.k[r], self.v[r] = np.concatenate((self.k[r], k)), np.concatenate((self.v[r], v))

    def attend(self, r, q, scale):
        """Softmax attention of the request's last rows; and the same of |v|, for the tolerance."""
        n, heads, dim = q.shape
        group = heads // self.k[r].shape[1]
        out, spread = np.zeros_like(q), np.zeros_like(q)
        for i in range(n):
            seen = len(self.k[r]) - n + i + 1
            for h in range(heads):
                s = self.k[r][:seen, h // group] @ q[i, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, h], spread[i, h] = w @ self.v[r][:seen, h // group], w @ np.abs(self.v[r][:seen, h // group])
        return out, spread


@pytest.mark.parametrize("kind", [F16, BF16])
def test_steps_of_a_layer_with_the_fp8_product(kind):
    """Norm to e4m3 -> fp8 product -> scales -> rotary write -> attention, for a prompt and three decoded tokens of three
    requests.  Each stage is compared with its 64-bit form on the values that the stage before it has left."""
    rng = np.random.default_rng(kind)
    R, hidden, heads, kv_heads, dim, page, width = 3, 256, 8, 2, 64, 16, 8
    rows_out = (heads + 2 * kv_heads) * dim
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    P = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    S = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    bits = lambda x: dev(to_bits(x, kind).view(np.int16))  # noqa: E731
    host = lambda t: from_bits(t.cpu().numpy().view(np.uint16), kind)  # noqa: E731
    norm_w = (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)
    w8 = rng.integers(0, 256, (hidden, rows_out)).astype(np.uint8)
    w8[np.isnan(fp8_values(w8, "e4m3"))] = 0
    w_scale = 1.0 / 1600.0
    cos, sin = angles(width * page, dim)
    free = rng.permutation(64).astype(np.int32)
    d_norm, d_w, d_cos, d_sin = dev(norm_w), dev(w8), dev(cos), dev(sin)
    kc, vc = (bits(rng.standard_normal((64, kv_heads, page, dim))) for _ in range(2))
    table = dev(np.full((R, width), -1, np.int32))
    kv = dev(np.zeros(R, np.int32))
    past, taken, scale = History(R, kv_heads, dim), 0, dim ** -0.5
    for new in ([37, 5, 70], [1, 1, 1], [1, 0, 1], [1, 1, 1]):
        T = sum(new)
        pad = T + 4
        x, res = rng.standard_normal((T, hidden)), 2 * rng.standard_normal((T, hidden))
        dx, dr = bits(x), bits(res)
        q8, s8 = torch.empty(T, hidden, dtype=torch.uint8, device="cuda"), torch.empty(T, device="cuda")
        B200Native.call("tb200_rmsnorm_quant", T, hidden, kind, P(dx), hidden, P(dr), P(dr), P(d_norm), 1e-5, 1, 0, P(q8), P(s8), S)
        y = torch.empty(T, rows_out, device="cuda")
        n = B200Native.load().tb200_igemm_workspace_bytes(rows_out, hidden)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        B200Native.call("tb200_fp8gemm_f32", T, rows_out, hidden, 0, P(q8), P(d_w), P(y), P(ws), n, S)
        qkv = torch.zeros(pad, rows_out, device="cuda")
        qkv[:T] = y * (s8 * w_scale)[:, None]
        # the step's layout: kv_lens of the step before are the cached lengths of this one
        cached, d_new, d_free = kv.clone(), dev(np.array(new, np.int32)), dev(free[taken:])
        cu, positions, slots, counts = (torch.empty(k, dtype=t, device="cuda") for k, t in ((R + 1, torch.int32), (pad, torch.int32), (pad, torch.int64), (4, torch.int32)))
        B200Native.call("tb200_paged_plan", R, page, width, pad, 64 - taken, P(cached), P(d_new), P(d_free), P(table), P(cu), P(kv), P(positions), P(slots), P(counts), S)
        q = torch.zeros(pad, heads, dim, dtype=torch.int16, device="cuda")
        at = qkv.data_ptr()
        B200Native.call("tb200_rope_append", pad, heads, kv_heads, dim, 0, at, at + 4 * heads * dim, at + 4 * (heads + kv_heads) * dim, rows_out, rows_out, rows_out,
                        P(d_cos), P(d_sin), width * page, dim, 0, P(positions), kind, P(q), page, 64, P(slots), P(kc), P(vc), S)
        out = torch.full((pad, heads, dim), 77, dtype=torch.int16, device="cuda")
        nb = B200Native.load().tb200_paged_attention_workspace_bytes(pad, R, heads, kv_heads, dim)
        aws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        B200Native.call("tb200_paged_attention", pad, R, max(new), heads, kv_heads, dim, kind, P(q), heads * dim, P(cu), P(kv), P(table), width, page, 64, P(kc), P(vc),
                        scale, 0, P(out), heads * dim, P(aws), nb, S)
        torch.cuda.synchronize()
        assert B200Native.device_status(32) == 0
        # norm: e4m3 values are off by 2**-4 of themselves at most, and by half the smallest step
        ratio, want_s, h = ol.rmsnorm_quant(from_bits(to_bits(x, kind), kind), from_bits(to_bits(res, kind), kind), norm_w, 1e-5, "e4m3", 0)
        assert np.allclose(s8.cpu().numpy(), want_s[:, 0], rtol=1e-5)
        v8 = fp8_values(q8.cpu().numpy(), "e4m3")
        assert np.all(np.abs(v8 - ratio) <= 2.0 ** -4 * np.abs(ratio) + 2.0 ** -10 + 1e-3 * np.abs(ratio))
        assert np.all(np.abs(host(dr) - h) <= HALF_STEP[kind] * np.abs(h) * 1.001 + 1e-7)
        prod = v8 @ fp8_values(w8, "e4m3") * s8.cpu().numpy().astype(np.float64)[:, None] * w_scale
        rows = qkv[:T].cpu().numpy().astype(np.float64)
        assert np.allclose(rows, prod, rtol=1e-4, atol=1e-4 * np.abs(prod).max())
        # layout and cache
        cnt = counts.cpu().numpy()
        assert cnt[0] == cnt[1] == T and cnt[2] == cnt[3]
        taken += int(cnt[2])
        pos = positions.cpu().numpy()
        assert np.all(pos[T:] == -1)
        rows = rows.reshape(T, heads + 2 * kv_heads, dim)
        turned = ol.rope(rows[:, :heads + kv_heads], cos, sin, pos[:T], False)
        got_q, got_out = host(q)[:T], host(out)
        assert np.all(np.abs(got_q - turned[:, :heads]) <= HALF_STEP[kind] * np.abs(turned[:, :heads]) + 1e-5)
        assert np.all(got_out[T:] == from_bits(np.full(1, 77, np.uint16), kind))
        start = 0
        for r in range(R):
            here = slice(start, start + new[r])
            store = lambda a: from_bits(to_bits(a, kind), kind)  # noqa: E731
            past.add(r, store(turned[here, heads:]), store(rows[here, heads + kv_heads:]))
            want, spread = past.attend(r, got_q[here], scale)
            # the result's and the probabilities' rounding; a key of the history may be one step off (1e-5 of its fp32
            # value moves it over a rounding border), which moves a score by 2 * half a step of |q| |k| scale at most
            u = HALF_STEP[kind]
            big = np.sqrt((got_q[here] ** 2).sum(-1)).max(initial=0) * max(np.sqrt((past.k[r] ** 2).sum(-1)).max(initial=0), 1e-9) * scale
            assert np.all(np.abs(got_out[here] - want) <= u * np.abs(want) + (3 * u + 1e-4 + 4 * u * big / np.sqrt(dim)) * spread + 1e-6)
            start += new[r]


@pytest.mark.parametrize("header", [16, 24])
@pytest.mark.parametrize("array", [HalfFloatArray, BFloat16Array])
def test_decode_graph_of_layer_tasks(header, array):
    """pagedPlan -> ropeAppend -> pagedAttention and the norm as library tasks, captured in the first execution and replayed
    for five tokens with the caches kept on the device."""
    rng = np.random.default_rng(header)
    kind = F16 if array is HalfFloatArray else BF16
    R, heads, kv_heads, dim, page, width, pages = 2, 4, 1, 64, 4, 6, 16
    per = (heads + 2 * kv_heads) * dim
    cos, sin = angles(width * page, dim)
    f = lambda a: FloatArray(np.asarray(a, np.float32), header)  # noqa: E731
    i = lambda a: IntArray(np.asarray(a, np.int32), header)  # noqa: E731
    qkv, cached, new = f(np.zeros(R * per)), i([0] * R), i([1] * R)
    table, cu, kv, positions, slots, counts = i(np.full(R * width, -1)), i([0] * (R + 1)), i([0] * R), i([0] * R), LongArray(np.zeros(R, np.int64), header), i([0] * 4)
    free = i(rng.permutation(pages))
    cache = pages * kv_heads * page * dim
    kc, vc, q, out = (array(np.zeros(n, np.uint16), header) for n in (cache, cache, R * heads * dim, R * heads * dim))
    x, res, w = array.from_float32(rng.standard_normal(R * 96), header), array.from_float32(rng.standard_normal(R * 96), header), f(rng.standard_normal(96))
    q8, s8 = Int8Array(np.zeros(R * 96, np.int8), header), f(np.zeros(R * 3))
    tg = (TaskGraph("layer")
          .transferToDevice(DataTransferMode.FIRST_EXECUTION, kc, vc, table, w, f(cos.ravel()), f(sin.ravel()))
          .transferToDevice(DataTransferMode.EVERY_EXECUTION, qkv, cached, new, free, x, res))
    d_cos, d_sin = tg.to_device[4][1], tg.to_device[5][1]
    tg = (tg.libraryTask("norm", B200.addRmsnormQuant, R, 96, x, res, w, 1e-5, "int8", 32, q8, s8)
          .libraryTask("plan", B200.pagedPlan, R, page, width, R, cached, new, free, table, cu, kv, positions, slots, counts)
          .libraryTask("rope", B200.ropeAppend, R, heads, kv_heads, dim, qkv, d_cos, d_sin, dim, True, positions, slots, page, q, kc, vc)
          .libraryTask("attend", B200.pagedAttention, R, R, 1, heads, kv_heads, dim, q, cu, kv, table, page, kc, vc, 0.125, 0, out)
          .transferToHost(DataTransferMode.EVERY_EXECUTION, out, q, counts, kv, q8, s8, res))
    past, order, used = History(R, kv_heads, dim), free.numpy().copy(), 0
    with TornadoExecutionPlan(tg).withCUDAGraph() as plan:
        for step in range(5):
            rows = rng.standard_normal((R, per)).astype(np.float32)
            x_h, r_h = rng.standard_normal(R * 96), rng.standard_normal(R * 96)
            qkv.numpy()[:] = rows.ravel()
            cached.numpy()[:] = step
            free.numpy()[:] = np.concatenate((order[used:], np.full(used, -1)))  # the pages that are left, in front
            x.numpy()[:], res.numpy()[:] = to_bits(x_h, kind), to_bits(r_h, kind)
            plan.execute()
            used += int(counts.numpy()[2])
            assert kv.numpy().tolist() == [step + 1] * R and counts.numpy()[0] == R
            r3 = rows.astype(np.float64).reshape(R, -1, dim)
            turned = ol.rope(r3[:, :heads + kv_heads], cos, sin, np.full(R, step), True)
            u, got_q = HALF_STEP[kind], from_bits(q.numpy(), kind).reshape(R, heads, dim)
            assert np.all(np.abs(got_q - turned[:, :heads]) <= u * np.abs(turned[:, :heads]) + 1e-5)
            got = from_bits(out.numpy(), kind).reshape(R, heads, dim)
            for r in range(R):
                store = lambda a: from_bits(to_bits(a, kind), kind)  # noqa: E731
                past.add(r, store(turned[r:r + 1, heads:]), store(r3[r:r + 1, heads + kv_heads:]))
                want, spread = past.attend(r, got_q[r:r + 1], 0.125)
                assert np.all(np.abs(got[r] - want[0]) <= u * np.abs(want[0]) + (3 * u + 1e-4 + 4 * u * 16) * spread[0] + 1e-6)
            ratio, scales, h = ol.rmsnorm_quant(from_bits(to_bits(x_h, kind), kind).reshape(R, 96), from_bits(to_bits(r_h, kind), kind).reshape(R, 96), w.numpy(), 1e-5, "int8", 32)
            assert np.allclose(s8.numpy().reshape(R, 3), scales, rtol=1e-5)
            assert np.all(np.abs(q8.numpy().reshape(R, 96) - ratio) <= 0.5 + 1e-2)
            assert np.all(np.abs(from_bits(res.numpy(), kind).reshape(R, 96) - h) <= u * np.abs(h) * 1.001 + 1e-7)
    assert B200Native.device_status(32) == 0
