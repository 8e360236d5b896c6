"""Factories of the ``b200/linalg`` library tasks.

Python twin of the Java class ``B200``; same shape as ``Cutlass``
(tornado-cutlass/.../Cutlass.java:44-191) and ``CuBlas``
(tornado-cublas/.../CuBlas.java:97-305): each factory validates shapes early
with a clear message and returns a LibraryTaskDescriptor whose parameter list
is what the provider later receives positionally.
"""
from __future__ import annotations

from dataclasses import dataclass

from .arrays import BFloat16Array, ByteArray, FloatArray, HalfFloatArray, Int8Array, IntArray, LongArray
from .descriptor import Access, LibraryTaskDescriptor

LIBRARY_NAME = "b200/linalg"
MAX_BATCH = 16
MAX_GROUP = 32
#: TaskGraph.libraryTask takes at most 20 arguments (TaskGraph.java:886): rows, cols, batch, x, y, options + 14 matrices
MAX_GROUP_TASK_ARGS = 14
#: tb200_type of an array, tb200_quant_format by name (include/tornado_b200.h)
ELEMENT_TYPES = {FloatArray: 0, HalfFloatArray: 1, BFloat16Array: 2}
QUANT_FORMATS = {"int8": 0, "e4m3": 1, "e5m2": 2}
MAX_PLAN_REQUESTS = 16384


@dataclass
class B200Options:
    """Per-call tuning object (LibraryTaskDescriptor.withTuning):
    ``exact_int`` selects the int8-activation / int32 block-dot arithmetic for
    the quantised mat-vec tasks; ``overlap_launches`` lets consecutive mat-vec
    kernels of the plan overlap (each prefetches its weights while the kernel
    before it drains), which requires that no task writes a weight array
    immediately before the mat-vec that reads it; ``host_results`` lets the
    grouped and packed mat-vec kernels store every result into the output array's pinned,
    device-mapped host segment as well as into its device buffer, when the
    graph copies that array to the host after every execution -- the plan
    then has no device-to-host copy left to issue for it."""
    exact_int: bool = False
    overlap_launches: bool = False
    host_results: bool = False


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError("[ERROR] " + msg)


def _desc(function, params, out_index, read_write=False, tuning=None):
    """``out_index``: the output's place in ``params``, or a dict of the outputs' places and their access."""
    access = [Access.READ_ONLY] * len(params)
    if isinstance(out_index, dict):
        for i, kind in out_index.items():
            access[i] = kind
    else:
        access[out_index] = Access.READ_WRITE if read_write else Access.WRITE_ONLY
    d = LibraryTaskDescriptor().withLibrary(LIBRARY_NAME).withFunction(function).withParameters(params).withAccess(access)
    if tuning is not None:
        d.withTuning(tuning)
    return d


class B200:
    LIBRARY_NAME = LIBRARY_NAME

    @staticmethod
    def sgemv(rows: int, cols: int, m: FloatArray, v: FloatArray, out: FloatArray):
        """out[i] = sum_j m[i*cols+j] * v[j] (README mxv, README.md:35-47)."""
        _check(rows >= 0 and cols >= 0, f"B200 sgemv requires non-negative sizes; got rows={rows}, cols={cols}")
        _check(m.getSize() >= rows * cols and v.getSize() >= cols and out.getSize() >= rows,
               "B200 sgemv: array smaller than rows x cols")
        return _desc("sgemv", [rows, cols, m, v, out], 4)

    @staticmethod
    def _check_q(name, rows, cols, batch, x, y):
        _check(cols % 32 == 0, f"B200 {name} requires cols to be a multiple of the 32-element block; got cols={cols}")
        _check(1 <= batch <= MAX_BATCH, f"B200 {name} requires 1 <= batch <= {MAX_BATCH}; got {batch}")
        _check(x.getSize() >= batch * cols and y.getSize() >= batch * rows, f"B200 {name}: x or y too small")

    @staticmethod
    def q8Gemv(rows, cols, batch, q: Int8Array, scales: HalfFloatArray, x: FloatArray, y: FloatArray, options=None):  # noqa: N802
        """Q8_0 mat-vec, split layout (matrixVectorGenericFinal, MatrixVectorRowMajor.java:409-423)."""
        B200._check_q("q8Gemv", rows, cols, batch, x, y)
        _check(q.getSize() >= rows * cols and scales.getSize() >= rows * cols // 32, "B200 q8Gemv: weights too small")
        return _desc("q8Gemv", [rows, cols, batch, q, scales, x, y], 6, tuning=options)

    @staticmethod
    def q8GemvBytes(rows, cols, batch, blocks: ByteArray, x: FloatArray, y: FloatArray, options=None):  # noqa: N802
        """Q8_0 mat-vec, 34-byte blocks (matrixVectorGenericQ8Byte, MatrixVectorRowMajor.java:428-524)."""
        B200._check_q("q8GemvBytes", rows, cols, batch, x, y)
        _check(blocks.getSize() >= rows * (cols // 32) * 34, "B200 q8GemvBytes: weights too small")
        return _desc("q8GemvBytes", [rows, cols, batch, blocks, x, y], 5, tuning=options)

    @staticmethod
    def q4GemvBytes(rows, cols, batch, blocks: ByteArray, x: FloatArray, y: FloatArray, options=None):  # noqa: N802
        """Q4_0 mat-vec, 18-byte blocks."""
        B200._check_q("q4GemvBytes", rows, cols, batch, x, y)
        _check(blocks.getSize() >= rows * (cols // 32) * 18, "B200 q4GemvBytes: weights too small")
        return _desc("q4GemvBytes", [rows, cols, batch, blocks, x, y], 5, tuning=options)

    @staticmethod
    def _grouped(name, block_bytes, rows, cols, batch, x, y, blocks, options):
        B200._check_q(name, rows, cols, batch, x, y)
        _check(1 <= len(blocks) <= MAX_GROUP_TASK_ARGS,
               f"B200 {name} requires 1 to {MAX_GROUP_TASK_ARGS} matrices (a library task carries 20 arguments); got {len(blocks)}; "
               f"use {name.replace('Grouped', 'Packed')} for up to {MAX_GROUP}")
        _check(y.getSize() >= len(blocks) * batch * rows, f"B200 {name}: y smaller than count x batch x rows")
        for b in blocks:
            _check(b.getSize() >= rows * (cols // 32) * block_bytes, f"B200 {name}: weights too small")
        _check(options is None or options.exact_int, f"B200 {name} computes in integer mode; exact_int must be set")
        return _desc(name, [len(blocks), rows, cols, batch, x, y, *blocks], 5, tuning=options or B200Options(exact_int=True))

    @staticmethod
    def q8GemvBytesGrouped(rows, cols, batch, x: FloatArray, y: FloatArray, *blocks: ByteArray, options=None):  # noqa: N802
        """Integer-mode Q8_0 mat-vec of several equally shaped matrices on the same activations in one launch:
        y[m][b][r] for matrix m.  The reference launches one task per matrix; its batched interfaces are the
        strided GEMMs (CuBlas.cublasSgemmStridedBatched, CuBlas.java:206-228)."""
        return B200._grouped("q8GemvBytesGrouped", 34, rows, cols, batch, x, y, blocks, options)

    @staticmethod
    def q4GemvBytesGrouped(rows, cols, batch, x: FloatArray, y: FloatArray, *blocks: ByteArray, options=None):  # noqa: N802
        """Q4_0 twin of q8GemvBytesGrouped."""
        return B200._grouped("q4GemvBytesGrouped", 18, rows, cols, batch, x, y, blocks, options)

    @staticmethod
    def _packed(name, block_bytes, count, rows, cols, batch, blocks, x, y, options):
        B200._check_q(name, rows, cols, batch, x, y)
        _check(1 <= count <= MAX_GROUP, f"B200 {name} requires 1 to {MAX_GROUP} matrices; got {count}")
        per = rows * (cols // 32) * block_bytes
        _check(count == 1 or per % 16 == 0, f"B200 {name} requires matrices of a multiple of 16 bytes; got {per}")
        _check(blocks.getSize() >= count * per, f"B200 {name}: weights smaller than count x rows x cols/32 x {block_bytes}")
        _check(y.getSize() >= count * batch * rows, f"B200 {name}: y smaller than count x batch x rows")
        _check(options is None or options.exact_int, f"B200 {name} computes in integer mode; exact_int must be set")
        return _desc(name, [count, rows, cols, batch, blocks, x, y], 6, tuning=options or B200Options(exact_int=True))

    @staticmethod
    def q8GemvBytesPacked(count, rows, cols, batch, blocks: ByteArray, x: FloatArray, y: FloatArray, options=None):  # noqa: N802
        """The grouped integer-mode mat-vec with its ``count`` (<= 32) equally shaped matrices back to back in ONE
        ByteArray, matrix m at byte m * rows * cols/32 * 34: seven arguments whatever the count, so that a whole
        decode step fits the 20-argument library-task interface (TaskGraph.java:886).  y is [count][batch][rows]."""
        return B200._packed("q8GemvBytesPacked", 34, count, rows, cols, batch, blocks, x, y, options)

    @staticmethod
    def q4GemvBytesPacked(count, rows, cols, batch, blocks: ByteArray, x: FloatArray, y: FloatArray, options=None):  # noqa: N802
        """Q4_0 twin of q8GemvBytesPacked (18-byte blocks)."""
        return B200._packed("q4GemvBytesPacked", 18, count, rows, cols, batch, blocks, x, y, options)

    @staticmethod
    def sgemm(m, n, k, alpha, a: FloatArray, b: FloatArray, beta, c: FloatArray):
        """C = alpha*A*B + beta*C, row-major; signature of Cutlass.cutlassSgemm (Cutlass.java:57-66)."""
        _check(m >= 0 and n >= 0 and k >= 0, f"B200 sgemm requires non-negative sizes; got m={m}, n={n}, k={k}")
        _check(a.getSize() >= m * k and b.getSize() >= k * n and c.getSize() >= m * n, "B200 sgemm: array too small")
        return _desc("sgemm", [m, n, k, float(alpha), a, b, float(beta), c], 7, read_write=(beta != 0.0))

    @staticmethod
    def hgemmF32(m, n, k, a: HalfFloatArray, b: HalfFloatArray, c: FloatArray):  # noqa: N802
        """C(fp32) = A(fp16) * B(fp16), row-major (operands of CuBlas.cublasGemmExFP16FP32, CuBlas.java:261-279)."""
        _check(m >= 0 and n >= 0 and k >= 0, f"B200 hgemmF32 requires non-negative sizes; got m={m}, n={n}, k={k}")
        _check(a.getSize() >= m * k and b.getSize() >= k * n and c.getSize() >= m * n, "B200 hgemmF32: array too small")
        return _desc("hgemmF32", [m, n, k, a, b, c], 5)

    # ---- fused epilogues, typed outputs, batches (tb200_gemm_ex) ---------------------------------------
    @staticmethod
    def _check_tc(name, m, n, k):
        _check(m >= 0 and n >= 0 and k >= 0, f"B200 {name} requires non-negative sizes; got m={m}, n={n}, k={k}")
        # the tensor-core tiles are fetched by TMA: rows of A and B must be multiples of 16 bytes (cf. Cutlass.java:68-77)
        _check(k % 8 == 0 and n % 8 == 0, f"B200 {name} requires k and n to be multiples of 8; got k={k}, n={n}")

    @staticmethod
    def hgemm(m, n, k, alpha, a: HalfFloatArray, b: HalfFloatArray, beta, d: HalfFloatArray):
        """D(fp16) = alpha*A*B + beta*D, fp32 accumulation; signature of Cutlass.cutlassHgemm (Cutlass.java:83-100)."""
        B200._check_tc("hgemm", m, n, k)
        _check(a.getSize() >= m * k and b.getSize() >= k * n and d.getSize() >= m * n, "B200 hgemm: array too small")
        return _desc("hgemm", [m, n, k, float(alpha), a, b, float(beta), d], 7, read_write=(beta != 0.0))

    @staticmethod
    def bgemm(m, n, k, alpha, a: BFloat16Array, b: BFloat16Array, beta, d: BFloat16Array):
        """bfloat16 twin of hgemm; signature of Cutlass.cutlassBgemm (Cutlass.java:102-117)."""
        B200._check_tc("bgemm", m, n, k)
        _check(a.getSize() >= m * k and b.getSize() >= k * n and d.getSize() >= m * n, "B200 bgemm: array too small")
        return _desc("bgemm", [m, n, k, float(alpha), a, b, float(beta), d], 7, read_write=(beta != 0.0))

    @staticmethod
    def _gemm_bias(act, m, n, k, a, b, bias, d):
        name = "gemmBias" + act
        B200._check_tc(name, m, n, k)
        _check(a.getSize() >= m * k and b.getSize() >= k * n and bias.getSize() >= n and d.getSize() >= m * n,
               f"B200 {name}: array too small")
        return _desc(name, [m, n, k, a, b, bias, d], 6)

    @staticmethod
    def gemmBiasRelu(m, n, k, a: HalfFloatArray, b: HalfFloatArray, bias: HalfFloatArray, d: HalfFloatArray):  # noqa: N802
        """D = relu(A*B + bias), bias broadcast over the rows; Cutlass.cutlassGemmBiasRelu (Cutlass.java:119-125)."""
        return B200._gemm_bias("Relu", m, n, k, a, b, bias, d)

    @staticmethod
    def gemmBiasGelu(m, n, k, a, b, bias, d):  # noqa: N802
        """Cutlass.cutlassGemmBiasGelu (Cutlass.java:127-135), erf form."""
        return B200._gemm_bias("Gelu", m, n, k, a, b, bias, d)

    @staticmethod
    def gemmBiasSilu(m, n, k, a, b, bias, d):  # noqa: N802
        return B200._gemm_bias("Silu", m, n, k, a, b, bias, d)

    @staticmethod
    def gemmBiasSigmoid(m, n, k, a, b, bias, d):  # noqa: N802
        return B200._gemm_bias("Sigmoid", m, n, k, a, b, bias, d)

    @staticmethod
    def gemmBiasTanh(m, n, k, a, b, bias, d):  # noqa: N802
        return B200._gemm_bias("Tanh", m, n, k, a, b, bias, d)

    @staticmethod
    def gemmBiasHardSwish(m, n, k, a, b, bias, d):  # noqa: N802
        return B200._gemm_bias("HardSwish", m, n, k, a, b, bias, d)

    @staticmethod
    def hgemmBatched(m, n, k, alpha, a: HalfFloatArray, b: HalfFloatArray, beta, d: HalfFloatArray, batchCount):  # noqa: N802,N803
        """batchCount independent fp16 GEMMs packed back to back; Cutlass.cutlassHgemmBatched (Cutlass.java:177-191)."""
        B200._check_tc("hgemmBatched", m, n, k)
        _check(batchCount >= 1, f"B200 hgemmBatched requires batchCount >= 1; got {batchCount}")
        _check(a.getSize() >= batchCount * m * k and b.getSize() >= batchCount * k * n and d.getSize() >= batchCount * m * n,
               "B200 hgemmBatched: array too small")
        return _desc("hgemmBatched", [m, n, k, float(alpha), a, b, float(beta), d, batchCount], 7, read_write=(beta != 0.0))

    # ---- decoder layer: what lies between its quantised products -------------------------------------------
    @staticmethod
    def _type(name, array, allowed=(FloatArray, HalfFloatArray, BFloat16Array)):
        for kind in allowed:
            if isinstance(array, kind):
                return ELEMENT_TYPES[kind]
        raise RuntimeError(f"[ERROR] B200 {name} does not take a {type(array).__name__}")

    @staticmethod
    def _norm(name, rows, cols, x, residual, weight, eps, fmt, group, q, scales):
        _check(rows >= 0 and 1 <= cols <= 1 << 30, f"B200 {name} requires rows >= 0 and 1 <= cols <= 2^30; got rows={rows}, cols={cols}")
        _check(fmt in QUANT_FORMATS, f"B200 {name} knows the formats {', '.join(QUANT_FORMATS)}; got {fmt}")
        _check(group in (0, 32, 64, 128), f"B200 {name} requires groups of 32, 64 or 128 columns, or 0 for a scale per row; got {group}")
        _check(0.0 <= eps < float("inf"), f"B200 {name} requires a finite eps >= 0; got {eps}")
        groups = -(-cols // group) if group else 1
        _check(x.getSize() >= rows * cols and weight.getSize() >= cols and q.getSize() >= rows * cols and scales.getSize() >= rows * groups
               and (residual is None or residual.getSize() >= rows * cols), f"B200 {name}: array too small")
        kind = B200._type(name, x)
        _check(residual is None or type(residual) is type(x), f"B200 {name}: x and residual differ in type")
        arrays = [x] if residual is None else [x, residual]
        params = [rows, cols, kind, *arrays, weight, float(eps), QUANT_FORMATS[fmt], group, q, scales]
        out = {len(params) - 2: Access.WRITE_ONLY, len(params) - 1: Access.WRITE_ONLY}
        if residual is not None:
            out[4] = Access.READ_WRITE
        return _desc(name, params, out)

    @staticmethod
    def rmsnormQuant(rows, cols, x, weight: FloatArray, eps, fmt, group, q, scales: FloatArray):  # noqa: N802
        """Root-mean-square norm of x's rows times ``weight`` as 8-bit values (``fmt``: int8, e4m3, e5m2) with an fp32
        scale per ``group`` columns (0: per row): the rows of A for igemm / fp8gemm, or the int8 blocks of the mat-vecs."""
        return B200._norm("rmsnormQuant", rows, cols, x, None, weight, eps, fmt, group, q, scales)

    @staticmethod
    def addRmsnormQuant(rows, cols, x, residual, weight: FloatArray, eps, fmt, group, q, scales: FloatArray):  # noqa: N802
        """rmsnormQuant of ``residual + x``; the sum, rounded to the arrays' type, replaces ``residual``."""
        return B200._norm("addRmsnormQuant", rows, cols, x, residual, weight, eps, fmt, group, q, scales)

    @staticmethod
    def pagedPlan(requests, pageSize, maxPages, maxTokens, cachedLens: IntArray, newLens: IntArray, freePages: IntArray,  # noqa: N802,N803
                  blockTable: IntArray, cuNew: IntArray, kvLens: IntArray, positions: IntArray, slots: LongArray, counts: IntArray):  # noqa: N803
        """Lays out a step of a paged cache: fresh pages from ``freePages`` into the table rows, and each token row's
        position and slot (tb200_paged_plan)."""
        _check(0 <= requests <= MAX_PLAN_REQUESTS, f"B200 pagedPlan requires 0 <= requests <= {MAX_PLAN_REQUESTS}; got {requests}")
        _check(pageSize >= 1 and maxPages >= 0 and maxPages * pageSize <= 1 << 30, "B200 pagedPlan requires pages of at least one position and at most 2^30 positions in a table row")
        _check(0 <= maxTokens <= 1 << 30, f"B200 pagedPlan requires 0 <= maxTokens <= 2^30; got {maxTokens}")
        _check(cachedLens.getSize() >= requests and newLens.getSize() >= requests and blockTable.getSize() >= requests * maxPages
               and cuNew.getSize() >= requests + 1 and kvLens.getSize() >= requests and positions.getSize() >= maxTokens
               and slots.getSize() >= maxTokens and counts.getSize() >= 4, "B200 pagedPlan: array too small")
        arrays = (blockTable, cuNew, kvLens, positions, slots, counts, cachedLens, newLens, freePages)
        _check(not any(out is other for i, out in enumerate(arrays[:6]) for other in arrays[i + 1:]), "B200 pagedPlan: an output and another array of the task are one array")
        params = [requests, pageSize, maxPages, maxTokens, freePages.getSize(), cachedLens, newLens, freePages, blockTable, cuNew, kvLens, positions, slots, counts]
        return _desc("pagedPlan", params, {8: Access.READ_WRITE} | {i: Access.WRITE_ONLY for i in range(9, 14)})

    @staticmethod
    def _cache(name, kvHeads, headDim, pageSize, kCache, vCache):  # noqa: N803
        _check(kvHeads >= 1 and headDim >= 1 and pageSize >= 1, f"B200 {name} requires kvHeads, headDim and pageSize >= 1")
        per = kvHeads * pageSize * headDim
        _check(kCache.getSize() == vCache.getSize() and kCache.getSize() % per == 0,
               f"B200 {name}: the caches are not both whole pages of kvHeads x pageSize x headDim = {per} elements")
        kind = B200._type(name, kCache, (HalfFloatArray, BFloat16Array))
        _check(type(vCache) is type(kCache), f"B200 {name}: the caches differ in type")
        return kind, kCache.getSize() // per

    @staticmethod
    def ropeAppend(tokens, qHeads, kvHeads, headDim, qkv, cosTable: FloatArray, sinTable: FloatArray, rotDim, interleaved, positions: IntArray,  # noqa: N802,N803
                   slots: LongArray, pageSize, q, kCache, vCache):  # noqa: N803
        """Rotates the queries and keys of projection rows [tokens][(qHeads + 2 kvHeads) headDim] by their positions,
        stores the queries in ``q`` and keys and values at their slots of the cache (tb200_rope_append)."""
        kind, pages = B200._cache("ropeAppend", kvHeads, headDim, pageSize, kCache, vCache)
        _check(tokens >= 0 and qHeads >= 0, f"B200 ropeAppend requires tokens >= 0 and qHeads >= 0; got {tokens}, {qHeads}")
        _check(0 <= rotDim <= headDim and rotDim % 2 == 0, f"B200 ropeAppend requires an even rotDim of at most headDim; got {rotDim}")
        rows = min(cosTable.getSize(), sinTable.getSize()) // (rotDim // 2) if rotDim else 0
        _check(qkv.getSize() >= tokens * (qHeads + 2 * kvHeads) * headDim and q.getSize() >= tokens * qHeads * headDim
               and positions.getSize() >= tokens and slots.getSize() >= tokens, "B200 ropeAppend: array too small")
        _check(type(q) is type(kCache), "B200 ropeAppend: q and the caches differ in type")
        params = [tokens, qHeads, kvHeads, headDim, B200._type("ropeAppend", qkv), qkv, cosTable, sinTable, rows, rotDim, int(bool(interleaved)), positions,
                  kind, q, pageSize, pages, slots, kCache, vCache]
        return _desc("ropeAppend", params, {i: Access.READ_WRITE for i in (13, 17, 18)})

    @staticmethod
    def pagedAttention(tokens, requests, maxNew, qHeads, kvHeads, headDim, q, cuNew: IntArray, kvLens: IntArray, blockTable: IntArray,  # noqa: N802,N803
                       pageSize, kCache, vCache, scale, window, out):  # noqa: N803
        """Causal attention of each request's new tokens over its pages of the cache, the new tokens included
        (tb200_paged_attention); ``window`` 0: no limit, ``maxNew`` 0: no bound known."""
        kind, pages = B200._cache("pagedAttention", kvHeads, headDim, pageSize, kCache, vCache)
        _check(tokens >= 0 and 1 <= requests <= 1 << 30 and maxNew >= 0 and window >= 0, "B200 pagedAttention requires tokens, maxNew, window >= 0 and 1 <= requests <= 2^30")
        _check(qHeads >= kvHeads and qHeads % kvHeads == 0, f"B200 pagedAttention requires qHeads to be a multiple of kvHeads; got {qHeads}, {kvHeads}")
        _check(headDim % 8 == 0 and headDim <= 256, f"B200 pagedAttention requires headDim to be a multiple of 8 up to 256; got {headDim}")
        _check(0.0 < scale < float("inf"), f"B200 pagedAttention requires a finite scale > 0; got {scale}")
        _check(blockTable.getSize() % requests == 0 and blockTable.getSize() // requests * pageSize <= 1 << 30, "B200 pagedAttention: the table is not [requests][maxPages], or a row holds over 2^30 positions")
        _check(q.getSize() >= tokens * qHeads * headDim and out.getSize() >= tokens * qHeads * headDim and cuNew.getSize() >= requests + 1
               and kvLens.getSize() >= requests, "B200 pagedAttention: array too small")
        _check(type(q) is type(kCache) and type(out) is type(kCache), "B200 pagedAttention: q, out and the caches differ in type")
        params = [tokens, requests, maxNew, qHeads, kvHeads, headDim, kind, q, cuNew, kvLens, blockTable, blockTable.getSize() // requests, pageSize, pages,
                  kCache, vCache, float(scale), window, out]
        return _desc("pagedAttention", params, {18: Access.READ_WRITE})
