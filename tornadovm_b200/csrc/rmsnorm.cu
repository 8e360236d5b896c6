// Root-mean-square norm of the residual stream with the residual's addition and an 8-bit output:
//
//     h = x + residual                       residual_out = h rounded to the arrays' type
//     y = h * (1 / sqrt(mean(h^2) + eps)) * weight
//     scale = max |y| / top                  over a group of 32, 64 or 128 columns, or over the row
//     q = y / scale                          int8: floor(. + 1/2), the rule of tb200_quantize_x; fp8: nearest even
//
// The norm is that of the unrounded fp32 sum h: residual_out's rounding is the only one before q.
//
// Bound by memory: x, residual, residual_out and q are each touched once (7 bytes an element for 16-bit arrays).  A
// row lives in the registers of one block across its reduction, so nothing is read twice.  The norm is one factor r for
// the whole row, so max |y| = r max |h * weight|: the sum of squares and the largest |h * weight| of a row are reduced
// together, behind one barrier, and a value costs one product with r / scale; the largest of a group is a shuffle among
// the 4, 8 or 16 lanes that hold it.  Rows that outgrow the registers (above 32768 columns) are read again instead.
//
// A thread holds eight consecutive columns per 16-byte load.  Few rows are a matter of latency: a thread for each eight
// columns.  Many rows are one of instructions and of bytes in flight: a thread for 16 columns, its weights in registers, and
// the next two rows of a block on their way to shared memory while it works on one (8192 x 4096 bf16 to e4m3: 42 us, 47 us
// with the weights read for each row, 75 us with a thread for each eight columns and no rows ahead).
#include <cuda_fp8.h>

#include <type_traits>

#define TB200_OP_CLASS TB200_PREPARE_LAYER
#include "layer_common.cuh"

namespace tb200 {

struct NormArgs {
    const void *x;
    const void *residual;
    void *residual_out;
    const float *weight;
    uint8_t *q;
    float *scales;
    long long x_stride;
    float eps, inv_cols;
    int rows, cols, group, group_shift, groups, format;
};

__device__ __forceinline__ float format_top(int format) { return format == TB200_Q_INT8 ? 127.0f : format == TB200_Q_E4M3 ? 448.0f : 57344.0f; }

// Scale and its reciprocal of a group whose largest |y| is `top_y`.  A group of zeros has the scale 1.  Where the
// quotient would be subnormal the smallest normal number stands in, so that the reciprocal stays finite.  A group that
// holds an infinity or a NaN has that as its scale and zeros as its values: every value it stands for is a NaN.
__device__ __forceinline__ float group_scale(float top_y, int format, float &inv) {
    const bool finite = top_y <= 3.402823466e38f;
    const float scale = top_y == 0.0f ? 1.0f : fmaxf(__fdiv_rn(top_y, format_top(format)), 1.17549435e-38f);
    inv = finite ? __fdiv_rn(1.0f, scale) : 0.0f;
    return finite ? scale : top_y;
}

// What turns eight values of h * weight into codes: the norm's factor over the scale, rounded once.  Where that product is
// beyond fp32 (the largest |h * weight| of the group is below top / 3.4e38, its y is not) the values become y first.
__device__ __forceinline__ float code_factor(float (&h)[8], float inv, float rstd) {
    const float factor = inv * rstd;
    if (factor <= 3.402823466e38f) return factor;
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] *= rstd;
    return inv;
}

// Eight values of h * weight, times `factor`, as eight bytes; inv 0: a group that is not finite.
__device__ __forceinline__ uint2 to_8bit(const float (&y)[8], float inv, float factor, int format) {
    if (inv == 0.0f) return make_uint2(0, 0);
    uint32_t w[2];
    if (format == TB200_Q_INT8) {  // floor(v + 1/2) in the low byte of the sum with 1.5 * 2^23, rounded down
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = (uint32_t)__float_as_int(__fadd_rd(__fadd_rn(__fmul_rn(y[4 * h + j], factor), 0.5f), 12582912.0f));
            w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 lo = make_float2(__fmul_rn(y[4 * h], factor), __fmul_rn(y[4 * h + 1], factor)), hi = make_float2(__fmul_rn(y[4 * h + 2], factor), __fmul_rn(y[4 * h + 3], factor));
            if (format == TB200_Q_E4M3)
                w[h] = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
            else
                w[h] = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E5M2) | (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E5M2) << 16;
        }
    }
    return make_uint2(w[0], w[1]);
}

// The sum of one value and the largest of another one over the block; every thread gets both.  `red`: 32 pairs that the
// reductions before and behind this one do not use, so that one barrier is enough.
__device__ __forceinline__ void block_reduce(float &sum, float &top, float2 *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o), top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (warps == 1) return;
    if (lane == 0) red[warp] = make_float2(sum, top);
    __syncthreads();
    const float2 v = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);  // squares and |h * w|: zero is neutral for both
    sum = v.x, top = v.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o), top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
}

// Columns c .. c + 7 of row `row` of h; columns past the row's end are zero.  ALIGN 0: element by element.
template <class T, int ALIGN>
__device__ __forceinline__ void load_sum(const NormArgs &a, long long row, int c, float (&h)[8]) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride + c;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.cols + c : nullptr;
    if constexpr (ALIGN != 0) {
        load8<ALIGN>(x, h);
        if (r) {
            float f[8];
            load8<ALIGN>(r, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] += f[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[j] = 0.0f;
            if (c + j < a.cols) h[j] = to_f32(x[j]) + (r ? to_f32(r[j]) : 0.0f);
        }
    }
}

// Columns c .. c + 7 of a row of an fp32 residual_out.
template <int ALIGN>
__device__ __forceinline__ void load_stored(const NormArgs &a, long long row, int c, float (&h)[8]) {
    const float *p = static_cast<const float *>(a.residual_out) + row * a.cols + c;
    if constexpr (ALIGN != 0) {
        load8<ALIGN>(p, h);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = c + j < a.cols ? p[j] : 0.0f;
    }
}

template <int ALIGN>
__device__ __forceinline__ void load_weight(const NormArgs &a, int c, float (&w)[8]) {
    if constexpr (ALIGN != 0) {
        load8<ALIGN>(a.weight + c, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = c + j < a.cols ? a.weight[c + j] : 0.0f;
    }
}

template <class T, int ALIGN>
__device__ __forceinline__ void store_sum(const NormArgs &a, long long row, int c, const float (&h)[8]) {
    if (!a.residual_out) return;
    T *p = static_cast<T *>(a.residual_out) + row * a.cols + c;
    if constexpr (ALIGN != 0) {
        store8<ALIGN>(p, h);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < a.cols) from_f32(p[j], h[j]);
    }
}

// the same from values that are rounded already
template <class T, int ALIGN>
__device__ __forceinline__ void store_rounded(const NormArgs &a, long long row, int c, const uint32_t (&w)[4]) {
    T *p = static_cast<T *>(a.residual_out) + row * a.cols + c;
    if constexpr (ALIGN == 16) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (ALIGN == 8) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2 *>(p + 4) = make_uint2(w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < a.cols) reinterpret_cast<uint16_t *>(p)[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
}

template <int ALIGN>
__device__ __forceinline__ void store_q(const NormArgs &a, long long row, int c, const float (&y)[8], float inv, float factor) {
    uint8_t *p = a.q + row * a.cols + c;
    const uint2 b = to_8bit(y, inv, factor, a.format);
    if constexpr (ALIGN != 0) {
        *reinterpret_cast<uint2 *>(p) = b;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < a.cols) p[j] = (uint8_t)((j < 4 ? b.x : b.y) >> (8 * (j & 3)));
    }
}

__device__ __forceinline__ float largest(const float (&y)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) m = max3_nan(m, fabsf(y[j]), fabsf(y[j + 1]));
    return m;
}
// over the lanes of a group: 8 columns a lane, so 4, 8 or 16 neighbouring lanes
__device__ __forceinline__ float group_max(float m, int group) {
    for (int o = 1; o < group / 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Rows whose squares, or whose products with the weight, leave fp32 while the norm does not.  With the norm's factor at 2^15
// and below, a product that is rounded as a subnormal moves y by 2^-135 at most, against scales of 2^-126 at least; above
// that, or with a sum of squares beyond fp32, the squares are summed at `unit`^4 of their size, and y is
// ((h * unit) * factor) * unit * weight, which leaves fp32 nowhere on the way.  Sums of two fp16 numbers are zero or between
// 2^-24 and 2^17: no such row.
template <class T>
__device__ __forceinline__ bool norm_is_far(float rstd) {
    return !std::is_same<T, __half>::value && __float_as_uint(rstd) - 1u >= __float_as_uint(0x1p15f);  // 0, above 2^15 or a NaN
}
// The whole row, by all threads of the block, read from memory: from an fp32 residual_out where that is `stored` (it holds
// the sum), else from x and the residual, which residual_out has not replaced yet.
template <class T, int ALIGN>
__device__ __forceinline__ void norm_far_row(const NormArgs &a, long long row, bool stored, float2 (*red)[32]) {
    const int step = blockDim.x * 8, mine = threadIdx.x * 8;
    const auto load = [&](int c, float (&h)[8]) {
        if (std::is_same<T, float>::value && stored) load_stored<ALIGN>(a, row, c, h);
        else load_sum<T, ALIGN>(a, row, c, h);
    };
    float unit = 1.0f, rstd = 0.0f, top = 0.0f, none = 0.0f, inv = 0.0f;
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
        float squares = 0.0f;
#pragma unroll 1
        for (int c = mine; c < a.cols; c += step) {
            float h[8];
            load(c, h);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = h[j] * unit * unit, squares = fmaf(h[j], h[j], squares);
        }
        __syncthreads();
        block_reduce(squares, none, red[turn]);
        rstd = rsqrtf(squares * a.inv_cols + a.eps * unit * unit * unit * unit);
        if (turn == 0) unit = !(squares <= 3.402823466e38f) ? 0x1p-48f : a.eps < 0x1p-100f && squares < 0x1p-80f ? 0x1p48f : 1.0f;
        if (unit == 1.0f) break;
    }
    if (a.group == 0) {
#pragma unroll 1
        for (int c = mine; c < a.cols; c += step) {
            float h[8], w[8];
            load(c, h);
            load_weight<ALIGN>(a, c, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = h[j] * unit * rstd * unit * w[j];
            top = max_nan(top, largest(h));
        }
        __syncthreads();
        block_reduce(none, top, red[0]);
        const float scale = group_scale(top, a.format, inv);
        if (threadIdx.x == 0) a.scales[row] = scale;
    }
#pragma unroll 1
    for (int c = mine; c - mine < a.cols; c += step) {  // whole warps take part in the groups' shuffles
        float h[8] = {}, w[8] = {};
        if (c < a.cols) {
            load(c, h);
            load_weight<ALIGN>(a, c, w);
            store_sum<T, ALIGN>(a, row, c, h);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = h[j] * unit * rstd * unit * w[j];
        if (a.group != 0) {
            const float scale = group_scale(group_max(largest(h), a.group), a.format, inv);
            if (c < a.cols && (c & (a.group - 1)) == 0) a.scales[row * a.groups + (c >> a.group_shift)] = scale;
        }
        if (c < a.cols) store_q<ALIGN>(a, row, c, h, inv, inv);
    }
}

__device__ __forceinline__ void norm_copy16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void norm_copy8(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// Rows far from 1 are remembered (a block has NORM_ROWS at most) and done again behind the others, where their code costs
// these no registers.  LATE: residual_out is x or the residual and of 16 bits, so that it waits until the row is known not to
// be such a one.
//
// NV pieces of eight columns a thread stay in registers: blockDim.x * 8 * NV >= cols.  STAGES > 0: the block's next rows are
// under way to shared memory while it works on this one (a thread copies what it will read itself, so no barrier orders
// them): a row's chain of loads, two reductions and stores would leave the memory idle otherwise.
constexpr int NORM_ROWS = 32;
template <class T, int ALIGN, int NV, int STAGES, bool LATE>
__global__ void __launch_bounds__(NV <= 2 && STAGES == 0 ? 1024 : 512) rmsnorm_kernel(NormArgs a) {
    constexpr int UNITS = sizeof(T) / 2;  // 16-byte pieces of eight columns
    extern __shared__ __align__(16) uint4 norm_stage[];  // [stage][x, residual][piece][unit][thread]
    __shared__ float2 red[2][32];  // in turn for odd and even rows
    // Weights stay in registers where there is room.  With many rows they are held at 2^24 of their size: inv is 2^126 at
    // most and the factor of a row near 1 is 2^15, so that inv times 2^-24 of the factor is finite for any group.
    constexpr bool KEEP = NV == 1 || STAGES > 0;
    constexpr float LIFT = STAGES > 0 ? 0x1p24f : 1.0f;
    float w[KEEP ? NV : 1][8] = {};
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
            if (c < a.cols) load_weight<ALIGN>(a, c, w[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[i][j] *= LIFT;
        }
    }
    auto slot = [&](int stage, int array, int i, int u) { return norm_stage + (((stage * 2 + array) * NV + i) * UNITS + u) * blockDim.x + threadIdx.x; };
    auto prefetch = [&](long long row, int stage) {
        if (row < a.rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * blockDim.x + threadIdx.x) * 8;
                if (c >= a.cols) continue;
#pragma unroll
                for (int array = 0; array < 2; ++array) {
                    if (array == 1 && !a.residual) continue;
                    const T *p = array == 0 ? static_cast<const T *>(a.x) + row * a.x_stride + c : static_cast<const T *>(a.residual) + row * a.cols + c;
#pragma unroll
                    for (int u = 0; u < UNITS; ++u) {
                        const char *src = reinterpret_cast<const char *>(p) + 16 * u;
                        char *dst = reinterpret_cast<char *>(slot(stage, array, i, u));
                        if constexpr (ALIGN == 16) norm_copy16(dst, src);
                        else norm_copy8(dst, src), norm_copy8(dst + 8, src + 8);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    [[maybe_unused]] auto staged_sum = [&](int stage, int i, float (&h)[8]) {
        uint4 raw[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) raw[u] = *slot(stage, 0, i, u);
        load8<16>(reinterpret_cast<const T *>(raw), h);
        if (a.residual) {
            float f[8];
#pragma unroll
            for (int u = 0; u < UNITS; ++u) raw[u] = *slot(stage, 1, i, u);
            load8<16>(reinterpret_cast<const T *>(raw), f);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] += f[j];
        }
    };
    if constexpr (STAGES > 0)
        for (int k = 0; k < STAGES - 1; ++k) prefetch(blockIdx.x + (long long)k * gridDim.x, k);
    int stage = 0, turn = 0;
    unsigned far_rows = 0, this_row = 1;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float h[NV][8], sum = 0.0f;
        if constexpr (STAGES > 0) {
            prefetch(row + (long long)(STAGES - 1) * gridDim.x, stage == 0 ? STAGES - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
            if (c >= a.cols) {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
                continue;
            }
            if constexpr (STAGES > 0) {
                staged_sum(stage, i, h[i]);
            } else {
                load_sum<T, ALIGN>(a, row, c, h[i]);
            }
        }
        float top = 0.0f, part[NV];
        [[maybe_unused]] uint32_t rounded[LATE && STAGES == 0 ? NV : 1][4];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
            if (c < a.cols) {
                if (!LATE) store_sum<T, ALIGN>(a, row, c, h[i]);
                if (!KEEP) load_weight<ALIGN>(a, c, w[0]);
            }
            if constexpr (LATE && STAGES == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) rounded[i][j] = pack2(h[i][2 * j], h[i][2 * j + 1], T());
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= w[KEEP ? i : 0][j];
            part[i] = largest(h[i]);
            top = max_nan(top, part[i]);
        }
        turn ^= 1;
        block_reduce(sum, top, red[turn]);
        const float rstd = rsqrtf(sum * a.inv_cols + a.eps);
        const bool far = norm_is_far<T>(rstd);
        if (far) far_rows |= this_row;
        this_row <<= 1;
        const float of_product = rstd * (1.0f / LIFT);
        float inv;
        if (a.group == 0) {
            const float scale = group_scale(top * of_product, a.format, inv);
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
            if (a.group != 0) {
                const float scale = group_scale(group_max(part[i], a.group) * of_product, a.format, inv);
                if (c < a.cols && (c & (a.group - 1)) == 0) a.scales[row * a.groups + (c >> a.group_shift)] = scale;
            }
            if (c < a.cols) {
                if constexpr (LATE && STAGES == 0)
                    if (!far) store_rounded<T, ALIGN>(a, row, c, rounded[i]);
                const float factor = STAGES > 0 ? inv * of_product : code_factor(h[i], inv, rstd);
                store_q<ALIGN>(a, row, c, h[i], inv, factor);
                if constexpr (LATE && STAGES > 0) {  // from shared memory once more: it does not fit the registers beside the weights
                    if (!far) {
                        staged_sum(stage, i, h[i]);
                        store_sum<T, ALIGN>(a, row, c, h[i]);
                    }
                }
            }
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    if constexpr (!std::is_same<T, __half>::value)
        for (; far_rows; far_rows &= far_rows - 1) norm_far_row<T, ALIGN>(a, blockIdx.x + (long long)(__ffs(far_rows) - 1) * gridDim.x, a.residual_out, red);
}

// Rows that outgrow the registers: the row is read once for its sum of squares and its largest value, and once for its
// values; residual_out is written in that second pass, so that it may be the residual (or x) itself.
template <class T, int ALIGN>
__global__ void __launch_bounds__(1024) rmsnorm_long_kernel(NormArgs a) {
    __shared__ float2 red[2][32], far_red[2][32];
    int turn = 0;
    const int step = blockDim.x * 8, spans = (a.cols + step - 1) / step;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float sum = 0.0f, top = 0.0f, inv = 0.0f;
        for (int c = threadIdx.x * 8; c < a.cols; c += step) {
            float h[8], w[8];
            load_sum<T, ALIGN>(a, row, c, h);
            load_weight<ALIGN>(a, c, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[j], h[j], sum), h[j] *= w[j];
            top = max_nan(top, largest(h));
        }
        turn ^= 1;
        block_reduce(sum, top, red[turn]);
        const float rstd = rsqrtf(sum * a.inv_cols + a.eps);
        if (norm_is_far<T>(rstd)) {  // nothing of the row has been stored yet
            norm_far_row<T, ALIGN>(a, row, false, far_red);
            continue;
        }
        if (a.group == 0) {
            const float scale = group_scale(top * rstd, a.format, inv);
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
        for (int s = 0; s < spans; ++s) {  // whole warps take part in the groups' shuffles
            const int c = s * step + threadIdx.x * 8;
            float h[8] = {}, w[8] = {};
            if (c < a.cols) {
                load_sum<T, ALIGN>(a, row, c, h);
                load_weight<ALIGN>(a, c, w);
                store_sum<T, ALIGN>(a, row, c, h);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] *= w[j];
            if (a.group != 0) {
                const float scale = group_scale(group_max(largest(h), a.group) * rstd, a.format, inv);
                if (c < a.cols && (c & (a.group - 1)) == 0) a.scales[row * a.groups + (c >> a.group_shift)] = scale;
            }
            if (c < a.cols) {
                const float factor = code_factor(h, inv, rstd);
                store_q<ALIGN>(a, row, c, h, inv, factor);
            }
        }
    }
}

template <class T, int ALIGN, int NV, int STAGES>
static int launch_norm(const NormArgs &a, int threads, const DeviceInfo *di, cudaStream_t s) {
    const size_t smem = (size_t)STAGES * 2 * NV * sizeof(T) * 8 * threads;
    int st;
    if constexpr (NV > 0) {
        constexpr int FLAGS = STAGES ? KERNEL_OPTIN_SMEM | KERNEL_MAX_CARVEOUT : 0;
        constexpr bool CAN_BE_LATE = std::is_same<T, __nv_bfloat16>::value;
        const bool late = CAN_BE_LATE && a.residual_out && (a.residual_out == a.residual || a.residual_out == a.x);
        st = late ? ensure_kernel<rmsnorm_kernel<T, ALIGN, NV, STAGES, CAN_BE_LATE>, FLAGS>(di) : ensure_kernel<rmsnorm_kernel<T, ALIGN, NV, STAGES, false>, FLAGS>(di);
        if (st) return st;
        const long long resident = min((long long)a.rows, STAGES ? max(1LL, (long long)di->sm_count * (long long)(200 * 1024 / (smem + 1024))) : (long long)di->sm_count * (2048 / threads));
        // whole waves of blocks of up to NORM_ROWS rows (20000 x 14336 bf16: 574 us in one wave, 669 us in 2.1 of them)
        const int grid = (int)min((long long)a.rows, resident * ((a.rows + resident * NORM_ROWS - 1) / (resident * NORM_ROWS)));
        if (late) rmsnorm_kernel<T, ALIGN, NV, STAGES, CAN_BE_LATE><<<grid, threads, smem, s>>>(a);
        else rmsnorm_kernel<T, ALIGN, NV, STAGES, false><<<grid, threads, smem, s>>>(a);
    } else {
        st = ensure_kernel<rmsnorm_long_kernel<T, ALIGN>, 0>(di);
        if (st) return st;
        const int grid = (int)min((long long)a.rows, (long long)di->sm_count * 2);
        rmsnorm_long_kernel<T, ALIGN><<<grid, threads, 0, s>>>(a);
    }
    return check_launch();
}

template <class T, int ALIGN>
static int dispatch_norm(const NormArgs &a, const DeviceInfo *di, cudaStream_t s) {
    const int pieces = (a.cols + 7) / 8;
    if (pieces <= 1024 && a.rows < 2 * di->sm_count) return launch_norm<T, ALIGN, 1, 0>(a, (pieces + 31) / 32 * 32, di, s);
    if constexpr (ALIGN != 0) {
        // three stages of rows of up to 8192 16-bit columns leave room for two blocks an SM at least
        if (pieces <= 1024 * 2 / (int)sizeof(T)) return launch_norm<T, ALIGN, 2, 3>(a, (pieces + 63) / 64 * 32, di, s);
    }
    if (pieces <= 2048) return launch_norm<T, ALIGN, 2, 0>(a, (pieces + 63) / 64 * 32, di, s);
    if (pieces <= 4096) return launch_norm<T, ALIGN, 8, 0>(a, (pieces + 255) / 256 * 32, di, s);
    return launch_norm<T, ALIGN, 0, 0>(a, 1024, di, s);
}

template <class T>
static int dispatch_norm_align(const NormArgs &a, const DeviceInfo *di, cudaStream_t s) {
    const bool rows8 = a.cols % 8 == 0 && a.x_stride % 8 == 0;
    auto all = [&](uintptr_t n) {
        return aligned_to(a.x, n) && (!a.residual || aligned_to(a.residual, n)) && (!a.residual_out || aligned_to(a.residual_out, n)) && aligned_to(a.weight, n);
    };
    if (rows8 && aligned_to(a.q, 8) && all(16)) return dispatch_norm<T, 16>(a, di, s);
    if (rows8 && aligned_to(a.q, 8) && all(8)) return dispatch_norm<T, 8>(a, di, s);
    return dispatch_norm<T, 0>(a, di, s);
}

}  // namespace tb200

using namespace tb200;

extern "C" int tb200_rmsnorm_quant(int rows, int cols, int type, const void *x, long long x_stride, const void *residual, void *residual_out,
                                   const float *weight, float eps, int format, int group, uint8_t *q, float *scales, tb200_stream_t stream) {
    // a thread's next column, up to 8192 behind the last one, is still a 32-bit number
    if (rows < 0 || cols < 1 || cols > (1 << 30) || !valid_type(type) || x_stride < cols) return TB200_ERR_INVALID_ARG;
    if (format < TB200_Q_INT8 || format > TB200_Q_E5M2 || !(group == 0 || group == 32 || group == 64 || group == 128)) return TB200_ERR_INVALID_ARG;
    if (!(eps >= 0.0f) || eps > 3.402823466e38f) return TB200_ERR_INVALID_ARG;
    if (rows == 0) return TB200_OK;
    if (!x || !weight || !q || !scales || (residual_out == x && x_stride != cols && rows > 1)) return TB200_ERR_INVALID_ARG;
    const uintptr_t b = (uintptr_t)type_bytes(type);
    if (!aligned_to(x, b) || (residual && !aligned_to(residual, b)) || (residual_out && !aligned_to(residual_out, b)) || !aligned_to(weight, 4) ||
        !aligned_to(scales, 4))
        return TB200_ERR_ALIGNMENT;
    int st;
    const DeviceInfo *di = device_info(&st);
    if (!di) return st;
    NormArgs a{x, residual, residual_out, weight, q, scales, x_stride, eps, 1.0f / (float)cols, rows, cols, group, group ? __builtin_ctz(group) : 0, group ? (cols + group - 1) / group : 1, format};
    cudaStream_t s = (cudaStream_t)stream;
    if (type == TB200_TYPE_F32) return dispatch_norm_align<float>(a, di, s);
    if (type == TB200_TYPE_F16) return dispatch_norm_align<__half>(a, di, s);
    return dispatch_norm_align<__nv_bfloat16>(a, di, s);
}
