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
// row lives in the registers of one block between the two reductions (sum of squares; the largest |y| of a group is a
// shuffle among the 4, 8 or 16 lanes that hold it, or a second block reduction for a scale a row), so nothing is read
// twice; rows that outgrow the registers (above 32768 columns) are read again instead.  A thread holds eight
// consecutive columns per 16-byte load, blocks are as wide as one such load of a row needs, and a grid of resident
// blocks walks the rows, which keeps the weight of rows of up to 8192 columns in registers.
#include <cuda_fp8.h>

#define TB200_OP_CLASS TB200_PREPARE_LAYER
#include "layer_common.cuh"

TB200_TU_STATUS(rmsnorm)

namespace tb200 {

struct NormArgs {
    const void *x;
    const void *residual;
    void *residual_out;
    const float *weight;
    uint8_t *q;
    float *scales;
    long long x_stride;
    float eps;
    int rows, cols, group, groups, format;
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

__device__ __forceinline__ uint32_t to_8bit(float y, float inv, int format) {
    if (inv == 0.0f) return 0;
    const float v = __fmul_rn(y, inv);
    if (format == TB200_Q_INT8)  // floor(v + 1/2) in the low byte of the sum with 1.5 * 2^23, rounded down
        return (uint32_t)__float_as_int(__fadd_rd(__fadd_rn(v, 0.5f), 12582912.0f)) & 0xFFu;
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, format == TB200_Q_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

// Block reduction of one value; every thread gets the result.  `red`: 33 floats, used by one reduction at a time.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    if (warps == 1) return v;
    __syncthreads();  // the last reduction's result has been read
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : 0.0f;  // |y| and squares: zero is neutral for both
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    return v;
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

template <int ALIGN>
__device__ __forceinline__ void store_q(const NormArgs &a, long long row, int c, const float (&y)[8], float inv) {
    uint8_t *p = a.q + row * a.cols + c;
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = to_8bit(y[j], inv, a.format);
    if constexpr (ALIGN != 0) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < a.cols) p[j] = (uint8_t)b[j];
    }
}

__device__ __forceinline__ float largest(const float (&y)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(y[j]));
    return m;
}
// over the lanes of a group: 8 columns a lane, so 4, 8 or 16 neighbouring lanes
__device__ __forceinline__ float group_max(float m, int group) {
    for (int o = 1; o < group / 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// NV pieces of eight columns a thread stay in registers: blockDim.x * 8 * NV >= cols.
template <class T, int ALIGN, int NV>
__global__ void __launch_bounds__(1024) rmsnorm_kernel(NormArgs a) {
    __shared__ float red[2][33];
    float w[8] = {};
    if (NV == 1 && threadIdx.x * 8 < a.cols) load_weight<ALIGN>(a, threadIdx.x * 8, w);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float h[NV][8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
            if (c < a.cols) {
                load_sum<T, ALIGN>(a, row, c, h[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
            if (c < a.cols) store_sum<T, ALIGN>(a, row, c, h[i]);
        }
        const float rstd = rsqrtf(__fdiv_rn(block_reduce<false>(sum, red[0]), (float)a.cols) + a.eps);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
            if (NV > 1 && c < a.cols) load_weight<ALIGN>(a, c, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * rstd * w[j];
            if (a.group == 0) top = max_nan(top, largest(h[i]));
        }
        float inv;
        if (a.group == 0) {
            const float scale = group_scale(block_reduce<true>(top, red[1]), a.format, inv);
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * 8;
            if (a.group != 0) {
                const float scale = group_scale(group_max(largest(h[i]), a.group), a.format, inv);
                if (c < a.cols && c % a.group == 0) a.scales[row * a.groups + c / a.group] = scale;
            }
            if (c < a.cols) store_q<ALIGN>(a, row, c, h[i], inv);
        }
    }
}

// Rows that outgrow the registers: the row is read once for its sum of squares, once more for a scale a row, and once
// for its values; residual_out is written in that last pass, so that it may be the residual (or x) itself.
template <class T, int ALIGN>
__global__ void __launch_bounds__(1024) rmsnorm_long_kernel(NormArgs a) {
    __shared__ float red[2][33];
    const int step = blockDim.x * 8, spans = (a.cols + step - 1) / step;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float sum = 0.0f, top = 0.0f, inv = 0.0f;
        for (int c = threadIdx.x * 8; c < a.cols; c += step) {
            float h[8];
            load_sum<T, ALIGN>(a, row, c, h);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[j], h[j], sum);
        }
        const float rstd = rsqrtf(__fdiv_rn(block_reduce<false>(sum, red[0]), (float)a.cols) + a.eps);
        if (a.group == 0) {
            for (int c = threadIdx.x * 8; c < a.cols; c += step) {
                float h[8], w[8];
                load_sum<T, ALIGN>(a, row, c, h);
                load_weight<ALIGN>(a, c, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = h[j] * rstd * w[j];
                top = max_nan(top, largest(h));
            }
            const float scale = group_scale(block_reduce<true>(top, red[1]), a.format, inv);
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
            for (int j = 0; j < 8; ++j) h[j] = h[j] * rstd * w[j];
            if (a.group != 0) {
                const float scale = group_scale(group_max(largest(h), a.group), a.format, inv);
                if (c < a.cols && c % a.group == 0) a.scales[row * a.groups + c / a.group] = scale;
            }
            if (c < a.cols) store_q<ALIGN>(a, row, c, h, inv);
        }
    }
}

template <class T, int ALIGN, int NV>
static int launch_norm(const NormArgs &a, int threads, const DeviceInfo *di, cudaStream_t s) {
    int st;
    if constexpr (NV > 0) {
        st = ensure_kernel<rmsnorm_kernel<T, ALIGN, NV>, 0>(di);
        if (st) return st;
        const int grid = (int)min((long long)a.rows, (long long)di->sm_count * (2048 / threads));
        rmsnorm_kernel<T, ALIGN, NV><<<grid, threads, 0, s>>>(a);
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
    const int threads = pieces >= 1024 ? 1024 : (pieces + 31) / 32 * 32;
    if (pieces <= 1024) return launch_norm<T, ALIGN, 1>(a, threads, di, s);
    if (pieces <= 2048) return launch_norm<T, ALIGN, 2>(a, (pieces + 63) / 64 * 32, di, s);
    if (pieces <= 4096) return launch_norm<T, ALIGN, 4>(a, (pieces + 127) / 128 * 32, di, s);
    return launch_norm<T, ALIGN, 0>(a, 1024, di, s);
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
    if (rows < 0 || cols < 1 || !valid_type(type) || x_stride < cols) return TB200_ERR_INVALID_ARG;
    if (format < TB200_Q_INT8 || format > TB200_Q_E5M2 || !(group == 0 || group == 32 || group == 64 || group == 128)) return TB200_ERR_INVALID_ARG;
    if (!(eps >= 0.0f) || eps > 3.402823466e38f) return TB200_ERR_INVALID_ARG;
    if (rows == 0) return TB200_OK;
    if (!x || !weight || !q || !scales) return TB200_ERR_INVALID_ARG;
    const uintptr_t b = (uintptr_t)type_bytes(type);
    if (!aligned_to(x, b) || (residual && !aligned_to(residual, b)) || (residual_out && !aligned_to(residual_out, b)) || !aligned_to(weight, 4) ||
        !aligned_to(scales, 4))
        return TB200_ERR_ALIGNMENT;
    int st;
    const DeviceInfo *di = device_info(&st);
    if (!di) return st;
    NormArgs a{x, residual, residual_out, weight, q, scales, x_stride, eps, rows, cols, group, group ? (cols + group - 1) / group : 1, format};
    cudaStream_t s = (cudaStream_t)stream;
    if (type == TB200_TYPE_F32) return dispatch_norm_align<float>(a, di, s);
    if (type == TB200_TYPE_F16) return dispatch_norm_align<__half>(a, di, s);
    return dispatch_norm_align<__nv_bfloat16>(a, di, s);
}
