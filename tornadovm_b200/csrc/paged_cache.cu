// The tables of a paged cache of keys and values, and the write of a step's rotated keys and values into it.
#define TB200_OP_CLASS TB200_PREPARE_LAYER
#include "layer_common.cuh"

TB200_TU_STATUS(paged_cache)

namespace tb200 {

// ---------------------------------------------------------------------------
// Block tables and slots from request lengths
// ---------------------------------------------------------------------------
// Two prefix sums over the requests (token rows, then fresh pages: the rows that fit decide the pages) and an
// expansion to token rows and table entries.  At the sizes of a step this is bound by latency, not by its few
// megabytes, so it is one launch: every block repeats the prefix sums over all requests (two coalesced arrays that L2
// serves, kept in shared memory: 8 bytes a request) and then writes its share of the rows and entries, found by a
// binary search in shared memory.  No block waits for another one, and no order of atomics reaches the result.
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_MAX_REQUESTS = 16384;

struct PlanArgs {
    const int32_t *cached_lens, *new_lens, *free_pages;
    int32_t *block_table, *cu_new, *kv_lens, *positions, *counts;
    int64_t *slots;
    int requests, page_size, max_pages, max_tokens, num_free;
};

// Exclusive prefix sums of one value a thread over the block, and the total, both held at `most` (a sum held at a limit is
// associative, and 32 bits take lengths whose true sum they could not).  `warp_sums`: 32 words.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned most, unsigned *warp_sums, unsigned &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    unsigned inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned w = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc = min(inc + w, most);
    }
    unsigned before = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) before = 0;
    __syncthreads();
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    unsigned winc = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned w = __shfl_up_sync(0xffffffffu, winc, o);
        if (lane >= o) winc = min(winc + w, most);
    }
    total = __shfl_sync(0xffffffffu, winc, 31);
    const unsigned others = __shfl_sync(0xffffffffu, winc, warp ? warp - 1 : 0);
    return warp ? min(others + before, most) : before;
}

// the last r with first[r] <= at (first[0] = 0 <= at; requests without rows share their successor's first row)
__device__ __forceinline__ int find_request(const int *first, int requests, int at) {
    int lo = 0, hi = requests - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= at) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// PER: requests a thread takes in the prefix sums (PER * blockDim.x >= requests), neighbours, in registers: their lengths
// are read once, all at the same time.
template <int PER>
__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(PlanArgs a) {
    extern __shared__ int plan_smem[];
    __shared__ unsigned warp_sums[32];
    int *first_row = plan_smem;                     // [requests + 1]
    int *first_page = plan_smem + a.requests + 1;   // [requests + 1]: fresh pages
    const int R = a.requests, P = a.page_size, r0 = threadIdx.x * PER;
    const int room = a.max_pages * P;
    const unsigned most = (unsigned)a.max_tokens;

    int c[PER], n[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        c[i] = r0 + i < R ? a.cached_lens[r0 + i] : 0;
        n[i] = r0 + i < R ? a.new_lens[r0 + i] : 0;
    }
    unsigned rows = 0, asked = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        c[i] = max(0, c[i]), n[i] = max(0, n[i]);
        asked = min(asked + (unsigned)n[i], 0x7FFFFFFFu);
        n[i] = min(n[i], max(0, room - min(c[i], room)));
        rows = min(rows + (unsigned)n[i], most);
    }
    unsigned total_rows, total_asked = 0, total_pages;
    unsigned at = block_scan(rows, most, warp_sums, total_rows);
    if (blockIdx.x == 0) block_scan(asked, 0x7FFFFFFFu, warp_sums, total_asked);  // only counts[] needs it
    unsigned pages = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = (int)at, e = (int)min(at + (unsigned)n[i], most);
        if (r0 + i < R) first_row[r0 + i] = b;
        at = (unsigned)e;
        n[i] = e > b ? (c[i] + (e - b) + P - 1) / P - (c[i] + P - 1) / P : 0;  // from here on its fresh pages
        pages += n[i];
    }
    const int used = (int)total_rows;
    int page = (int)block_scan(pages, 0x7FFFFFFFu, warp_sums, total_pages);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (r0 + i < R) first_page[r0 + i] = page;
        page += n[i];
    }
    if (threadIdx.x == 0) first_row[R] = used, first_page[R] = (int)total_pages;
    __syncthreads();

    if (blockIdx.x == 0) {
        for (int r = threadIdx.x; r < R; r += blockDim.x) {
            a.cu_new[r] = first_row[r];
            a.kv_lens[r] = max(0, a.cached_lens[r]) + first_row[r + 1] - first_row[r];
        }
        if (threadIdx.x == 0) {
            a.cu_new[R] = used;
            a.counts[0] = used;
            a.counts[1] = (int)total_asked;
            a.counts[2] = min((int)total_pages, a.num_free);
            a.counts[3] = (int)total_pages;
        }
    }
    const long long stride = (long long)gridDim.x * blockDim.x, me = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const bool wide = (((uintptr_t)a.positions | (uintptr_t)a.slots) & 15) == 0;
    // four rows in a line a thread: one search, one division and one table entry serve what they share
    for (long long t0 = 4 * me; t0 < a.max_tokens; t0 += 4 * stride) {
        int r = 0, position = 0, off = 0, end = -1, p[4];
        long long page_slot = -1, slot[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long t = t0 + i;
            p[i] = -1, slot[i] = -1;
            if (t >= used) continue;
            const bool next = t >= end;
            if (next) {
                if (end < 0) r = find_request(first_row, R, (int)t);
                else do ++r;
                    while (first_row[r + 1] <= t);
                end = first_row[r + 1];
                position = max(0, a.cached_lens[r]) + (int)t - first_row[r];
                off = position % P;
            }
            if (next || off == P) {
                if (!next) off = 0;
                // entries below `held` are not written by this launch; the others come from the free list directly
                const int index = position / P, held = (max(0, a.cached_lens[r]) + P - 1) / P, f = first_page[r] + index - held;
                const int entry = index < held ? a.block_table[(long long)r * a.max_pages + index] : f < a.num_free ? a.free_pages[f] : -1;
                page_slot = entry >= 0 ? (long long)entry * P : -1;
            }
            p[i] = position++;
            if (page_slot >= 0) slot[i] = page_slot + off;
            ++off;
        }
        if (wide && t0 + 4 <= a.max_tokens) {
            *reinterpret_cast<int4 *>(a.positions + t0) = make_int4(p[0], p[1], p[2], p[3]);
            *reinterpret_cast<longlong2 *>(a.slots + t0) = make_longlong2(slot[0], slot[1]);
            *reinterpret_cast<longlong2 *>(a.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t0 + i < a.max_tokens) a.positions[t0 + i] = p[i], a.slots[t0 + i] = slot[i];
        }
    }
    for (long long f = me; f < (long long)total_pages; f += stride) {
        const int r = find_request(first_page, R, (int)f);
        const int index = (max(0, a.cached_lens[r]) + P - 1) / P + (int)f - first_page[r];
        a.block_table[(long long)r * a.max_pages + index] = f < a.num_free ? a.free_pages[f] : -1;
    }
}

template <int PER>
static int launch_plan(const PlanArgs &a, int threads, const DeviceInfo *di, cudaStream_t s) {
    const int st = ensure_kernel<paged_plan_kernel<PER>>(di);
    if (st) return st;
    const int grid = max(1, min((a.max_tokens + 4 * threads - 1) / (4 * threads), di->sm_count));
    paged_plan_kernel<PER><<<grid, threads, 2 * (size_t)(a.requests + 1) * sizeof(int), s>>>(a);
    return check_launch();
}

// ---------------------------------------------------------------------------
// Rotary positions and the write into the cache
// ---------------------------------------------------------------------------
// Bound by memory: every element is read once and written once (4 bytes for 16-bit projections, 6 for fp32 ones).  A
// thread turns 16 elements of a head, eight and the eight that they pair with, as two wide loads and stores; threads
// next to one another hold the rest of the head, so that a warp moves whole lines of the projection row and of the
// cache (a head's row of a page is head_dim elements in one piece).  The angles of a row are read by all of its heads
// and come out of L1.  8192 rows of 48 heads of 128 into slots in random order: 49.5 us, 0.63 of the copy rate: a thread's
// source and angles are asked for behind its position, and its stores wait for the slot, three dependent latencies for 32
// bytes in and out; and with interleaved pairs a thread's two 16-byte pieces lie side by side, so that an access of a warp
// fills half of each sector it touches.  Four heads a thread, with the angles and the slot read once for all four, took 47 us.
struct AppendArgs {
    const void *q, *k, *v;
    const float *cos_table, *sin_table;
    const int32_t *positions;
    const int64_t *slots;
    void *q_out, *k_cache, *v_cache;
    long long q_stride, k_stride, v_stride, num_slots;
    int tokens, q_heads, kv_heads, head_dim, table_rows, rot_dim, interleaved, page_size;
};

// Destination of (token, head); false: nothing to write.
template <class C>
__device__ __forceinline__ bool append_target(const AppendArgs &a, int token, int head, int position, C *&dst) {
    if (head < a.q_heads) {
        dst = static_cast<C *>(a.q_out) + ((long long)token * a.q_heads + head) * a.head_dim;
        return true;
    }
    const long long slot = a.slots[token];
    if (slot < 0 || slot >= a.num_slots) return false;
    long long page;
    int off;
    if (slot <= 0x7FFFFFFFLL) {  // the 32-bit division is several times cheaper
        page = (int)slot / a.page_size;
        off = (int)slot - (int)page * a.page_size;
    } else {
        page = slot / a.page_size;
        off = (int)(slot - page * a.page_size);
    }
    int h = head - a.q_heads;
    void *cache = a.k_cache;
    if (h >= a.kv_heads) h -= a.kv_heads, cache = a.v_cache;
    dst = static_cast<C *>(cache) + ((page * a.kv_heads + h) * a.page_size + off) * a.head_dim;
    return true;
}

template <class T>
__device__ __forceinline__ const T *append_source(const AppendArgs &a, int token, int head) {
    if (head < a.q_heads) return static_cast<const T *>(a.q) + token * a.q_stride + (long long)head * a.head_dim;
    head -= a.q_heads;
    if (head < a.kv_heads) return static_cast<const T *>(a.k) + token * a.k_stride + (long long)head * a.head_dim;
    return static_cast<const T *>(a.v) + token * a.v_stride + (long long)(head - a.kv_heads) * a.head_dim;
}

// A row to turn, or nothing to do; a position beyond the tables is recorded.
__device__ __forceinline__ bool append_position(const AppendArgs &a, int token, int &position) {
    position = a.positions[token];
    if (position < 0) return false;
    if (position >= a.table_rows && a.rot_dim > 0) {
        g_device_status = TB200_ERR_INVALID_ARG;
        return false;
    }
    return true;
}

// head_dim and rot_dim multiples of 16, every row and array at ALIGN bytes
template <class T, class C, int ALIGN>
__global__ void __launch_bounds__(256) rope_append_kernel(AppendArgs a) {
    const int heads = a.q_heads + 2 * a.kv_heads, pieces = a.head_dim / 16, half = a.rot_dim / 2;
    const unsigned per_token = (unsigned)heads * pieces;
    const long long total = (long long)a.tokens * per_token, stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const int token = total <= 0x7FFFFFFFLL ? (int)((unsigned)i / per_token) : (int)(i / per_token);
        const unsigned in = (unsigned)(i - (long long)token * per_token);
        const int head = in / pieces, j = in - head * pieces;
        int position;
        C *dst;
        if (!append_position(a, token, position) || !append_target<C>(a, token, head, position, dst)) continue;
        const T *src = append_source<T>(a, token, head);
        const bool turn = head < a.q_heads + a.kv_heads && 16 * j < a.rot_dim;
        const int lo = turn && !a.interleaved ? 8 * j : 16 * j, hi = turn && !a.interleaved ? half + 8 * j : 16 * j + 8;
        float x[8], y[8];
        load8<ALIGN>(src + lo, x);
        load8<ALIGN>(src + hi, y);
        if (turn) {
            float c[8], s[8];
            load8<ALIGN>(a.cos_table + (long long)position * half + 8 * j, c);
            load8<ALIGN>(a.sin_table + (long long)position * half + 8 * j, s);
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = x[2 * e], r = x[2 * e + 1], u = y[2 * e], w = y[2 * e + 1];
                    x[2 * e] = p * c[e] - r * s[e], x[2 * e + 1] = p * s[e] + r * c[e];
                    y[2 * e] = u * c[4 + e] - w * s[4 + e], y[2 * e + 1] = u * s[4 + e] + w * c[4 + e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = x[e], r = y[e];
                    x[e] = p * c[e] - r * s[e], y[e] = p * s[e] + r * c[e];
                }
            }
        }
        store8<ALIGN>(dst + lo, x);
        store8<ALIGN>(dst + hi, y);
    }
}

// any even rot_dim, any head_dim, any element alignment: a thread turns one pair, or carries one element over
template <class T, class C>
__global__ void __launch_bounds__(256) rope_append_any_kernel(AppendArgs a) {
    const int heads = a.q_heads + 2 * a.kv_heads, half = a.rot_dim / 2, units = a.head_dim - half;
    const long long per_token = (long long)heads * units, total = a.tokens * per_token, stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const int token = (int)(i / per_token), in = (int)(i - token * per_token), head = in / units, j = in - head * units;
        int position;
        C *dst;
        if (!append_position(a, token, position) || !append_target<C>(a, token, head, position, dst)) continue;
        const T *src = append_source<T>(a, token, head);
        if (j >= half) {  // behind the rotated elements
            from_f32(dst[j + half], to_f32(src[j + half]));
            continue;
        }
        const int lo = a.interleaved ? 2 * j : j, hi = a.interleaved ? 2 * j + 1 : j + half;
        float x = to_f32(src[lo]), y = to_f32(src[hi]);
        if (head < a.q_heads + a.kv_heads) {
            const float c = a.cos_table[(long long)position * half + j], s = a.sin_table[(long long)position * half + j];
            const float p = x, r = y;
            x = p * c - r * s, y = p * s + r * c;
        }
        from_f32(dst[lo], x);
        from_f32(dst[hi], y);
    }
}

template <class T, class C>
static int dispatch_append(const AppendArgs &a, const DeviceInfo *di, cudaStream_t s) {
    auto all = [&](uintptr_t n) {
        const long long e = (long long)n / (long long)sizeof(T);  // rows keep the alignment
        return a.head_dim % 16 == 0 && a.rot_dim % 16 == 0 && aligned_to(a.q, n) && aligned_to(a.k, n) && aligned_to(a.v, n) && aligned_to(a.q_out, n) &&
               aligned_to(a.k_cache, n) && aligned_to(a.v_cache, n) && aligned_to(a.cos_table, n) && aligned_to(a.sin_table, n) &&
               a.q_stride % e == 0 && a.k_stride % e == 0 && a.v_stride % e == 0;
    };
    const long long heads = a.q_heads + 2LL * a.kv_heads;
    auto grid_of = [&](long long items) { return (unsigned)min((items + 255) / 256, (long long)di->sm_count * 64); };
    int st;
    if (all(16)) {
        st = ensure_kernel<rope_append_kernel<T, C, 16>, 0>(di);
        if (st) return st;
        rope_append_kernel<T, C, 16><<<grid_of(a.tokens * heads * (a.head_dim / 16)), 256, 0, s>>>(a);
    } else if (all(8)) {
        st = ensure_kernel<rope_append_kernel<T, C, 8>, 0>(di);
        if (st) return st;
        rope_append_kernel<T, C, 8><<<grid_of(a.tokens * heads * (a.head_dim / 16)), 256, 0, s>>>(a);
    } else {
        st = ensure_kernel<rope_append_any_kernel<T, C>, 0>(di);
        if (st) return st;
        rope_append_any_kernel<T, C><<<grid_of(a.tokens * heads * (a.head_dim - a.rot_dim / 2)), 256, 0, s>>>(a);
    }
    return check_launch();
}

}  // namespace tb200

using namespace tb200;

extern "C" int tb200_paged_plan(int requests, int page_size, int max_pages, int max_tokens, int num_free, const int32_t *cached_lens,
                                const int32_t *new_lens, const int32_t *free_pages, int32_t *block_table, int32_t *cu_new, int32_t *kv_lens,
                                int32_t *positions, int64_t *slots, int32_t *counts, tb200_stream_t stream) {
    if (requests < 0 || requests > PLAN_MAX_REQUESTS || page_size < 1 || max_pages < 0 || max_tokens < 0 || max_tokens > (1 << 30) || num_free < 0)
        return TB200_ERR_INVALID_ARG;
    if ((long long)max_pages * page_size > (1LL << 30)) return TB200_ERR_INVALID_ARG;
    if (!cu_new || !counts || (max_tokens > 0 && (!positions || !slots)) || (num_free > 0 && !free_pages)) return TB200_ERR_INVALID_ARG;
    if (requests > 0 && (!cached_lens || !new_lens || !kv_lens || (max_pages > 0 && !block_table))) return TB200_ERR_INVALID_ARG;
    const void *words[] = {cached_lens, new_lens, free_pages, block_table, cu_new, kv_lens, positions, counts};
    for (const void *p : words)
        if (!aligned_to(p, 4)) return TB200_ERR_ALIGNMENT;
    if (!aligned_to(slots, 8)) return TB200_ERR_ALIGNMENT;
    // Blocks read the lengths and the free list while others write: an output over another array would be a race.
    const long long R = requests;
    const struct { const void *at; long long bytes; } arrays[] = {{block_table, R * max_pages * 4}, {cu_new, (R + 1) * 4}, {kv_lens, R * 4}, {positions, max_tokens * 4LL},
                                                                   {slots, max_tokens * 8LL}, {counts, 16}, {cached_lens, R * 4}, {new_lens, R * 4}, {free_pages, num_free * 4LL}};
    for (int i = 0; i < 6; ++i)  // the outputs
        for (int j = i + 1; j < 9; ++j) {
            const uintptr_t a = (uintptr_t)arrays[i].at, b = (uintptr_t)arrays[j].at;
            if (arrays[i].bytes > 0 && arrays[j].bytes > 0 && a < b + arrays[j].bytes && b < a + arrays[i].bytes) return TB200_ERR_INVALID_ARG;
        }
    int st;
    const DeviceInfo *di = device_info(&st);
    if (!di) return st;
    PlanArgs a{cached_lens, new_lens, free_pages, block_table, cu_new, kv_lens, positions, counts, slots, requests, page_size, max_pages, max_tokens, num_free};
    cudaStream_t s = (cudaStream_t)stream;
    if (requests <= 256 && max_tokens <= 1024) return launch_plan<1>(a, 256, di, s);
    if (requests <= PLAN_THREADS) return launch_plan<1>(a, PLAN_THREADS, di, s);
    if (requests <= 4 * PLAN_THREADS) return launch_plan<4>(a, PLAN_THREADS, di, s);
    return launch_plan<16>(a, PLAN_THREADS, di, s);
}

extern "C" int tb200_rope_append(int tokens, int q_heads, int kv_heads, int head_dim, int in_type, const void *q, const void *k, const void *v,
                                 long long q_stride, long long k_stride, long long v_stride, const float *cos_table, const float *sin_table,
                                 int table_rows, int rot_dim, int interleaved, const int32_t *positions, int cache_type, void *q_out, int page_size,
                                 int num_pages, const int64_t *slots, void *k_cache, void *v_cache, tb200_stream_t stream) {
    if (tokens < 0 || q_heads < 0 || kv_heads < 1 || head_dim < 1 || head_dim > 65536 || q_heads > 65536 || kv_heads > 65536) return TB200_ERR_INVALID_ARG;
    if (!valid_type(in_type) || (cache_type != TB200_TYPE_F16 && cache_type != TB200_TYPE_BF16)) return TB200_ERR_INVALID_ARG;
    if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 || table_rows < 0 || page_size < 1 || num_pages < 0) return TB200_ERR_INVALID_ARG;
    if (((long long)q_heads + 2LL * kv_heads) * head_dim > 0x7FFFFFFFLL) return TB200_ERR_INVALID_ARG;
    if (q_stride < (long long)q_heads * head_dim || k_stride < (long long)kv_heads * head_dim || v_stride < (long long)kv_heads * head_dim)
        return TB200_ERR_INVALID_ARG;
    if (tokens == 0) return TB200_OK;
    if (!k || !v || !positions || !slots || (q_heads > 0 && (!q || !q_out)) || (num_pages > 0 && (!k_cache || !v_cache)) ||
        (rot_dim > 0 && (!cos_table || !sin_table)))
        return TB200_ERR_INVALID_ARG;
    const uintptr_t b = (uintptr_t)type_bytes(in_type);
    if (!aligned_to(q, b) || !aligned_to(k, b) || !aligned_to(v, b) || !aligned_to(q_out, 2) || !aligned_to(k_cache, 2) || !aligned_to(v_cache, 2) ||
        !aligned_to(cos_table, 4) || !aligned_to(sin_table, 4) || !aligned_to(positions, 4) || !aligned_to(slots, 8))
        return TB200_ERR_ALIGNMENT;
    // a thread's results may replace what it has read itself, and nothing else
    if (q_heads > 0 && q_out == q && (in_type != cache_type || (q_stride != (long long)q_heads * head_dim && tokens > 1))) return TB200_ERR_INVALID_ARG;
    if (num_pages > 0 && k_cache == v_cache) return TB200_ERR_INVALID_ARG;
    int st;
    const DeviceInfo *di = device_info(&st);
    if (!di) return st;
    AppendArgs a{q, k, v, cos_table, sin_table, positions, slots, q_out, k_cache, v_cache, q_stride, k_stride, v_stride,
                 (long long)num_pages * page_size, tokens, q_heads, kv_heads, head_dim, table_rows, rot_dim, interleaved, page_size};
    cudaStream_t s = (cudaStream_t)stream;
    if (cache_type == TB200_TYPE_F16) {
        if (in_type == TB200_TYPE_F32) return dispatch_append<float, __half>(a, di, s);
        if (in_type == TB200_TYPE_F16) return dispatch_append<__half, __half>(a, di, s);
        return dispatch_append<__nv_bfloat16, __half>(a, di, s);
    }
    if (in_type == TB200_TYPE_F32) return dispatch_append<float, __nv_bfloat16>(a, di, s);
    if (in_type == TB200_TYPE_F16) return dispatch_append<__half, __nv_bfloat16>(a, di, s);
    return dispatch_append<__nv_bfloat16, __nv_bfloat16>(a, di, s);
}
