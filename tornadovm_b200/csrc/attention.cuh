// Paged attention: arguments, the division of the work over the blocks, and the joining of split rows.
//
// A call's work is a list of items (request, kv head, tile of query rows), each a run of key tiles.  The query rows of a
// request for one kv head are its new tokens times the query heads that share the kv head, tokens first: row =
// token * group + head of the group, so a decoding request has `group` rows and short chunks still fill a tile.  All
// key tiles of all items, in order, are divided evenly over the grid: a block starts and ends inside an item, at most
// two of its items are shared with neighbouring blocks, and every block has the same number of tiles whatever the
// lengths are.  Lengths live on the device, so each block repeats the prefix sum over the requests by itself (reads
// that L2 serves), and no block waits for another.
//
// An item counts as its key tiles and ITEM tiles more that stand for what it costs besides; these come first and have no
// keys, so a block that ends inside them leaves the item to the next block altogether.
//
// A block that holds a whole item normalises and stores it.  Otherwise it leaves the running maximum, sum and
// unnormalised output of its part in the workspace, in one of two places that belong to the block: 0 for an item that
// an earlier block began, 1 for an item that it begins itself.  A second kernel joins the parts in the order of blocks.
#pragma once

#include "layer_common.cuh"

namespace tb200 {

struct AttnArgs {
    const void *q, *k_cache, *v_cache;
    const int32_t *cu_new, *kv_lens, *block_table;
    void *out;
    float *parts;        // [grid][2] parts of output, reference and sum: [rows of a tile][pitch] in attention.cu, [columns][rows] in attention_tc.cu
    int4 *joins;         // [grid]: item that the block begins and another one ends: (request, kv head, row tile, last block), x < 0: none
    long long q_stride, out_stride;
    float scale_log2;    // scale * log2(e): probabilities are powers of two
    int tokens, requests, q_heads, kv_heads, group, head_dim, max_pages, page_size, num_pages, window, page_shift;  // page_shift: log2, or -1
    int whole;  // items are not split: every gridDim.x-th (request, kv head) belongs to a block
};

struct AttnRequest {
    int first, rows, new_tokens;  // first token row; rows for one kv head; tokens in this step
    int kv_len, visible;          // cached + new; keys that have a place in the table
};

// Lengths as they are used: whatever the arrays hold, nothing outside [0, tokens) and the table row is touched.
__device__ __forceinline__ AttnRequest attn_request(const AttnArgs &a, int r) {
    AttnRequest q;
    const int b = min(max(a.cu_new[r], 0), a.tokens), e = min(max(a.cu_new[r + 1], b), a.tokens);
    q.first = b, q.new_tokens = e - b;
    const long long rows = (long long)q.new_tokens * a.group;
    q.rows = (int)rows;
    q.kv_len = min(max(a.kv_lens[r], 0), 1 << 30);
    q.visible = (int)min((long long)q.kv_len, (long long)a.max_pages * a.page_size);
    return q;
}

// Key tiles [first, first + count) that a tile of query rows sees; one (empty) tile where it sees none, so that every
// row is written by somebody.
template <int ROWS, int KEYS>
__device__ __forceinline__ void attn_key_tiles(const AttnArgs &a, const AttnRequest &q, int tile, int &first, int &count) {
    const int row0 = tile * ROWS, row1 = min(q.rows, row0 + ROWS) - 1;
    const int base = q.kv_len - q.new_tokens;
    const int lowest = base + row0 / a.group, highest = min(base + row1 / a.group, q.visible - 1);
    first = a.window > 0 ? max(0, lowest - a.window + 1) / KEYS : 0;
    const int last = highest < 0 ? -1 : highest / KEYS;
    count = max(1, last - first + 1);
}

// Key tiles of all row tiles of a request for one head: by one thread, and by a warp.
template <int ROWS, int KEYS, int ITEM>
__device__ __forceinline__ long long attn_head_tiles(const AttnArgs &a, const AttnRequest &q) {
    long long n = 0;
    for (int t = 0; (long long)t * ROWS < q.rows; ++t) {
        int first, count;
        attn_key_tiles<ROWS, KEYS>(a, q, t, first, count);
        n += ITEM + count;
    }
    return n;
}
template <int ROWS, int KEYS, int ITEM>
__device__ __forceinline__ long long attn_head_tiles_warp(const AttnArgs &a, const AttnRequest &q) {
    long long n = 0;
    for (int t = threadIdx.x & 31; (long long)t * ROWS < q.rows; t += 32) {
        int first, count;
        attn_key_tiles<ROWS, KEYS>(a, q, t, first, count);
        n += ITEM + count;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

// First tile of block `b` of `blocks` over `total` tiles, and the block that has tile `u`.  blocks <= total: every block
// between two that share an item has a part of it.
// (64-bit divisions are subroutines of some hundred instructions: calls of less than 2^32 tiles, which all are, avoid them.)
__device__ __forceinline__ long long attn_div(long long n, long long d) {
    return ((n | d) >> 32) == 0 ? (long long)((unsigned)n / (unsigned)d) : n / d;
}
__device__ __forceinline__ long long attn_block_begin(long long total, int b, int blocks) {
    const long long each = attn_div(total, blocks);
    return each * b + (unsigned)(total - each * blocks) * (unsigned)b / (unsigned)blocks;
}
__device__ __forceinline__ int attn_block_of(long long total, int blocks, long long u) {
    int b = (int)min((long long)blocks - 1, attn_div(u * blocks, total));  // exact up to rounding: step to the block that has it
    while (b > 0 && attn_block_begin(total, b, blocks) > u) --b;
    while (b + 1 < blocks && attn_block_begin(total, b + 1, blocks) <= u) ++b;
    return b;
}

struct AttnStart {
    long long total, begin, end;  // tiles of the call; this block's
    int blocks;                   // blocks that have tiles
    int request;                  // request in which the block begins
    long long request_begin;      // first tile of that request
};

// Run by all threads of the block; `scan`: 32 words of shared memory.  Few requests are counted by a warp each (a long
// prompt has hundreds of row tiles), many by a thread each.
template <int THREADS, int ROWS, int KEYS, int ITEM>
__device__ __forceinline__ void attn_find_start(const AttnArgs &a, AttnStart *out, long long *scan) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool few = a.requests <= 32;
    long long mine = 0;
    int r0 = 0, r1 = 0;
    if (few) {
        for (int r = warp; r < a.requests; r += THREADS / 32) {
            const long long n = attn_head_tiles_warp<ROWS, KEYS, ITEM>(a, attn_request(a, r)) * a.kv_heads;
            if (lane == 0) scan[r] = n;
        }
        __syncthreads();
        mine = lane < a.requests ? scan[lane] : 0;  // every warp: a request per lane
    } else {
        const int per = (a.requests + THREADS - 1) / THREADS;
        r0 = min(a.requests, (int)threadIdx.x * per), r1 = min(a.requests, r0 + per);
        for (int r = r0; r < r1; ++r) mine += attn_head_tiles<ROWS, KEYS, ITEM>(a, attn_request(a, r)) * a.kv_heads;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long w = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += w;
    }
    long long before = inc - mine, total = 0;
    if (few) {
        total = __shfl_sync(0xffffffffu, inc, 31);
    } else {
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += scan[w];
            total += scan[w];
        }
    }
    const int blocks = (int)max(1LL, min((long long)gridDim.x, total)), b = blockIdx.x;
    const long long begin = b < blocks ? attn_block_begin(total, b, blocks) : total, end = b < blocks ? attn_block_begin(total, b + 1, blocks) : total;
    if (threadIdx.x == 0) out->total = total, out->begin = begin, out->end = end, out->blocks = blocks;
    if (begin < end && before <= begin && begin < before + mine && (warp == 0 || !few)) {  // one thread
        long long at = before;
        int r = few ? lane : r0;
        for (; !few && r < r1; ++r) {
            const long long n = attn_head_tiles<ROWS, KEYS, ITEM>(a, attn_request(a, r)) * a.kv_heads;
            if (begin < at + n) break;
            at += n;
        }
        out->request = r, out->request_begin = at;
    }
    __syncthreads();
}

// The block's walk over its items.
template <int ROWS, int KEYS, int ITEM>
struct AttnWalk {
    AttnRequest q;
    int request, head, tile;    // the item
    int first, count;           // its key tiles
    int from, to;               // this block's of them: [from, to) of [0, count)
    long long item_begin;       // the item's first tile in the call

    // The first item of which the block has key tiles, false if there is none; run by whole warps, whose lanes look at 32
    // row tiles at a time.
    __device__ __forceinline__ bool seek(const AttnArgs &a, const AttnStart &s) {
        const int lane = threadIdx.x & 31;
        request = s.request;
        q = attn_request(a, request);
        const long long per_head = attn_head_tiles_warp<ROWS, KEYS, ITEM>(a, q);
        const long long in = s.begin - s.request_begin;
        head = (int)attn_div(in, per_head);
        item_begin = s.request_begin + head * per_head;
        for (tile = 0; (long long)tile * ROWS < q.rows; tile += 32) {
            int f = 0, n = 0;
            if ((long long)(tile + lane) * ROWS < q.rows) attn_key_tiles<ROWS, KEYS>(a, q, tile + lane, f, n);
            const int units = (long long)(tile + lane) * ROWS < q.rows ? ITEM + n : 0;
            long long inc = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, s.begin < item_begin + inc);
            if (past) {
                const int l = __ffs(past) - 1;
                tile += l, item_begin += __shfl_sync(0xffffffffu, inc - units, l);
                first = __shfl_sync(0xffffffffu, f, l), count = __shfl_sync(0xffffffffu, n, l);
                break;
            }
            item_begin += __shfl_sync(0xffffffffu, inc, 31);
        }
        return clip(s) || next(a, s);
    }
    __device__ __forceinline__ bool clip(const AttnStart &s) {
        from = (int)max(0LL, s.begin - item_begin - ITEM);
        to = (int)min((long long)count, s.end - item_begin - ITEM);
        return from < to;
    }
    // The next item; false when the block's tiles are done.
    __device__ __forceinline__ bool next(const AttnArgs &a, const AttnStart &s) {
        if (item_begin + ITEM + count >= s.end) return false;
        item_begin += ITEM + count;
        ++tile;
        if ((long long)tile * ROWS >= q.rows) {
            tile = 0;
            if (++head >= a.kv_heads) {
                head = 0;
                do {
                    if (++request >= a.requests) return false;  // lengths that changed meanwhile must not lead past the arrays
                    q = attn_request(a, request);
                } while (q.rows == 0);
            }
        }
        attn_key_tiles<ROWS, KEYS>(a, q, tile, first, count);
        return clip(s);  // only the block's last item can be without key tiles of it
    }
    // The walk over whole items: row tiles of (request, kv head) `pair`, of every gridDim.x-th pair from there on.
    int pair;
    __device__ __forceinline__ bool first_whole(const AttnArgs &a) {
        pair = (int)blockIdx.x - (int)gridDim.x, tile = 0, q.rows = 0;
        return next_whole(a);
    }
    __device__ __forceinline__ bool next_whole(const AttnArgs &a) {
        ++tile;
        while ((long long)tile * ROWS >= q.rows) {
            if ((long long)pair + gridDim.x >= (long long)a.requests * a.kv_heads) return false;
            pair += gridDim.x, tile = 0;
            request = pair / a.kv_heads, head = pair - request * a.kv_heads;
            q = attn_request(a, request);
        }
        attn_key_tiles<ROWS, KEYS>(a, q, tile, first, count);
        from = 0, to = count;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return from == 0 && to == count; }
};

// Joins the parts of the items that more than one block worked on.  Block x takes the item that block x of the main
// kernel began and another one ended; the rows of the tile are spread over gridDim.y.  A long context has hundreds of
// parts, so their maxima and sums are read side by side first, a part a thread, and become weights in shared memory;
// then each of the eight warps adds up every eighth part, a lane DPAD / 32 columns, with eight reads under way at once.
constexpr int JOIN_PARTS = 512;  // weights held at a time
constexpr int JOIN_WARPS = 8;
// floats of a row of a part: the output, the maximum, the sum, and what keeps rows at 16 bytes
__host__ __device__ constexpr int attn_part_pitch(int dpad) { return dpad + 4; }
template <class T, int ROWS, int DPAD>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attn_join_kernel(AttnArgs a) {
    constexpr int PITCH = attn_part_pitch(DPAD), COLS = DPAD / 32, THREADS = JOIN_WARPS * 32;
    __shared__ float acc_s[JOIN_WARPS][DPAD], weight[JOIN_PARTS], red[JOIN_WARPS][2];
    pdl_wait();
    const int4 item = a.joins[blockIdx.x];
    if (item.x < 0) return;
    const AttnRequest q = attn_request(a, item.x);
    const int rows = min(ROWS, q.rows - item.z * ROWS), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int parts = item.w - (int)blockIdx.x + 1;
    for (int row = blockIdx.y; row < rows; row += gridDim.y) {
        // part i: block x + i, in the place for an item that it began (the first one) or found begun
        auto part = [&](int i) { return a.parts + (((long long)(blockIdx.x + i) * 2 + (i == 0)) * ROWS + row) * PITCH; };
        float top = -INFINITY;
        for (int i = threadIdx.x; i < parts; i += THREADS) {
            const float2 ml = *reinterpret_cast<const float2 *>(part(i) + DPAD);
            if (ml.y != 0.0f) top = fmaxf(top, ml.x);  // a part that saw nothing has the sum 0
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        __syncthreads();
        if (lane == 0) red[warp][0] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) top = fmaxf(top, red[w][0]);
        float sum = 0.0f, acc[COLS] = {};
        for (int p0 = 0; p0 < parts; p0 += JOIN_PARTS) {
            const int n = min(JOIN_PARTS, parts - p0);
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += THREADS) {
                const float2 ml = *reinterpret_cast<const float2 *>(part(p0 + i) + DPAD);
                const float w = ml.y == 0.0f ? 0.0f : exp2f(ml.x - top);
                weight[i] = w;
                sum += ml.y * w;
            }
            __syncthreads();
#pragma unroll 8
            for (int i = warp; i < n; i += JOIN_WARPS) {
                const float w = weight[i];
                const float *v = part(p0 + i) + lane * COLS;
#pragma unroll
                for (int c = 0; c < COLS; c += 2) {
                    const float2 f = *reinterpret_cast<const float2 *>(v + c);
                    if (w != 0.0f) acc[c] += f.x * w, acc[c + 1] += f.y * w;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) red[warp][1] = sum;
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc_s[warp][lane * COLS + c] = acc[c];
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) sum += red[w][1];
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int at = item.z * ROWS + row, token = at / a.group, head = item.y * a.group + at % a.group;
        T *dst = static_cast<T *>(a.out) + (q.first + token) * a.out_stride + (long long)head * a.head_dim;
        for (int d = threadIdx.x; d < a.head_dim; d += THREADS) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < JOIN_WARPS; ++w) v += acc_s[w][d];
            from_f32(dst[d], v * inv);
        }
    }
}

// attention_tc.cu
bool attn_tc_eligible(const AttnArgs &a);
int attn_tc_launch(const AttnArgs &a, int type, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s);
size_t attn_tc_workspace(int head_dim);

}  // namespace tb200
