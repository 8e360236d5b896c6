// Attention of new tokens over a paged cache, for requests of any shape: decoding requests (a few query rows over a long
// context) and whatever the tensor-memory kernel of attention_tc.cu does not take.
//
//     out = softmax(scale * q K^T, visible keys) V,  one pass over K and V with a running maximum m and sum l per row:
//     m' = max(m, max_j s_j),  p_j = 2^(s_j - m'),  l' = l 2^(m - m') + sum p_j,  O' = O 2^(m - m') + p V
//
// A decoding request reads its whole cache for `group` rows: bound by memory, floor = the bytes of K and V.  So the key
// tiles of all requests are divided evenly over the resident blocks (attention.cuh), each of which keeps one to three
// tiles of 64 keys in flight with 16-byte asynchronous copies; a page may have any size, since every row of a tile is
// fetched through its own table entry, looked up two tiles ahead.  Rows that no query row of the tile sees are filled
// with zeros and not read.  The products run as mma.sync.m16n8k16 with fp32 accumulators: with up to 16 rows the four
// warps share a tile's keys (16 each) and are joined once per item, with more each warp has 16 rows of a 64-row tile.
#define TB200_OP_CLASS TB200_PREPARE_LAYER
#include "attention.cuh"

namespace tb200 {

constexpr int AT_THREADS = 128, AT_KEYS = 64;
constexpr int AT_ITEM = 1;       // what an item costs besides its key tiles, in such tiles
constexpr int AT_TC_ROWS = 16;   // requests of more rows go to the tensor-memory kernel (45 requests of 32 rows over 3420 keys: 108 us there, 193 us here)
constexpr int AT_WHOLE_TILES = 4;  // contexts of up to this many key tiles are not split
constexpr int AT_MAX_SMS = 148;  // the workspace is sized without asking the device

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void at_copy16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void at_copy8(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void at_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void at_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void at_ldm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void at_ldm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void at_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void at_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What is taken off a row's scores: their maximum.  bf16 has fp32's exponents.  An fp16 power is a subnormal below 2^-14, off
// by up to 2^-25, and vanishes from the product with V, though not from the sum, below that: the powers are raised by 2^15 (of
// fp16's 2^16), which the sum and O share, so that a long tail of small probabilities is held to 2^-40 of the largest one.
// Not where a step of fp32 could lift them further.
__device__ __forceinline__ float at_shift(float m, __nv_bfloat16) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ float at_shift(float m, __half) { return m == -INFINITY ? 0.0f : fabsf(m) < 0x1p20f ? m - 15.0f : m; }

template <int DPAD, bool SPLIT_KEYS>
struct AtShape {
    static constexpr int ROWS = SPLIT_KEYS ? 16 : 64;
    // The copies in flight hide the memory's latency, several blocks an SM each other's arithmetic: with 128 columns three
    // blocks of two stages read 64 requests of up to 8192 keys in 242 us where two of three took 302 us (196 us since the
    // copies' addresses cost less); with 64 columns
    // four blocks of three stages in 113 us, three of four in 127 us.
    static constexpr int STAGES = DPAD == 64 ? (SPLIT_KEYS ? 3 : 4) : DPAD == 128 ? 2 : SPLIT_KEYS ? 3 : 2;
    static constexpr int BLOCKS_PER_SM = DPAD == 256 ? 1 : !SPLIT_KEYS ? 2 : DPAD == 64 ? 4 : 3;
    static constexpr int ROW_BYTES = DPAD * 2, TILE_BYTES = AT_KEYS * ROW_BYTES, Q_BYTES = ROWS * ROW_BYTES;
    static constexpr int RING = STAGES + 1;  // tiles whose rows have been looked up
    static constexpr int SMEM = Q_BYTES + STAGES * 2 * TILE_BYTES + RING * AT_KEYS * 8 + RING * 2 * 4;
    static constexpr int GRID = AT_MAX_SMS * BLOCKS_PER_SM;
    static constexpr size_t PART_FLOATS = (size_t)ROWS * attn_part_pitch(DPAD);
    static constexpr size_t WORKSPACE = GRID * sizeof(int4) + GRID * 2 * PART_FLOATS * 4;
    static_assert(!SPLIT_KEYS || STAGES * 2 * TILE_BYTES >= 4 * 16 * (DPAD + 2) * 4, "the warps' results fit the drained stages");
};

// 16-byte piece `chunk` of row `row`, XOR-swizzled so that eight rows of one column fall into different banks
template <int DPAD>
__device__ __forceinline__ uint32_t at_swizzle(int row, int chunk) { return row * (DPAD * 2) + ((chunk ^ (row & 7)) << 4); }

template <class T, int DPAD, bool SPLIT_KEYS>
__global__ void __launch_bounds__(AT_THREADS, AtShape<DPAD, SPLIT_KEYS>::BLOCKS_PER_SM) attn_kernel(AttnArgs a) {
    using S = AtShape<DPAD, SPLIT_KEYS>;
    constexpr int ROWS = S::ROWS, STAGES = S::STAGES, RING = S::RING, TILE_BYTES = S::TILE_BYTES;
    constexpr int WKEYS = SPLIT_KEYS ? 16 : AT_KEYS;  // keys of a tile that a warp works on
    constexpr bool Q_IN_REGS = DPAD <= 128;
    extern __shared__ __align__(1024) unsigned char at_smem[];
    unsigned char *q_s = at_smem, *kv_s = at_smem + S::Q_BYTES;
    long long *row_s = reinterpret_cast<long long *>(kv_s + STAGES * 2 * TILE_BYTES);  // [RING][64]: place in the cache, -1: none
    int *hole_s = reinterpret_cast<int *>(row_s + RING * AT_KEYS);                     // [RING][2]: a row of the tile's half is missing
    __shared__ AttnStart start;
    __shared__ long long scan[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int D = a.head_dim, ksteps = (D + 15) / 16, dchunks = D / 8, lchunks = 2 * ksteps;
    const int warp_key = SPLIT_KEYS ? warp * 16 : 0, warp_row = SPLIT_KEYS ? 0 : warp * 16;
    const long long v_ahead = static_cast<const char *>(a.v_cache) - static_cast<const char *>(a.k_cache);
    const bool copy16 = ((uintptr_t)a.k_cache & 15) == 0 && ((uintptr_t)a.v_cache & 15) == 0;

    if (!a.whole) {
        attn_find_start<AT_THREADS, ROWS, AT_KEYS, AT_ITEM>(a, &start, scan);
        if (start.begin >= start.end) {
            if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
            pdl_launch_dependents();
            return;
        }
    }
    AttnWalk<ROWS, AT_KEYS, AT_ITEM> w;
    bool more = a.whole ? w.first_whole(a) : w.seek(a, start);
    int4 join = make_int4(-1, 0, 0, 0);

    while (more) {
        const AttnRequest rq = w.q;
        const int row0 = w.tile * ROWS, rows = min(ROWS, rq.rows - row0), base = rq.kv_len - rq.new_tokens;
        const int pos_first = base + row0 / a.group, pos_last = base + (row0 + rows - 1) / a.group;
        const int key_lo = a.window > 0 ? max(0, pos_first - a.window + 1) : 0, key_hi = min(pos_last, rq.visible - 1);
        const int tile0 = w.first + w.from, ntiles = w.to - w.from;
        const int32_t *table = a.block_table + (long long)w.request * a.max_pages;

        // where in the cache key `key` of the request lies for this head, in bytes
        auto look_up = [&](int key) -> long long {
            if (key < key_lo || key > key_hi) return -1;
            const int index = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
            const int page = table[index];
            if (page < 0 || page >= a.num_pages) return -1;
            return (((long long)page * a.kv_heads + w.head) * a.page_size + (key - index * a.page_size)) * (2 * D);
        };
        auto put_row = [&](int slot, long long row) {  // warps 0 and 1
            row_s[slot * AT_KEYS + tid] = row;
            const bool hole = __any_sync(0xffffffffu, row < 0);
            if (lane == 0) hole_s[slot * 2 + warp] = hole;
        };
        // a thread copies one 16-byte column of every RSTEP-th row
        auto load_tile = [&](int i) {
            constexpr int CHUNKS = DPAD / 8, RSTEP = AT_THREADS / CHUNKS;
            const int chunk = tid % CHUNKS, r0 = tid / CHUNKS;
            if (chunk >= lchunks) return;
            const uint32_t ks = smem_u32(kv_s) + (i % STAGES) * 2 * TILE_BYTES;
            const long long *rows_of = row_s + (i % RING) * AT_KEYS;
            const char *column = static_cast<const char *>(a.k_cache) + chunk * 16;
#pragma unroll
            for (int n = 0; n < AT_KEYS / RSTEP; ++n) {
                const int row = r0 + n * RSTEP;
                const long long at = rows_of[row];
                const bool there = at >= 0 && chunk < dchunks;
                const char *k = there ? column + at : static_cast<const char *>(a.k_cache);
                const uint32_t dst = ks + at_swizzle<DPAD>(row, chunk);
                if (copy16) {
                    at_copy16(dst, k, there ? 16 : 0);
                    at_copy16(dst + TILE_BYTES, k + v_ahead, there ? 16 : 0);
                } else {
                    const int step = there ? 8 : 0;
                    at_copy8(dst, k, step), at_copy8(dst + 8, k + step, step);
                    at_copy8(dst + TILE_BYTES, k + v_ahead, step), at_copy8(dst + TILE_BYTES + 8, k + v_ahead + step, step);
                }
            }
        };

        __syncthreads();  // the item before is done with shared memory
        if (tid < AT_KEYS)
            for (int i = 0; i < STAGES; ++i) put_row(i, i < ntiles ? look_up((tile0 + i) * AT_KEYS + tid) : -1);
        // query rows, zeros behind the last one and behind head_dim
        const bool q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 8 == 0;
        for (int e = tid; e < ROWS * lchunks; e += AT_THREADS) {
            const int row = e / lchunks, chunk = e - row * lchunks, at = row0 + row;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < rows && chunk < dchunks) {
                const int token = at / a.group, head = w.head * a.group + (at - token * a.group);
                const T *src = static_cast<const T *>(a.q) + (rq.first + token) * a.q_stride + (long long)head * D + chunk * 8;
                if (q_vec) {
                    v = *reinterpret_cast<const uint4 *>(src);
                } else {
                    const uint16_t *h = reinterpret_cast<const uint16_t *>(src);
                    v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
                }
            }
            *reinterpret_cast<uint4 *>(q_s + at_swizzle<DPAD>(row, chunk)) = v;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            if (i < ntiles) load_tile(i);
            at_commit();
        }
        uint32_t qf[Q_IN_REGS ? DPAD / 16 : 1][4];
        auto load_q = [&](int kk, uint32_t (&r)[4]) { at_ldm(smem_u32(q_s) + at_swizzle<DPAD>(warp_row + (lane & 15), 2 * kk + (lane >> 4)), r); };
        if constexpr (Q_IN_REGS) {
#pragma unroll
            for (int kk = 0; kk < DPAD / 16; ++kk)
                if (kk < ksteps) load_q(kk, qf[kk]);
        }

        // this thread's rows of the warp's 16: lane / 4 and 8 behind it
        const int my_row = warp_row + lane / 4;
        int pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) pos[h] = my_row + 8 * h < rows ? base + (row0 + my_row + 8 * h) / a.group : -1;
        float o[DPAD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < DPAD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        const bool warp_active = warp_row < rows;

        for (int i = 0; i < ntiles; ++i) {
            at_wait<STAGES - 2>();
            __syncthreads();  // tile i is there, and everybody is done with tile i - 1
            if (i + STAGES - 1 < ntiles) load_tile(i + STAGES - 1);
            at_commit();
            // the table entry of a tile further on is under way while this one is worked on
            long long next_row = -1;
            if (tid < AT_KEYS && i + STAGES < ntiles) next_row = look_up((tile0 + i + STAGES) * AT_KEYS + tid);

            if (warp_active) {
                const int key0 = (tile0 + i) * AT_KEYS + warp_key, slot = i % RING;
                const uint32_t ks = smem_u32(kv_s + (i % STAGES) * 2 * TILE_BYTES), vs = ks + TILE_BYTES;
                float s[WKEYS / 8][4];
#pragma unroll
                for (int n = 0; n < WKEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < DPAD / 16; ++kk) {
                    if (kk >= ksteps) break;
                    uint32_t qr[4];
                    if constexpr (!Q_IN_REGS) load_q(kk, qr);
#pragma unroll
                    for (int n = 0; n < WKEYS / 16; ++n) {
                        uint32_t b[4];
                        at_ldm(ks + at_swizzle<DPAD>(warp_key + 16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)), b);
                        if constexpr (Q_IN_REGS) {
                            at_mma(s[2 * n], qf[kk], b[0], b[1], T());
                            at_mma(s[2 * n + 1], qf[kk], b[2], b[3], T());
                        } else {
                            at_mma(s[2 * n], qr, b[0], b[1], T());
                            at_mma(s[2 * n + 1], qr, b[2], b[3], T());
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] *= a.scale_log2;
                // keys that some row of the tile does not see
                const bool edge = key0 + WKEYS - 1 > pos_first || (a.window > 0 && key0 <= pos_last - a.window);
                const bool masked = edge || hole_s[slot * 2] || hole_s[slot * 2 + 1];
                if (masked) {
#pragma unroll
                    for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int in = 8 * n + 2 * (lane & 3) + (e & 1), key = key0 + in, p = pos[e >> 1];
                            const bool seen = key <= p && (a.window == 0 || key > p - a.window) && row_s[slot * AT_KEYS + warp_key + in] >= 0;
                            if (!seen) s[n][e] = -INFINITY;
                        }
                }
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < WKEYS / 8; ++n) {
                    top[0] = fmaxf(top[0], fmaxf(s[n][0], s[n][1]));
                    top[1] = fmaxf(top[1], fmaxf(s[n][2], s[n][3]));
                }
                float shift[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                    top[h] = fmaxf(top[h], m[h]);
                    shift[h] = at_shift(top[h], T());
                }
                if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
                    const float f0 = m[0] == -INFINITY ? 0.0f : ex2(at_shift(m[0], T()) - shift[0]), f1 = m[1] == -INFINITY ? 0.0f : ex2(at_shift(m[1], T()) - shift[1]);
                    l[0] *= f0, l[1] *= f1;
#pragma unroll
                    for (int n = 0; n < DPAD / 8; ++n) o[n][0] *= f0, o[n][1] *= f0, o[n][2] *= f1, o[n][3] *= f1;
                    m[0] = top[0], m[1] = top[1];
                }
                // A value of V that one row sees and another one does not may be infinite or a NaN: 0 * V would carry it
                // to the other row.  Tiles at an edge of several tokens are looked over, and summed key by key if so.
                bool by_key = false;
                if (edge && pos_first != pos_last) {
                    bool odd = false;
                    for (int e = lane; e < WKEYS * lchunks; e += 32) {
                        const int row = warp_key + e / lchunks, chunk = e % lchunks;
                        uint32_t u[4];
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(vs + at_swizzle<DPAD>(row, chunk)));
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 f = unpack2(u[c], T());
                            odd |= !(fabsf(f.x) <= 3.402823466e38f) || !(fabsf(f.y) <= 3.402823466e38f);
                        }
                    }
                    by_key = __any_sync(0xffffffffu, odd);
                }
                if (!by_key) {
#pragma unroll
                    for (int n = 0; n < WKEYS / 16; ++n) {
                        uint32_t p[4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float p0 = ex2(s[2 * n + h][0] - shift[0]), p1 = ex2(s[2 * n + h][1] - shift[0]);
                            const float p2 = ex2(s[2 * n + h][2] - shift[1]), p3 = ex2(s[2 * n + h][3] - shift[1]);
                            l[0] += p0 + p1, l[1] += p2 + p3;
                            p[2 * h] = pack2(p0, p1, T()), p[2 * h + 1] = pack2(p2, p3, T());  // half a step of `type`, relative to p (fp16: 2^-25 below 2^-14)
                        }
#pragma unroll
                        for (int d = 0; d < DPAD / 16; ++d) {
                            if (d >= ksteps) break;
                            uint32_t b[4];
                            at_ldm_t(vs + at_swizzle<DPAD>(warp_key + 16 * n + (lane & 15), 2 * d + (lane >> 4)), b);
                            at_mma(o[2 * d], p, b[0], b[1], T());
                            at_mma(o[2 * d + 1], p, b[2], b[3], T());
                        }
                    }
                } else {
                    float pv[WKEYS / 8][4];
#pragma unroll
                    for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + 8 * n + 2 * (lane & 3) + (e & 1), p = pos[e >> 1];
                            const bool seen = key <= p && (a.window == 0 || key > p - a.window) && row_s[slot * AT_KEYS + key - key0 + warp_key] >= 0;
                            const float f = ex2(s[n][e] - shift[e >> 1]);
                            l[e >> 1] += seen ? f : 0.0f;
                            pv[n][e] = seen ? unpack2(pack2(f, 0.0f, T()), T()).x : -1.0f;
                        }
#pragma unroll 1
                    for (int k = 0; k < WKEYS; ++k) {
                        const int from = (lane & ~3) | ((k >> 1) & 3);
                        const float p0 = __shfl_sync(0xffffffffu, pv[k >> 3][k & 1], from), p1 = __shfl_sync(0xffffffffu, pv[k >> 3][2 + (k & 1)], from);
#pragma unroll
                        for (int d = 0; d < DPAD / 8; ++d) {
                            if (d >= 2 * ksteps) break;
                            uint32_t u;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(vs + at_swizzle<DPAD>(warp_key + k, d) + (lane & 3) * 4));
                            const float2 f = unpack2(u, T());
                            if (!(p0 < 0.0f)) o[d][0] += p0 * f.x, o[d][1] += p0 * f.y;
                            if (!(p1 < 0.0f)) o[d][2] += p1 * f.x, o[d][3] += p1 * f.y;
                        }
                    }
                }
            }
            if (tid < AT_KEYS) put_row((i + STAGES) % RING, next_row);
        }
        at_wait<0>();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }

        const bool whole = w.whole();
        if (!whole && w.from == 0 && tid == 0)
            join = make_int4(w.request, w.head, w.tile, attn_block_of(start.total, start.blocks, w.item_begin + AT_ITEM + w.count - 1));
        float *part = a.parts + ((long long)blockIdx.x * 2 + (w.from == 0)) * S::PART_FLOATS;
        // one row's columns d, d + 1 of the result or of the part
        const bool out2 = ((uintptr_t)a.out & 3) == 0 && a.out_stride % 2 == 0;
        auto put = [&](int row, int d, float x, float y, float inv) {
            if (whole) {
                if (d >= D) return;
                const int at = row0 + row, token = at / a.group, head = w.head * a.group + (at - token * a.group);
                T *dst = static_cast<T *>(a.out) + (rq.first + token) * a.out_stride + (long long)head * D + d;
                if (out2) {
                    *reinterpret_cast<uint32_t *>(dst) = pack2(x * inv, y * inv, T());
                } else {
                    from_f32(dst[0], x * inv);
                    from_f32(dst[1], y * inv);
                }
            } else {
                *reinterpret_cast<float2 *>(part + row * attn_part_pitch(DPAD) + d) = make_float2(x, y);
            }
        };
        if constexpr (SPLIT_KEYS) {
            // every warp has the same 16 rows over its keys
            float *acc = reinterpret_cast<float *>(kv_s), *ml = acc + 4 * 16 * DPAD;
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = lane / 4 + 8 * h;
                if ((lane & 3) == 0) ml[(warp * 16 + row) * 2] = at_shift(m[h], T()), ml[(warp * 16 + row) * 2 + 1] = l[h];
#pragma unroll
                for (int n = 0; n < DPAD / 8; ++n)
                    *reinterpret_cast<float2 *>(acc + (warp * 16 + row) * DPAD + 8 * n + 2 * (lane & 3)) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
            }
            __syncthreads();
            for (int e = tid; e < rows * (DPAD / 2); e += AT_THREADS) {
                const int row = e / (DPAD / 2), d = 2 * (e - row * (DPAD / 2));
                float top = -INFINITY, sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = *reinterpret_cast<const float2 *>(ml + (k * 16 + row) * 2);
                    if (v.y != 0.0f) top = fmaxf(top, v.x);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = *reinterpret_cast<const float2 *>(ml + (k * 16 + row) * 2);
                    if (v.y == 0.0f) continue;  // saw nothing
                    const float f = ex2(v.x - top);
                    const float2 c = *reinterpret_cast<const float2 *>(acc + (k * 16 + row) * DPAD + d);
                    sum += v.y * f, x += c.x * f, y += c.y * f;
                }
                put(row, d, x, y, sum == 0.0f ? 0.0f : 1.0f / sum);
                if (!whole && d == 0) part[row * attn_part_pitch(DPAD) + DPAD] = top, part[row * attn_part_pitch(DPAD) + DPAD + 1] = sum;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = my_row + 8 * h;
                if (row < rows) {
                    const float inv = l[h] == 0.0f ? 0.0f : 1.0f / l[h];
                    if (__builtin_expect(l[h] == 0.0f, 0)) {  // saw nothing, or only scores of -infinity, times values that need not be finite
#pragma unroll
                        for (int n = 0; n < DPAD / 8; ++n) o[n][2 * h] = o[n][2 * h + 1] = 0.0f;
                    }
#pragma unroll
                    for (int n = 0; n < DPAD / 8; ++n) put(row, 8 * n + 2 * (lane & 3), o[n][2 * h], o[n][2 * h + 1], inv);
                    if (!whole && (lane & 3) == 0) part[row * attn_part_pitch(DPAD) + DPAD] = at_shift(m[h], T()), part[row * attn_part_pitch(DPAD) + DPAD + 1] = l[h];
                }
            }
        }
        more = a.whole ? w.next_whole(a) : w.next(a, start);
    }
    if (a.whole) return;
    if (tid == 0) a.joins[blockIdx.x] = join;
    pdl_launch_dependents();
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <class T, int DPAD, bool SPLIT_KEYS>
static int attn_launch(AttnArgs a, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    using S = AtShape<DPAD, SPLIT_KEYS>;
    int st = ensure_kernel<attn_kernel<T, DPAD, SPLIT_KEYS>, KERNEL_OPTIN_SMEM | KERNEL_MAX_CARVEOUT>(di);
    if (st) return st;
    st = ensure_kernel<attn_join_kernel<T, S::ROWS, DPAD>, 0>(di);
    if (st) return st;
    int grid = min(di->sm_count, AT_MAX_SMS) * S::BLOCKS_PER_SM;
    // Short contexts: the search for a block's share and the join take longer than a whole item does.  Six requests of 157
    // keys: 16.4 us split, 12.0 us whole; eight of 500 keys: 15.5 us split, 19.9 us whole.  (Measured on single tokens; the
    // rule does not count row tiles, which a block takes one after another: a prompt of 250 tokens on 8 kv heads takes 42 us
    // with pages of 20, on 8 blocks, and 25 us with pages of 16 on the other kernel.)
    const long long keys = min((long long)a.max_pages * a.page_size, a.window > 0 ? (long long)a.window + longest_rows / a.group : 1LL << 40);
    a.whole = keys <= AT_WHOLE_TILES * AT_KEYS && (long long)a.requests * a.kv_heads <= 0x3FFFFFFF;
    if (a.whole) {
        grid = (int)min((long long)grid, (long long)a.requests * a.kv_heads);
        return launch_kernel(attn_kernel<T, DPAD, SPLIT_KEYS>, dim3(grid), dim3(AT_THREADS), S::SMEM, s, false, a);
    }
    a.joins = static_cast<int4 *>(workspace);
    a.parts = reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + S::GRID * sizeof(int4));
    st = launch_kernel(attn_kernel<T, DPAD, SPLIT_KEYS>, dim3(grid), dim3(AT_THREADS), S::SMEM, s, false, a);
    if (st) return st;
    // the join waits for the main kernel by itself (programmatic launch): its start-up is hidden behind it
    return launch_kernel(attn_join_kernel<T, S::ROWS, DPAD>, dim3(grid, min(longest_rows, 8)), dim3(JOIN_WARPS * 32), 0, s, true, a);
}

template <class T, int DPAD>
static int attn_launch_rows(const AttnArgs &a, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    return longest_rows <= 16 ? attn_launch<T, DPAD, true>(a, longest_rows, workspace, di, s) : attn_launch<T, DPAD, false>(a, longest_rows, workspace, di, s);
}

template <class T>
static int attn_launch_dim(const AttnArgs &a, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    if (a.head_dim <= 64) return attn_launch_rows<T, 64>(a, longest_rows, workspace, di, s);
    if (a.head_dim <= 128) return attn_launch_rows<T, 128>(a, longest_rows, workspace, di, s);
    return attn_launch_rows<T, 256>(a, longest_rows, workspace, di, s);
}

int attn_any_launch(AttnArgs a, int type, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    return type == TB200_TYPE_F16 ? attn_launch_dim<__half>(a, longest_rows, workspace, di, s) : attn_launch_dim<__nv_bfloat16>(a, longest_rows, workspace, di, s);
}

size_t attn_any_workspace(int head_dim) {
    if (head_dim <= 64) return max(AtShape<64, true>::WORKSPACE, AtShape<64, false>::WORKSPACE);
    if (head_dim <= 128) return max(AtShape<128, true>::WORKSPACE, AtShape<128, false>::WORKSPACE);
    return max(AtShape<256, true>::WORKSPACE, AtShape<256, false>::WORKSPACE);
}

}  // namespace tb200

using namespace tb200;

static bool attn_shape_ok(int tokens, int requests, int q_heads, int kv_heads, int head_dim) {
    return tokens >= 0 && requests >= 0 && requests <= (1 << 30) && kv_heads >= 1 && q_heads >= kv_heads && q_heads % kv_heads == 0 && head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0 &&
           (long long)tokens * (q_heads / kv_heads) <= (1LL << 30) && q_heads <= 65536;
}

extern "C" size_t tb200_paged_attention_workspace_bytes(int tokens, int requests, int q_heads, int kv_heads, int head_dim) {
    if (!attn_shape_ok(tokens, requests, q_heads, kv_heads, head_dim)) return 0;
    return max(attn_any_workspace(head_dim), attn_tc_workspace(head_dim));
}

extern "C" int tb200_paged_attention(int tokens, int requests, int max_new, int q_heads, int kv_heads, int head_dim, int type, const void *q,
                                     long long q_stride, const int32_t *cu_new, const int32_t *kv_lens, const int32_t *block_table, int max_pages,
                                     int page_size, int num_pages, const void *k_cache, const void *v_cache, float scale, int window, void *out,
                                     long long out_stride, void *workspace, size_t workspace_bytes, tb200_stream_t stream) {
    if (!attn_shape_ok(tokens, requests, q_heads, kv_heads, head_dim) || (type != TB200_TYPE_F16 && type != TB200_TYPE_BF16)) return TB200_ERR_INVALID_ARG;
    if (max_new < 0 || max_pages < 0 || page_size < 1 || num_pages < 0 || window < 0 || (long long)max_pages * page_size > (1LL << 30)) return TB200_ERR_INVALID_ARG;
    if (!(scale > 0.0f) || scale > 3.402823466e38f) return TB200_ERR_INVALID_ARG;
    if (q_stride < (long long)q_heads * head_dim || out_stride < (long long)q_heads * head_dim) return TB200_ERR_INVALID_ARG;
    if (tokens == 0 || requests == 0) return TB200_OK;
    if (!q || !out || !cu_new || !kv_lens || (max_pages > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache))) return TB200_ERR_INVALID_ARG;
    if (!aligned_to(q, 2) || !aligned_to(out, 8) || !aligned_to(k_cache, 8) || !aligned_to(v_cache, 8) || !aligned_to(cu_new, 4) || !aligned_to(kv_lens, 4) ||
        !aligned_to(block_table, 4))
        return TB200_ERR_ALIGNMENT;
    if (!workspace || workspace_bytes < tb200_paged_attention_workspace_bytes(tokens, requests, q_heads, kv_heads, head_dim)) return TB200_ERR_WORKSPACE;
    if (!aligned_to(workspace, 16)) return TB200_ERR_ALIGNMENT;
    // A block reads a tile's query rows before anybody stores that tile's results, and nobody else reads them: out may be q,
    // but not at another pitch, where a row's results land on other rows.
    if (out == q && out_stride != q_stride && tokens > 1) return TB200_ERR_INVALID_ARG;
    int st;
    const DeviceInfo *di = device_info(&st);
    if (!di) return st;
    AttnArgs a{};
    if (num_pages == 0) k_cache = v_cache = workspace;  // never read; an address for copies of no bytes
    a.q = q, a.k_cache = k_cache, a.v_cache = v_cache, a.cu_new = cu_new, a.kv_lens = kv_lens, a.block_table = block_table, a.out = out;
    a.q_stride = q_stride, a.out_stride = out_stride, a.scale_log2 = scale * 1.4426950408889634f;
    a.tokens = tokens, a.requests = requests, a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads, a.head_dim = head_dim;
    a.max_pages = max_pages, a.page_size = page_size, a.num_pages = num_pages;
    a.window = window < (1 << 30) ? window : 0;  // positions are below 2^30: a wider window limits nothing, and a position minus a window stays a 32-bit number
    a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
    const long long longest = (long long)(max_new > 0 ? min(max_new, tokens) : tokens) * a.group;
    const int rows = (int)min(longest, 0x7FFFFFFFLL);
    // Heads of more than 128 columns leave room for one block an SM here, too few for the memory's latency: 45 requests of
    // 1183 keys on 8 heads of 256 take 111 us here and 79 us there.
    if ((rows > AT_TC_ROWS || head_dim > 128) && attn_tc_eligible(a)) return attn_tc_launch(a, type, rows, workspace, di, (cudaStream_t)stream);
    return attn_any_launch(a, type, rows, workspace, di, (cudaStream_t)stream);
}
