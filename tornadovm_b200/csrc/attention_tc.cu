// Attention of chunks of new tokens over a paged cache on the 5th-generation tensor cores.
//
// One persistent block per SM works on tiles of 256 query rows (two of 128, one per lane of tensor memory) against key
// tiles of 128:
//   * warp 8 fetches K and V tiles into a ring of shared-memory slots, one TMA box per page and 64 columns (lanes look
//     the pages up side by side, a tile ahead); a page that no row sees, or that is none of the cache's, is fetched from
//     behind the end of the tensor map and arrives as zeros;
//   * warp 9 issues tcgen05.mma: S_t = Q_t K^T into tensor memory (fp32), and O_t += P_t V with P_t read from tensor
//     memory, where it overlies S_t;
//   * warps 0-3 and 4-7 hold the softmax of one 128-row tile each, a row per thread: S from tensor memory, the running
//     maximum and sum in registers, P back as 16-bit values.  While one tile's probabilities are computed the tensor
//     cores work on the other tile.  O stays in tensor memory; it is rescaled only when a row's maximum has grown by
//     more than 2^8 since its reference was set (P then reaches 256 at most, well inside fp16, and the quotient O / l
//     does not depend on the reference), which after the first tiles of a row hardly ever happens.
// Bound: two products of 128 x 128 x head_dim and 128 x 128 powers of two per (row tile, key tile).  The key tiles of all
// items are divided evenly over the blocks and split rows are joined afterwards (attention.cuh).
//
// Every wait is bounded: on expiry the block records TB200_ERR_TIMEOUT, all roles leave their loops, copies in flight are
// waited for (bounded again) and tensor memory is released.
#define TB200_OP_CLASS TB200_PREPARE_LAYER
#include "attention.cuh"
#include "tcgen05.cuh"

TB200_TU_STATUS(attention_tc)

namespace tb200 {

constexpr int TC_ROWS = 256, TC_KEYS = 128, TC_THREADS = 384;  // three warpgroups; the last one's warps 8 and 9 work
// Registers: 384 threads are launched with 168 each, which the softmax threads (128 scores in registers) outgrow, so the
// warpgroups share them anew: 2 * 216 + 72 = 3 * 168.
constexpr int TC_SOFTMAX_REGS = 216, TC_OTHER_REGS = 72;
static_assert(2 * TC_SOFTMAX_REGS + TC_OTHER_REGS == 3 * 168, "the shares add up to what the block was launched with");

template <int DPAD>
struct TcShape {
    static constexpr int PANELS = DPAD / 64;                // 64 columns = 128 bytes: the swizzled rows of a tile
    static constexpr int PANEL_BYTES = TC_KEYS * 128;
    static constexpr int TILE_BYTES = PANELS * PANEL_BYTES;  // K or V tile, and 128 query rows
    static constexpr int SLOTS = DPAD == 128 ? 5 : 10;
    static constexpr int SMEM = (2 + SLOTS) * TILE_BYTES + 1024;
    static constexpr int GRID = 148;
    static constexpr size_t PART_FLOATS = (size_t)TC_ROWS * (DPAD + 2);
    static constexpr size_t WORKSPACE = GRID * sizeof(int4) + GRID * 2 * PART_FLOATS * 4;
    // tensor memory: S_0, S_1 (128 columns each; P_t in the first 64 of S_t), O_0, O_1
    static constexpr uint32_t O_COL = 256, TMEM_COLS = 512;
};

__device__ __forceinline__ float tc_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ bool tc_not_finite(uint32_t w, __half) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }
__device__ __forceinline__ bool tc_not_finite(uint32_t w, __nv_bfloat16) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; }
__device__ __forceinline__ uint32_t tc_finite_only(uint32_t w, __half) {
    return ((w & 0x7C00u) == 0x7C00u ? 0u : w & 0xFFFFu) | ((w & 0x7C000000u) == 0x7C000000u ? 0u : w & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t tc_finite_only(uint32_t w, __nv_bfloat16) {
    return ((w & 0x7F80u) == 0x7F80u ? 0u : w & 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0u : w & 0xFFFF0000u);
}

struct TcShared {
    uint64_t slot_full[10], slot_empty[10], q_full[2], s_full[2], p_full[2], o_full[2], drained;
    AttnStart start;
    long long scan[TC_THREADS / 32 + 1];
    uint32_t tmem_base;
    int abort_flag;
    int odd_values;        // some value of V at an edge was not finite: the rows that see it get it in the epilogue
    uint32_t holes[8];     // per key tile (a ring): pages of the tile that are none of the cache's
};

// What the rows of an item see.
struct TcItem {
    int row0, rows, base, pos_first, pos_last, key_lo, key_hi, tile0, ntiles;
    __device__ __forceinline__ TcItem(const AttnArgs &a, const AttnWalk<TC_ROWS, TC_KEYS> &w) {
        row0 = w.tile * TC_ROWS, rows = min(TC_ROWS, w.q.rows - row0), base = w.q.kv_len - w.q.new_tokens;
        pos_first = base + row0 / a.group, pos_last = base + (row0 + rows - 1) / a.group;
        key_lo = a.window > 0 ? max(0, pos_first - a.window + 1) : 0, key_hi = min(pos_last, w.q.visible - 1);
        tile0 = w.first + w.from, ntiles = w.to - w.from;
    }
};

template <class T, int DPAD>
__global__ void __launch_bounds__(TC_THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a, uint32_t idesc_qk,
               uint32_t idesc_pv) {
    using S = TcShape<DPAD>;
    constexpr int PANELS = S::PANELS, SLOTS = S::SLOTS;
    extern __shared__ __align__(128) unsigned char tc_smem[];
    __shared__ __align__(16) TcShared sh;
    unsigned char *q_s = reinterpret_cast<unsigned char *>(((uintptr_t)tc_smem + 1023) & ~(uintptr_t)1023);  // swizzled tiles: 1024-byte bases
    unsigned char *kv_s = q_s + 2 * S::TILE_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        sh.abort_flag = 0, sh.odd_values = 0;
        for (int i = 0; i < SLOTS; ++i) mbar_init(&sh.slot_full[i], 1), mbar_init(&sh.slot_empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&sh.q_full[i], 128), mbar_init(&sh.s_full[i], 1), mbar_init(&sh.p_full[i], 4), mbar_init(&sh.o_full[i], 1);
        mbar_init(&sh.drained, 1);
        mbar_fence_init();
    }
    if (warp == 8 && lane == 0) tma_prefetch_map(&map_k), tma_prefetch_map(&map_v);
    attn_find_start<TC_THREADS, TC_ROWS, TC_KEYS>(a, &sh.start, sh.scan);
    if (sh.start.begin >= sh.start.end) {
        if (threadIdx.x == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
        pdl_launch_dependents();
        return;
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(S::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    volatile int *abortp = &sh.abort_flag;
    AttnWalk<TC_ROWS, TC_KEYS> w;
    w.seek(a, sh.start);
    bool more = true, ok = true;

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_OTHER_REGS));
    if (warp == 8) {
        // ---------------- producer ----------------
        const int box_keys = min(a.page_size, TC_KEYS), boxes = TC_KEYS / box_keys;
        const int behind = a.num_pages * a.kv_heads * a.page_size;  // first row behind the cache: zeros
        uint32_t it = 0, tiles = 0;
        while (more && ok) {
            const TcItem t(a, w);
            const int32_t *table = a.block_table + (long long)w.request * a.max_pages;
            // lane b: row of the cache at which box b of a tile begins, and whether its page is missing
            auto look_up = [&](int tile, bool &hole) -> int {
                const int key = tile * TC_KEYS + lane * box_keys;
                hole = false;
                if (lane >= boxes || key > t.key_hi || key + box_keys <= t.key_lo) return behind;
                const int index = key >> a.page_shift, page = table[index];
                hole = page < 0 || page >= a.num_pages;
                return hole ? behind : (page * a.kv_heads + w.head) * a.page_size + (key - (index << a.page_shift));
            };
            bool hole;
            int row = look_up(t.tile0, hole);
            for (int j = 0; j < t.ntiles && ok; ++j, ++tiles) {
                bool next_hole = false;
                const int next_row = j + 1 < t.ntiles ? look_up(t.tile0 + j + 1, next_hole) : behind;
                const uint32_t holes = __ballot_sync(0xffffffffu, hole);
                if (lane == 0) sh.holes[tiles & 7] = holes;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++it) {
                    const int s = it % SLOTS;
                    const uint32_t use = it / SLOTS;
                    if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.slot_empty[s], (use - 1) & 1, abortp));
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&sh.slot_full[s], S::TILE_BYTES);
                    __syncwarp();
                    for (int i = lane; i < ((boxes * PANELS + 31) & ~31); i += 32) {
                        const int b = i / PANELS, panel = i % PANELS;
                        const int y = __shfl_sync(0xffffffffu, row, b & 31);
                        if (b < boxes)
                            tma_load_2d(kv_s + s * S::TILE_BYTES + panel * S::PANEL_BYTES + b * box_keys * 128, kv == 0 ? &map_k : &map_v, panel * 64, y,
                                        &sh.slot_full[s]);
                    }
                }
                row = next_row, hole = next_hole;
            }
            more = w.next(a, sh.start);
        }
        // copies in flight when a wait has expired (in the normal course all have been waited for by their readers)
        if (!ok && lane == 0)
            for (uint32_t k = it > SLOTS ? it - SLOTS : 0; k < it; ++k)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(&sh.slot_full[k % SLOTS], (k / SLOTS) & 1); ++i) {
                }
    } else if (warp == 9) {
        // ---------------- products ----------------
        if (lane == 0) {
            uint32_t it = 0, q_use[2] = {0, 0}, p_use[2] = {0, 0};
            const uint32_t q_addr = smem_u32(q_s), kv_addr = smem_u32(kv_s);
            // S_t = Q_t K^T: both operands K-major, rows of 128 bytes, 16 columns = 32 bytes per instruction
            auto qk = [&](int t, uint32_t slot) {
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k) {
                    const uint32_t at = (k / 4) * S::PANEL_BYTES + (k % 4) * 32;
                    tc_mma_f16(tmem + t * 128, make_smem_desc(q_addr + t * S::TILE_BYTES + at, 16, 1024), make_smem_desc(kv_addr + slot * S::TILE_BYTES + at, 16, 1024),
                               idesc_qk, k > 0);
                }
                tc_commit(&sh.s_full[t]);
            };
            // O_t (+)= P_t V: P in tensor memory (16 keys = 8 columns), V with its columns contiguous, 16 keys = 2048 bytes
            auto pv = [&](int t, uint32_t slot, bool add) {
                const uint64_t v = make_smem_desc(kv_addr + slot * S::TILE_BYTES, S::PANEL_BYTES, 1024);
#pragma unroll
                for (int k = 0; k < TC_KEYS / 16; ++k) tc_mma_f16_ta(tmem + S::O_COL + t * 128, tmem + t * 128 + k * 8, v + (uint64_t)(k * 128), idesc_pv, add || k > 0);
            };
            auto wait_slot = [&]() { return mbar_wait_abortable(&sh.slot_full[it % SLOTS], (it / SLOTS) & 1, abortp); };
            auto wait_p = [&](int t) {
                const bool r = mbar_wait_abortable(&sh.p_full[t], p_use[t]++ & 1, abortp);
                tc_fence_after();
                return r;
            };
            while (more && ok) {
                const TcItem t(a, w);
                const bool two = t.rows > 128;
                ok = mbar_wait_abortable(&sh.q_full[0], q_use[0]++ & 1, abortp) && (!two || mbar_wait_abortable(&sh.q_full[1], q_use[1]++ & 1, abortp));
                uint32_t v_slot = 0;
                for (int j = 0; j < t.ntiles && ok; ++j) {
                    const uint32_t k_slot = it % SLOTS;
                    if (!(ok = wait_slot())) break;
                    tc_fence_after();
                    ++it;
                    qk(0, k_slot);
                    if (two) {
                        if (j > 0) {
                            if (!(ok = wait_p(1))) break;
                            pv(1, v_slot, j > 1);
                            tc_commit(&sh.slot_empty[v_slot]);
                        }
                        qk(1, k_slot);
                    }
                    tc_commit(&sh.slot_empty[k_slot]);
                    v_slot = it % SLOTS;
                    if (!(ok = wait_slot())) break;
                    ++it;
                    if (!(ok = wait_p(0))) break;
                    pv(0, v_slot, j > 0);
                    if (!two) tc_commit(&sh.slot_empty[v_slot]);
                }
                if (ok) tc_commit(&sh.o_full[0]);
                if (ok && two && (ok = wait_p(1))) {
                    pv(1, v_slot, t.ntiles > 1);
                    tc_commit(&sh.slot_empty[v_slot]);
                    tc_commit(&sh.o_full[1]);
                }
                more = w.next(a, sh.start);
            }
            tc_commit(&sh.drained);  // nothing of this block's products is under way when tensor memory is released
            for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(&sh.drained, 0); ++i) {
            }
        }
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_SOFTMAX_REGS));
        // ---------------- softmax ----------------
        const int t = warp >> 2, row_in = threadIdx.x & 127, D = a.head_dim, chunks = D / 8;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + S::O_COL + t * 128;
        const bool q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 8 == 0;
        unsigned char *my_q = q_s + t * S::TILE_BYTES;
        uint32_t it = 0, tiles = 0, s_use = 0, o_use = 0;
        while (more && ok) {
            const TcItem im(a, w);
            if (t == 1 && im.rows <= 128) {
                it += 2 * im.ntiles, tiles += im.ntiles;
                more = w.next(a, sh.start);
                continue;
            }
            // query rows: 8 threads of a warp share a row's 16-byte pieces, so that the reads are whole lines
            for (int e = row_in; e < 128 * (DPAD / 8); e += 128) {
                const int r = e / (DPAD / 8), c = e % (DPAD / 8), row = t * 128 + r, at = im.row0 + row;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row < im.rows && c < chunks) {
                    const int token = at / a.group, head = w.head * a.group + (at - token * a.group);
                    const T *src = static_cast<const T *>(a.q) + (w.q.first + token) * a.q_stride + (long long)head * D + c * 8;
                    if (q_vec) {
                        v = *reinterpret_cast<const uint4 *>(src);
                    } else {
                        const uint16_t *h = reinterpret_cast<const uint16_t *>(src);
                        v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
                    }
                }
                *reinterpret_cast<uint4 *>(my_q + (c >> 3) * S::PANEL_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
            }
            fence_async_shared();
            mbar_arrive(&sh.q_full[t]);

            const int my_row = t * 128 + row_in;
            const bool have = my_row < im.rows, warp_has = t * 128 + (warp & 3) * 32 < im.rows;
            const int pos = have ? im.base + (im.row0 + my_row) / a.group : -1;
            const int see_hi = min(pos, w.q.visible - 1), see_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < im.ntiles; ++j, ++tiles, it += 2) {
                ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.s_full[t], s_use++ & 1, abortp));
                if (!ok) break;
                tc_fence_after();
                const int key0 = (im.tile0 + j) * TC_KEYS;
                const uint32_t holes = sh.holes[tiles & 7];
                const bool edge = key0 + TC_KEYS - 1 > min(im.pos_first, im.key_hi) || (a.window > 0 && key0 <= im.pos_last - a.window);
                if (warp_has) {
                    uint32_t s[128];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc_ld_32cols(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
                    tc_wait_ld();
                    if (edge) {
                        const int lo = see_lo - key0, hi = see_hi - key0;
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (i > hi || i < lo) s[i] = 0xFF800000u;
                    }
                    if (holes) {
                        const int shift = min(a.page_shift, 7);
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if ((holes >> (i >> shift)) & 1) s[i] = 0xFF800000u;
                    }
                    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 128; ++i) x[i & 3] = fmaxf(x[i & 3], __uint_as_float(s[i]));
                    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale_log2;
                    if (j == 0) {
                        m = top;
                    } else if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                        const float next = fmaxf(m, top), f = next == m ? 1.0f : tc_ex2(m - next);
#pragma unroll
                        for (int c = 0; c < DPAD / 32; ++c) {
                            uint32_t o[32];
                            tc_ld_32cols(o_addr + c * 32, o);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc_st_32cols(o_addr + c * 32, o);
                        }
                        l *= f, m = next;
                    }
                    const float shift = m == -INFINITY ? 0.0f : m;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t p[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float p0 = tc_ex2(fmaf(__uint_as_float(s[64 * c + 2 * i]), a.scale_log2, -shift));
                            const float p1 = tc_ex2(fmaf(__uint_as_float(s[64 * c + 2 * i + 1]), a.scale_log2, -shift));
                            sum[i & 3] += p0 + p1;
                            p[i] = pack2(p0, p1, T());  // half a step of `type`, relative to p
                        }
                        tc_st_32cols(s_addr + c * 32, p);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc_wait_st();
                }
                if (edge) {
                    // A place that no row sees may hold anything, and one that some rows see and others do not may hold
                    // an infinity or a NaN: 0 * V would carry it to rows that do not see it.  The former become zeros
                    // here; of the latter the values that are not finite do, and the epilogue gives them to their rows.
                    ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.slot_full[(it + 1) % SLOTS], ((it + 1) / SLOTS) & 1, abortp));
                    if (!ok) break;
                    const int key = key0 + row_in;
                    unsigned char *v_row = kv_s + ((it + 1) % SLOTS) * S::TILE_BYTES + row_in * 128;
                    if (key > im.key_hi || key < im.key_lo) {
#pragma unroll
                        for (int c = 0; c < DPAD / 8; ++c) *reinterpret_cast<uint4 *>(v_row + (c >> 3) * S::PANEL_BYTES + (((c & 7) ^ (row_in & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    } else if (key > im.pos_first || (a.window > 0 && key <= im.pos_last - a.window)) {
#pragma unroll
                        for (int c = 0; c < DPAD / 8; ++c) {
                            uint4 *at = reinterpret_cast<uint4 *>(v_row + (c >> 3) * S::PANEL_BYTES + (((c & 7) ^ (row_in & 7)) << 4));
                            const uint4 v = *at;
                            if (tc_not_finite(v.x, T()) || tc_not_finite(v.y, T()) || tc_not_finite(v.z, T()) || tc_not_finite(v.w, T())) {
                                sh.odd_values = 1;
                                *at = make_uint4(tc_finite_only(v.x, T()), tc_finite_only(v.y, T()), tc_finite_only(v.z, T()), tc_finite_only(v.w, T()));
                            }
                        }
                    }
                    fence_async_shared();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (!ok) break;
            ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.o_full[t], o_use++ & 1, abortp));
            if (!ok) break;
            tc_fence_after();
            const bool whole = w.whole(), odd = *reinterpret_cast<volatile int *>(&sh.odd_values) != 0;
            if (warp_has) {
                const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
                const int at = im.row0 + my_row, token = at / a.group, head = w.head * a.group + (at - token * a.group);
                T *dst = static_cast<T *>(a.out) + (w.q.first + token) * a.out_stride + (long long)head * D;
                const bool vec8 = ((uintptr_t)dst & 7) == 0;
                float *part = a.parts + ((long long)blockIdx.x * 2 + (w.from == 0)) * S::PART_FLOATS + my_row;
#pragma unroll 1
                for (int c = 0; c < DPAD / 32; ++c) {
                    uint32_t o[32];
                    tc_ld_32cols(o_addr + c * 32, o);
                    tc_wait_ld();
                    if (odd && have) {
                        // keys at this item's edges, of this block's tiles, that this row sees: their infinities and NaN
                        const int lo = max(max(see_lo, im.key_lo), im.tile0 * TC_KEYS), hi = min(see_hi, (im.tile0 + im.ntiles) * TC_KEYS - 1);
                        for (int key = lo; key <= hi; ++key) {
                            if (key <= im.pos_first && !(a.window > 0 && key <= im.pos_last - a.window)) continue;
                            const int index = key >> a.page_shift, page = a.block_table[(long long)w.request * a.max_pages + index];
                            if (page < 0 || page >= a.num_pages) continue;
                            const T *v = static_cast<const T *>(a.v_cache) + (((long long)page * a.kv_heads + w.head) * a.page_size + (key - (index << a.page_shift))) * D;
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float f = c * 32 + i < D ? to_f32(v[c * 32 + i]) : 0.0f;
                                if (!(fabsf(f) <= 3.402823466e38f)) o[i] = __float_as_uint(__uint_as_float(o[i]) + f);
                            }
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) part[(c * 32 + i) * TC_ROWS] = __uint_as_float(o[i]);
                    } else if (have) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            if (c * 32 + i >= D) break;
                            const float f[4] = {__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv, __uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv};
                            if (vec8) {
                                *reinterpret_cast<uint2 *>(dst + c * 32 + i) = make_uint2(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()));
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e) from_f32(dst[c * 32 + i + e], f[e]);
                            }
                        }
                    }
                }
                if (!whole) part[DPAD * TC_ROWS] = m, part[(DPAD + 1) * TC_ROWS] = l;
            }
            if (!whole && w.from == 0 && threadIdx.x == 0)
                a.joins[blockIdx.x] = make_int4(w.request, w.head, w.tile, attn_block_of(sh.start.total, sh.start.blocks, w.item_begin + w.count - 1));
            more = w.next(a, sh.start);
            if (!more && (whole || w.from != 0) && threadIdx.x == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
        if (!ok && threadIdx.x == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
    }
    pdl_launch_dependents();
}

// The parts of a split tile lie column by column ([DPAD + 2][256], the last two the maximum and the sum): a warp's lanes
// are 32 rows, its columns 16 of the head's.  Block (x, y): the item that block x of the main kernel began, rows 32 y ...
template <class T, int DPAD>
__global__ void __launch_bounds__(DPAD * 2) attn_tc_join_kernel(AttnArgs a) {
    pdl_wait();
    const int4 item = a.joins[blockIdx.x];
    if (item.x < 0) return;
    const AttnRequest q = attn_request(a, item.x);
    const int row = blockIdx.y * 32 + (threadIdx.x & 31), d0 = (threadIdx.x >> 5) * 16, rows = min(TC_ROWS, q.rows - item.z * TC_ROWS);
    if (row >= rows || d0 >= a.head_dim) return;
    const int parts = item.w - (int)blockIdx.x + 1;
    float m = -INFINITY, l = 0.0f, acc[16] = {};
    for (int i = 0; i < parts; ++i) {
        const float *p = a.parts + ((long long)(blockIdx.x + i) * 2 + (i == 0)) * TcShape<DPAD>::PART_FLOATS + row;
        const float pm = p[DPAD * TC_ROWS], pl = p[(DPAD + 1) * TC_ROWS];
        float v[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = p[(d0 + c) * TC_ROWS];
        if (pl == 0.0f) continue;  // a part that saw nothing
        const float top = fmaxf(m, pm), w0 = exp2f(m - top), w1 = exp2f(pm - top);
        l = l * w0 + pl * w1, m = top;
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[c] = acc[c] * w0 + v[c] * w1;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int at = item.z * TC_ROWS + row, token = at / a.group, head = item.y * a.group + at % a.group;
    T *dst = static_cast<T *>(a.out) + (q.first + token) * a.out_stride + (long long)head * a.head_dim + d0;
#pragma unroll
    for (int c = 0; c < 16; ++c)
        if (d0 + c < a.head_dim) from_f32(dst[c], acc[c] * inv);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// A cache as rows of head_dim elements; boxes of 64 columns by the keys that a page and a tile share.
static int attn_map(CUtensorMap *map, const void *cache, const AttnArgs &a, bool bf16) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return TB200_ERR_DRIVER;
    const cuuint64_t dims[2] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.num_pages * a.kv_heads * a.page_size}, strides[1] = {(cuuint64_t)a.head_dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)min(a.page_size, TC_KEYS)}, estr[2] = {1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(cache), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TB200_OK : TB200_ERR_DRIVER;
}

template <class T, int DPAD>
static int attn_tc_launch_dim(AttnArgs a, bool bf16, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    using S = TcShape<DPAD>;
    int st = ensure_kernel<attn_tc_kernel<T, DPAD>, KERNEL_OPTIN_SMEM>(di);
    if (st) return st;
    st = ensure_kernel<attn_tc_join_kernel<T, DPAD>, 0>(di);
    if (st) return st;
    CUtensorMap map_k, map_v;
    st = attn_map(&map_k, a.k_cache, a, bf16);
    if (st) return st;
    st = attn_map(&map_v, a.v_cache, a, bf16);
    if (st) return st;
    const int grid = min(di->sm_count, S::GRID);
    a.joins = static_cast<int4 *>(workspace);
    a.parts = reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + S::GRID * sizeof(int4));
    // kind::f16, fp32 accumulators: operand format at [7,10) and [10,13) (0 = fp16, 1 = bf16), bit 16: B with N contiguous
    const uint32_t fmt = bf16 ? 1u : 0u, common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
    const uint32_t idesc_qk = common | ((TC_KEYS >> 3) << 17), idesc_pv = common | (1u << 16) | ((DPAD >> 3) << 17);
    st = launch_kernel(attn_tc_kernel<T, DPAD>, dim3(grid), dim3(TC_THREADS), S::SMEM, s, false, map_k, map_v, a, idesc_qk, idesc_pv);
    if (st) return st;
    return launch_kernel(attn_tc_join_kernel<T, DPAD>, dim3(grid, min((longest_rows + 31) / 32, TC_ROWS / 32)), dim3(DPAD * 2), 0, s, true, a);
}

// Shapes the kernel takes: heads of up to 128, pages of a power of two of keys from 8 on (a box of 8 rows is the
// swizzle's period), 16-byte aligned caches whose rows a 32-bit coordinate counts.
bool attn_tc_eligible(const AttnArgs &a) {
    return a.head_dim <= 128 && a.page_shift >= 3 && a.num_pages > 0 && aligned_to(a.k_cache, 16) && aligned_to(a.v_cache, 16) &&
           (long long)a.num_pages * a.kv_heads * a.page_size < (1LL << 31) - 1024 && encode_tiled_fn();
}

int attn_tc_launch(const AttnArgs &a, int type, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    const bool bf16 = type == TB200_TYPE_BF16;
    if (a.head_dim <= 64)
        return bf16 ? attn_tc_launch_dim<__nv_bfloat16, 64>(a, true, longest_rows, workspace, di, s) : attn_tc_launch_dim<__half, 64>(a, false, longest_rows, workspace, di, s);
    return bf16 ? attn_tc_launch_dim<__nv_bfloat16, 128>(a, true, longest_rows, workspace, di, s) : attn_tc_launch_dim<__half, 128>(a, false, longest_rows, workspace, di, s);
}

size_t attn_tc_workspace(int head_dim) { return head_dim <= 64 ? TcShape<64>::WORKSPACE : head_dim <= 128 ? TcShape<128>::WORKSPACE : 0; }

}  // namespace tb200
