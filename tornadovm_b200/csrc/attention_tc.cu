// Attention of chunks of new tokens over a paged cache on the 5th-generation tensor cores.
//
// One persistent block per SM works on tiles of 256 query rows (two of 128, a row per lane of tensor memory; one with heads
// of more than 128 columns) against key tiles of 64:
//   * warp 8 fetches K and V tiles into two rings of shared-memory slots, one TMA box per page and 64 columns (lanes look
//     the pages up side by side, a tile ahead); a page that no row sees, or that is none of the cache's, is fetched from
//     behind the end of the tensor map and arrives as zeros;
//   * warps 9 and 10 issue the tcgen05.mma of one row tile each: S = Q K^T into tensor memory (fp32), and O += P V with P read from tensor memory, where
//     it overlies S.  Each row tile has two score buffers: the product of key tile n + 2 follows that of P(n) V, so that
//     the scores of tile n + 1 are there when the softmax is done with tile n and never waits in the steady state;
//   * warp 11 fetches the query rows;
//   * warps 0-3 and 4-7 hold the softmax of one 128-row tile each, a row per thread: S from tensor memory, the running
//     maximum and sum in registers, P back as 16-bit values.  O stays in tensor memory; it is rescaled only when a row's
//     maximum has grown by more than 2^8 since its reference was set (P then reaches 2^8 at most, 2^15 as
//     fp16 holds it, and the quotient O / l does not depend on the reference), which after the first tiles of a row hardly ever happens.
// Bound: per row tile and key tile two products of 128 x 64 x head_dim, and 128 x 64 powers of two.  The key tiles of all
// items are divided evenly over the blocks and split rows are joined afterwards (attention.cuh).  Code that runs once an
// item stays in rolled loops: unrolled, its instructions arrived from L2 at 15 cycles each (fetching the query rows took
// 15,000 cycles, more than the products of three key tiles).
//
// Every wait is bounded: on expiry the block records TB200_ERR_TIMEOUT, all roles leave their loops, copies in flight are
// waited for (bounded again) and tensor memory is released.
#define TB200_OP_CLASS TB200_PREPARE_LAYER
#include "attention.cuh"
#include "tcgen05.cuh"

TB200_TU_STATUS(attention_tc)

namespace tb200 {

// An item costs its block about as much beside its key tiles (edge tiles, the rows' store) as this many of them.
constexpr int TC_ITEM = 8;
constexpr int TC_KEYS = 64, TC_THREADS = 384;  // three warpgroups
// Registers: 384 threads are launched with 168 each, which the softmax threads (64 scores and 32 words of P in registers) outgrow, so the
// warpgroups share them anew: 2 * 192 + 120 = 3 * 168.
constexpr int TC_SOFTMAX_REGS = 192, TC_OTHER_REGS = 120;
static_assert(2 * TC_SOFTMAX_REGS + TC_OTHER_REGS == 3 * 168, "the shares add up to what the block was launched with");

template <int DPAD>
struct TcShape {
    static constexpr int TILES = DPAD == 256 ? 1 : 2, ROWS = 128 * TILES;  // 256 columns fill tensor and shared memory with one row tile
    static constexpr int PANELS = DPAD / 64;  // 64 columns = 128 bytes: the swizzled rows of a tile
    static constexpr int KV_PANEL = TC_KEYS * 128, KV_BYTES = PANELS * KV_PANEL;   // K or V tile
    static constexpr int Q_PANEL = 128 * 128, Q_BYTES = PANELS * Q_PANEL;          // 128 query rows
    static constexpr int SLOTS = DPAD == 256 ? 2 : DPAD == 128 ? 5 : 10;           // each a K and a V tile
    static constexpr int SMEM = TILES * Q_BYTES + 2 * SLOTS * KV_BYTES + 1024;
    static constexpr int GRID = 148;
    static constexpr size_t PART_FLOATS = (size_t)ROWS * (DPAD + 2);
    static constexpr size_t WORKSPACE = GRID * sizeof(int4) + GRID * 2 * PART_FLOATS * 4;
    // tensor memory: two score buffers of 64 columns for each row tile (P in the first 32 of a buffer), then O_0 and O_1
    static constexpr uint32_t O_COL = 256, TMEM_COLS = 512;
};

// ---- pairs of floats: the packed fp32 instructions do two at once ----
__device__ __forceinline__ uint64_t tc_pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void tc_split(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t tc_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t tc_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
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

// References from which on the step of fp32 matters.  A power of two is that of s * scale - m in one fused step, whose product
// is not rounded; m = max s * scale is, by up to half a step, and from 2^28 on that alone takes fp16 powers beyond their
// range.  Rows of such references round the products first.
__device__ __forceinline__ bool tc_far(float m) { return fabsf(m) >= 0x1p20f && m != -INFINITY; }

// What is taken off a row's scores.  bf16 has fp32's exponents.  An fp16 power is a subnormal below 2^-14, off by up to 2^-25,
// and vanishes from P, though not from the sum, below that: P is raised by 2^7 (2^8 over the reference it reaches 2^15, of
// 2^16), which the sum and O share, so that a long tail of small probabilities is held to 2^-32 of the largest one.  Not
// where a step of fp32 could lift it further.
__device__ __forceinline__ float tc_shift(float m, __nv_bfloat16) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ float tc_shift(float m, __half) { return m == -INFINITY ? 0.0f : tc_far(m) ? m : m - 7.0f; }

struct TcShared {
    uint64_t kv_full[10], kv_empty[10];
    uint64_t q_full[2], q_empty[2], s_full[2][2], p_full[2][2], pv_done[2], o_full[2], drained[2];  // [row tile][score buffer]
    AttnStart start;
    long long scan[32];
    uint32_t tmem_base;
    int abort_flag;
    int odd_values;        // some value of V at an edge was not finite: the rows that see it get it in the epilogue
    uint32_t holes[16];    // per key tile (a ring): pages of the tile that are none of the cache's
};

// Eight 16-bit values; `phase`: an address that dst differs from by a multiple of 16 bytes.
template <class T>
__device__ __forceinline__ void tc_store8(T *dst, const uint32_t (&h)[4], uintptr_t phase) {
    if ((phase & 15) == 0) {
        *reinterpret_cast<uint4 *>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
    } else if ((phase & 3) == 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t *>(dst + 2 * k) = h[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) reinterpret_cast<uint16_t *>(dst)[2 * k] = (uint16_t)h[k], reinterpret_cast<uint16_t *>(dst)[2 * k + 1] = (uint16_t)(h[k] >> 16);
    }
}

// What the rows of an item see.
template <int DPAD>
struct TcItem {
    static constexpr int ROWS = TcShape<DPAD>::ROWS;
    int row0, rows, base, pos_first, pos_last, key_lo, key_hi, tile0, ntiles;
    __device__ __forceinline__ TcItem(const AttnArgs &a, const AttnWalk<ROWS, TC_KEYS, TC_ITEM> &w) {
        row0 = w.tile * ROWS, rows = min(ROWS, w.q.rows - row0), base = w.q.kv_len - w.q.new_tokens;
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
    constexpr int PANELS = S::PANELS, SLOTS = S::SLOTS, ROWS = S::ROWS;
    extern __shared__ __align__(128) unsigned char tc_smem[];
    __shared__ __align__(16) TcShared sh;
    unsigned char *q_s = reinterpret_cast<unsigned char *>(((uintptr_t)tc_smem + 1023) & ~(uintptr_t)1023);  // swizzled tiles: 1024-byte bases
    unsigned char *kv_s = q_s + S::TILES * S::Q_BYTES;  // slot: K tile, V tile
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        sh.abort_flag = 0, sh.odd_values = 0;
        for (int i = 0; i < SLOTS; ++i) mbar_init(&sh.kv_full[i], 1), mbar_init(&sh.kv_empty[i], 2);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 1), mbar_init(&sh.q_empty[i], 1), mbar_init(&sh.pv_done[i], 1), mbar_init(&sh.o_full[i], 1), mbar_init(&sh.drained[i], 1);
            for (int b = 0; b < 2; ++b) mbar_init(&sh.s_full[i][b], 1), mbar_init(&sh.p_full[i][b], 4);
        }
        mbar_fence_init();
    }
    if (warp == 8 && lane == 0) tma_prefetch_map(&map_k), tma_prefetch_map(&map_v);
    attn_find_start<TC_THREADS, ROWS, TC_KEYS, TC_ITEM>(a, &sh.start, sh.scan);
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
    AttnWalk<ROWS, TC_KEYS, TC_ITEM> w;
    bool more = w.seek(a, sh.start), ok = true;
    if (!more && threadIdx.x == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_OTHER_REGS));
    if (warp == 8) {
        // ---------------- producer ----------------
        const int box_keys = min(a.page_size, TC_KEYS), boxes = TC_KEYS / box_keys;
        const int behind = a.num_pages * a.kv_heads * a.page_size;  // first row behind the cache: zeros
        uint32_t nslot = 0, nkv = 0;
        while (more && ok) {
            const TcItem<DPAD> t(a, w);
            const int32_t *table = a.block_table + (long long)w.request * a.max_pages;
            // lane b: row of the cache at which box b of a tile begins, and whether its page is missing
            auto look_up = [&](int n, bool &hole) -> int {
                const int key = (t.tile0 + n) * TC_KEYS + lane * box_keys;
                hole = false;
                if (n >= t.ntiles || lane >= boxes || key > t.key_hi || key + box_keys <= t.key_lo) return behind;
                const int index = key >> a.page_shift, page = table[index];
                hole = page < 0 || page >= a.num_pages;
                return hole ? behind : (page * a.kv_heads + w.head) * a.page_size + (key - (index << a.page_shift));
            };
            // a box per page and panel, from the row that the box's lane has looked up (boxes * PANELS <= 32 lanes)
            auto fetch = [&](const CUtensorMap *map, unsigned char *tile, uint64_t *full, int row) {
                const int y = __shfl_sync(0xffffffffu, row, lane / PANELS);
                if (lane < boxes * PANELS)
                    tma_load_2d(tile + (lane % PANELS) * S::KV_PANEL + (lane / PANELS) * box_keys * 128, map, (lane % PANELS) * 64, y, full);
            };
            // slots in order of use: K(0) | K(1) | V(0), K(2) | V(1), K(3) | ... | V(last)
            const int lead = min(2, t.ntiles);
            bool hole = false, next_hole;
            int row = look_up(0, hole), row1 = behind, row2 = behind;  // rows of tiles i, i - 1, i - 2
#pragma unroll 1
            for (int i = 0; i < t.ntiles + lead; ++i, ++nslot) {
                const int next_row = look_up(i + 1, next_hole);
                const int s = nslot % SLOTS;
                const uint32_t use = nslot / SLOTS;
                if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.kv_empty[s], (use - 1) & 1, abortp));
                if (!ok) break;
                const bool has_k = i < t.ntiles, has_v = i >= lead;
                unsigned char *slot = kv_s + s * 2 * S::KV_BYTES;
                if (has_k) {
                    const uint32_t holes = __ballot_sync(0xffffffffu, hole);
                    if (lane == 0) sh.holes[nkv & 15] = holes;
                    ++nkv;
                }
                if (lane == 0) mbar_expect_tx(&sh.kv_full[s], (has_k ? S::KV_BYTES : 0) + (has_v ? S::KV_BYTES : 0));
                __syncwarp();
                if (has_v) fetch(&map_v, slot + S::KV_BYTES, &sh.kv_full[s], lead == 2 ? row2 : row1);
                if (has_k) fetch(&map_k, slot, &sh.kv_full[s], row);
                row2 = row1, row1 = row, row = next_row, hole = next_hole;
            }
            more = w.next(a, sh.start);
        }
        // copies in flight when a wait has expired (in the normal course all have been waited for by their readers)
        if (!ok && lane == 0)
            for (uint32_t k = nslot > SLOTS ? nslot - SLOTS : 0; k < nslot; ++k)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(&sh.kv_full[k % SLOTS], (k / SLOTS) & 1); ++i) {
                }
    } else if (warp <= 10) {
        // ---------------- products, a warp per row tile ----------------
        // A wait costs this warp some 200 cycles even where nothing is left to wait for, a commit 75, and products are
        // issued at the rate at which they run.  So a row tile has a warp of its own, and a step of it is two waits (the
        // slot with V(n) and K(n + 2); P(n)), twelve products and one commit: the scores' barrier, after which the softmax
        // also releases the slot.  The whole warp walks the loop, so that addresses stay in uniform registers; a lane issues.
        const int t = warp - 9;
        const bool leader = lane == 0;
        uint32_t nslot = 0, q_use = 0, g_s = 0, g_p = 0;  // slots of the block so far; items and score tiles (begun, used) of the row tile
        const uint64_t q_desc = make_smem_desc(smem_u32(q_s) + t * S::Q_BYTES, 16, 1024), k_desc = make_smem_desc(smem_u32(kv_s), 16, 1024);
        const uint64_t v_desc = make_smem_desc(smem_u32(kv_s) + S::KV_BYTES, S::KV_PANEL, 1024);
        // S = Q K^T: both operands K-major, rows of 128 bytes, 16 columns = 32 bytes per instruction
        auto qk = [&](uint32_t slot) {
            const uint64_t k = k_desc + (uint64_t)(slot * (2 * S::KV_BYTES >> 4));
            const uint32_t b = g_s++ & 1, d = tmem + t * 128 + b * 64;
            if (leader) {
#pragma unroll
                for (int i = 0; i < DPAD / 16; ++i)
                    tc_mma_f16(d, q_desc + (uint64_t)(((i / 4) * S::Q_PANEL + (i % 4) * 32) >> 4), k + (uint64_t)(((i / 4) * S::KV_PANEL + (i % 4) * 32) >> 4), idesc_qk, i > 0);
                tc_commit(&sh.s_full[t][b]);
            }
        };
        // O (+)= P V: P in tensor memory (16 keys = 8 columns), V with its columns contiguous, 16 keys = 2048 bytes
        auto pv = [&](uint32_t slot, bool add) {
            const uint64_t v = v_desc + (uint64_t)(slot * (2 * S::KV_BYTES >> 4));
            const uint32_t b = g_p & 1, p = tmem + t * 128 + b * 64, d = tmem + S::O_COL + t * 128;
            if (!__all_sync(0xffffffffu, mbar_wait_abortable(&sh.p_full[t][b], (g_p >> 1) & 1, abortp))) return false;
            ++g_p;
            tc_fence_after();
            if (leader) {
#pragma unroll
                for (int i = 0; i < TC_KEYS / 16; ++i) tc_mma_f16_ta(d, p + i * 8, v + (uint64_t)(i * 128), idesc_pv, add || i > 0);
            }
            return true;
        };
        auto wait_slot = [&]() { return __all_sync(0xffffffffu, mbar_wait_abortable(&sh.kv_full[nslot % SLOTS], (nslot / SLOTS) & 1, abortp)); };
        while (more && ok) {
            const TcItem<DPAD> im(a, w);
            const int lead = min(2, im.ntiles);
            if (t == 1 && im.rows <= 128) {  // nothing to multiply: this row tile's share of the slots is released in turn
#pragma unroll 1
                for (int i = 0; i < im.ntiles + lead && ok; ++i, ++nslot) {
                    ok = wait_slot();
                    if (ok && leader) mbar_arrive(&sh.kv_empty[nslot % SLOTS]);
                }
                more = w.next(a, sh.start);
                continue;
            }
            ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.q_full[t], q_use++ & 1, abortp));
#pragma unroll 1
            for (int n = 0; n < lead && ok; ++n) {
                if (!(ok = wait_slot())) break;
                tc_fence_after();
                qk(nslot++ % SLOTS);
            }
            if (ok && leader && im.ntiles <= 2) tc_commit(&sh.q_empty[t]);
#pragma unroll 1
            for (int n = 0; n < im.ntiles && ok; ++n, ++nslot) {
                const uint32_t slot = nslot % SLOTS;
                if (!(ok = wait_slot())) break;
                if (!(ok = pv(slot, n > 0))) break;
                if (n + 2 < im.ntiles) {
                    qk(slot);
                    if (n + 3 == im.ntiles && leader) tc_commit(&sh.q_empty[t]);
                } else if (leader) {
                    tc_commit(n + 1 == im.ntiles ? &sh.o_full[t] : &sh.pv_done[t]);
                }
            }
            more = w.next(a, sh.start);
        }
        if (leader) {
            tc_commit(&sh.drained[t]);  // nothing of this block's products is under way when tensor memory is released
            for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(&sh.drained[t], 0); ++i) {
            }
        }
        __syncwarp();
    } else {
        // ---------------- query rows ----------------
        // An item's rows go to shared memory by asynchronous copies as soon as the products of the item before have read
        // theirs, which is two key tiles and an epilogue before they are needed.  DPAD / 8 lanes share a row, so that the
        // reads are whole lines.
        const bool q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 8 == 0;
        const int chunks = a.head_dim / 8;
        constexpr int CPR = DPAD / 8, STEP = 32 / CPR;
        const int c = lane % CPR, r0 = lane / CPR, token_step = STEP / a.group, in_step = STEP - token_step * a.group;
        uint32_t use[2] = {0, 0};
        while (more && ok) {
            const int item_rows = min(ROWS, w.q.rows - w.tile * ROWS);
            const T *q = static_cast<const T *>(a.q) + w.q.first * a.q_stride + (long long)w.head * a.group * a.head_dim + c * 8;
#pragma unroll 1
            for (int t = 0; t < 2 && ok && item_rows > t * 128; ++t) {
                if (use[t] > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.q_empty[t], (use[t] - 1) & 1, abortp)))) break;
                ++use[t];
                unsigned char *dst = q_s + t * S::Q_BYTES + (c >> 3) * S::Q_PANEL;
                int row = w.tile * ROWS + t * 128 + r0, token = row / a.group, in = row - token * a.group;  // head of the group
                if (q_vec) {
#pragma unroll 4
                    for (int r = r0; r < 128; r += STEP, row += STEP) {
                        const bool there = row < w.q.rows && c < chunks;
                        const T *src = there ? q + token * a.q_stride + (long long)in * a.head_dim : static_cast<const T *>(a.q);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4))), "l"(src), "r"(there ? 16 : 0)
                                     : "memory");
                        token += token_step, in += in_step;
                        if (in >= a.group) in -= a.group, ++token;
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                } else {
#pragma unroll 1
                    for (int r = r0; r < 128; r += STEP, row += STEP) {
                        const bool there = row < w.q.rows && c < chunks;
                        const uint16_t *src = reinterpret_cast<const uint16_t *>(q + token * a.q_stride + (long long)in * a.head_dim);
                        uint32_t h[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) h[i] = there ? src[i] : 0;
                        *reinterpret_cast<uint4 *>(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                        token += token_step, in += in_step;
                        if (in >= a.group) in -= a.group, ++token;
                    }
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_full[t]);
            }
            more = w.next(a, sh.start);
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_SOFTMAX_REGS));
        // ---------------- softmax ----------------
        const int t = warp >> 2, row_in = threadIdx.x & 127, D = a.head_dim;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + S::O_COL + t * 128;
        uint32_t nkv = 0, nslot = 0, g = 0, o_use = 0, pv_use = 0;  // key tiles and slots of the block so far; score tiles and items of the row tile
        // the next item that has rows for this tile
        auto take_item = [&]() {
            while (more && t == 1 && min(ROWS, w.q.rows - w.tile * ROWS) <= 128) {
                nkv += w.to - w.from, nslot += w.to - w.from + min(2, w.to - w.from);
                more = w.next(a, sh.start);
            }
        };
        take_item();
        while (more && ok) {
            const TcItem<DPAD> im(a, w);
            const int my_row = t * 128 + row_in;
            const bool have = my_row < im.rows, warp_has = t * 128 + (warp & 3) * 32 < im.rows;
            const int pos = have ? im.base + (im.row0 + my_row) / a.group : -1;
            const int see_hi = min(pos, w.q.visible - 1), see_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            const uint64_t scale2 = tc_pair(a.scale_log2, a.scale_log2);
            const int lead = min(2, im.ntiles);
            pv_use += lead - 1;  // an item of two tiles or more commits the last product but one
            float m = -INFINITY, l = 0.0f;
            bool far = false;
#pragma unroll 1
            for (int n = 0; n < im.ntiles; ++n, ++nkv, ++nslot, ++g) {
                const uint32_t b = g & 1;
                ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.s_full[t][b], (g >> 1) & 1, abortp));
                if (!ok) break;
                tc_fence_after();
                if (row_in == 0) mbar_arrive(&sh.kv_empty[nslot % SLOTS]);  // the products that read K(n) and V(n - 2) are done
                const int key0 = (im.tile0 + n) * TC_KEYS;
                const uint32_t holes = sh.holes[nkv & 15];
                const bool edge = key0 + TC_KEYS - 1 > min(im.pos_first, im.key_hi) || (a.window > 0 && key0 <= im.pos_last - a.window);
                uint32_t s[64];
                float top = -INFINITY;
                if (warp_has) {
                    tc_ld_32cols(s_addr + b * 64, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
                    tc_ld_32cols(s_addr + b * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
                    tc_wait_ld();
                    if (__builtin_expect(edge, 0)) {
                        const int lo = see_lo - key0, hi = see_hi - key0;
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (i > hi || i < lo) s[i] = 0xFF800000u;
                    }
                    if (__builtin_expect(holes != 0, 0)) {
                        const int shift = min(a.page_shift, 6);
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if ((holes >> (i >> shift)) & 1) s[i] = 0xFF800000u;
                    }
                    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 64; i += 2) x[(i >> 1) & 3] = max3_nan(x[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                    top = max3_nan(max3_nan(x[0], x[1], x[2]), x[3], x[3]) * a.scale_log2;
                }
                if (__builtin_expect(edge, 0)) {
                    // A place that no row sees may hold anything, and one that some rows see and others do not may hold
                    // an infinity or a NaN: 0 * V would carry it to rows that do not see it.  The former become zeros
                    // here; of the latter the values that are not finite do, and the epilogue gives them to their rows.
                    // (Both tiles' warps do so, two threads a key; they write the same.)
                    const uint32_t vs = nslot + lead;
                    ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.kv_full[vs % SLOTS], (vs / SLOTS) & 1, abortp));
                    if (!ok) break;
                    const int in = row_in >> 1, key = key0 + in;
                    unsigned char *v_row = kv_s + (vs % SLOTS) * 2 * S::KV_BYTES + S::KV_BYTES + in * 128;
                    const bool unseen = key > im.key_hi || key < im.key_lo;
                    if (unseen || key > im.pos_first || (a.window > 0 && key <= im.pos_last - a.window)) {
#pragma unroll 1
                        for (int c = row_in & 1; c < DPAD / 8; c += 2) {
                            uint4 *at = reinterpret_cast<uint4 *>(v_row + (c >> 3) * S::KV_PANEL + (((c & 7) ^ (in & 7)) << 4));
                            const uint4 v = *at;
                            const bool odd = tc_not_finite(v.x, T()) || tc_not_finite(v.y, T()) || tc_not_finite(v.z, T()) || tc_not_finite(v.w, T());
                            if (odd && !unseen) sh.odd_values = 1;
                            if (unseen) *at = make_uint4(0, 0, 0, 0);
                            else if (odd) *at = make_uint4(tc_finite_only(v.x, T()), tc_finite_only(v.y, T()), tc_finite_only(v.z, T()), tc_finite_only(v.w, T()));
                        }
                    }
                    fence_async_shared();
                }
                if (warp_has) {
                    uint64_t by = scale2;
                    if (n == 0) m = top, far = tc_far(m);
                    if (__builtin_expect(__any_sync(0xffffffffu, top - m > 8.0f || far), 0)) {
                        if (__any_sync(0xffffffffu, top - m > 8.0f)) {
                            // The product before this one may still be adding to O.  The next scores' product follows it; behind
                            // the last scores it has a barrier of its own.
                            ok = __all_sync(0xffffffffu, n + 1 < im.ntiles ? mbar_wait_abortable(&sh.s_full[t][b ^ 1], ((g + 1) >> 1) & 1, abortp)
                                                                           : mbar_wait_abortable(&sh.pv_done[t], (pv_use - 1) & 1, abortp));
                            if (!ok) break;
                            tc_fence_after();
                            const float next = fmaxf(m, top), f = next == m ? 1.0f : m == -INFINITY ? 0.0f : tc_ex2(tc_shift(m, T()) - tc_shift(next, T()));
#pragma unroll 1
                            for (int c = 0; c < DPAD / 32; ++c) {
                                uint32_t o[32];
                                tc_ld_32cols(o_addr + c * 32, o);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc_st_32cols(o_addr + c * 32, o);
                            }
                            l *= f, m = next, far = tc_far(m);
                        }
                        if (__any_sync(0xffffffffu, far)) {  // rounded like `top`, so that the difference to m is exact
#pragma unroll
                            for (int i = 0; i < 64; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * a.scale_log2);
                            by = tc_pair(1.0f, 1.0f);
                        }
                    }
                    const float shift = -tc_shift(m, T());
                    const uint64_t shift2 = tc_pair(shift, shift);
                    uint64_t sum[2] = {0, 0};
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float p0, p1;
                        tc_split(tc_fma2(tc_pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), by, shift2), p0, p1);
                        p0 = tc_ex2(p0), p1 = tc_ex2(p1);
                        sum[i & 1] = tc_add2(sum[i & 1], tc_pair(p0, p1));
                        p[i] = pack2(p0, p1, T());  // half a step of `type`, relative to p (fp16: 2^-25 below 2^-14)
                    }
                    tc_st_32cols(s_addr + b * 64, p);
                    float s0, s1;
                    tc_split(tc_add2(sum[0], sum[1]), s0, s1);
                    l += s0 + s1;
                    if (__builtin_expect(!(top < INFINITY), 0)) l = __int_as_float(0x7FC00000);  // a score of +infinity or NaN: the row is NaN
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t][b]);
            }
            if (!ok) break;
            const AttnWalk<ROWS, TC_KEYS, TC_ITEM> done = w;
            const uint32_t nslot_done = nslot;  // the slots of the last products
            nslot += lead;
            more = w.next(a, sh.start);
            const bool last = !more;
            take_item();
            ok = __all_sync(0xffffffffu, mbar_wait_abortable(&sh.o_full[t], o_use++ & 1, abortp));
            if (!ok) break;
            tc_fence_after();
            if (row_in == 0)
                for (int i = 0; i < lead; ++i) mbar_arrive(&sh.kv_empty[(nslot_done + i) % SLOTS]);
            const bool whole = done.whole(), odd = *reinterpret_cast<volatile int *>(&sh.odd_values) != 0;
            if (warp_has) {
                const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
                const int at = im.row0 + my_row, token = at / a.group, head = done.head * a.group + (at - token * a.group);
                T *dst = static_cast<T *>(a.out) + (done.q.first + token) * a.out_stride + (long long)head * D;
                float *part = a.parts + ((long long)blockIdx.x * 2 + (done.from == 0)) * S::PART_FLOATS + my_row;
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
                            const int index = key >> a.page_shift, page = a.block_table[(long long)done.request * a.max_pages + index];
                            if (page < 0 || page >= a.num_pages) continue;
                            const T *v = static_cast<const T *>(a.v_cache) + (((long long)page * a.kv_heads + done.head) * a.page_size + (key - (index << a.page_shift))) * D;
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float f = c * 32 + i < D ? to_f32(v[c * 32 + i]) : 0.0f;
                                if (!(fabsf(f) <= 3.402823466e38f)) o[i] = __float_as_uint(__uint_as_float(o[i]) + f);
                            }
                        }
                    }
                    if (__builtin_expect(l == 0.0f, 0)) {  // saw nothing, or only scores of -infinity, times values that need not be finite
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0;
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) part[(c * 32 + i) * ROWS] = __uint_as_float(o[i]);
                    } else if (have) {
                        T *d = dst + c * 32;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {  // pieces of 8 columns
                            if (c * 32 + i * 8 >= D) break;
                            uint32_t h[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) h[k] = pack2(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv, T());
                            tc_store8(d + i * 8, h, (uintptr_t)d);
                        }
                    }
                }
                if (!whole) part[DPAD * ROWS] = tc_shift(m, T()), part[(DPAD + 1) * ROWS] = l;
            }
            if (threadIdx.x == 0) {
                if (!whole && done.from == 0)
                    a.joins[blockIdx.x] = make_int4(done.request, done.head, done.tile, attn_block_of(sh.start.total, sh.start.blocks, done.item_begin + TC_ITEM + done.count - 1));
                else if (last)
                    a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
            }
            tc_fence_before();  // this item's O has been read before the next one's products are let on it
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

// The parts of a split tile lie column by column ([DPAD + 2][ROWS], the last two the maximum and the sum): a warp's lanes
// are 32 rows, its columns 16 of the head's.  Block (x, y): the item that block x of the main kernel began, every gridDim.y-th
// 32 rows of it from 32 y on.
template <class T, int DPAD>
__global__ void __launch_bounds__(DPAD * 2) attn_tc_join_kernel(AttnArgs a) {
    constexpr int ROWS = TcShape<DPAD>::ROWS;
    pdl_wait();
    const int4 item = a.joins[blockIdx.x];
    if (item.x < 0) return;
    const AttnRequest q = attn_request(a, item.x);
    const int d0 = (threadIdx.x >> 5) * 16, rows = min(ROWS, q.rows - item.z * ROWS), parts = item.w - (int)blockIdx.x + 1;
    if (d0 >= a.head_dim) return;
    // gridDim.y follows a hint, the rows do not
    for (int row = blockIdx.y * 32 + (threadIdx.x & 31); row < rows; row += gridDim.y * 32) {
        float m = -INFINITY, l = 0.0f, acc[16] = {};
        for (int i = 0; i < parts; ++i) {
            const float *p = a.parts + ((long long)(blockIdx.x + i) * 2 + (i == 0)) * TcShape<DPAD>::PART_FLOATS + row;
            const float pm = p[DPAD * ROWS], pl = p[(DPAD + 1) * ROWS];
            float v[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) v[c] = p[(d0 + c) * ROWS];
            if (pl == 0.0f) continue;  // a part that saw nothing
            const float top = fmaxf(m, pm), w0 = exp2f(m - top), w1 = exp2f(pm - top);
            l = l * w0 + pl * w1, m = top;
#pragma unroll
            for (int c = 0; c < 16; ++c) acc[c] = acc[c] * w0 + v[c] * w1;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int at = item.z * ROWS + row, token = at / a.group, head = item.y * a.group + at % a.group;
        T *dst = static_cast<T *>(a.out) + (q.first + token) * a.out_stride + (long long)head * a.head_dim + d0;
        const uintptr_t phase = (uintptr_t)dst;
#pragma unroll
        for (int c = 0; c < 16; c += 8) {  // whole sectors where the alignment allows it
            if (d0 + c >= a.head_dim) break;
            uint32_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = pack2(acc[c + 2 * i] * inv, acc[c + 2 * i + 1] * inv, T());
            tc_store8(dst + c, h, phase);
        }
    }
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
    return launch_kernel(attn_tc_join_kernel<T, DPAD>, dim3(grid, min((longest_rows + 31) / 32, S::ROWS / 32)), dim3(DPAD * 2), 0, s, true, a);
}

// Shapes the kernel takes: heads of up to 256, pages of a power of two of keys from 8 on (a box of 8 rows is the
// swizzle's period), caches whose rows a 32-bit coordinate counts, 16-byte aligned as tensor maps and the start of a copy's
// innermost coordinate have to be.  What it does not take runs in attention.cu: caches at 8 modulo 16 take four chunks of up to
// 512 tokens over 8000 keys from 229 to 1399 us and a prompt of 8192 from 649 to 4441 us, pages of 20 to 1226 and 4171 us.
bool attn_tc_eligible(const AttnArgs &a) {
    return a.head_dim <= 256 && a.page_shift >= 3 && a.num_pages > 0 && aligned_to(a.k_cache, 16) && aligned_to(a.v_cache, 16) &&
           (long long)a.num_pages * a.kv_heads * a.page_size < (1LL << 31) - 1024 && encode_tiled_fn();
}

int attn_tc_launch(const AttnArgs &a, int type, int longest_rows, void *workspace, const DeviceInfo *di, cudaStream_t s) {
    const bool bf16 = type == TB200_TYPE_BF16;
    if (a.head_dim <= 64)
        return bf16 ? attn_tc_launch_dim<__nv_bfloat16, 64>(a, true, longest_rows, workspace, di, s) : attn_tc_launch_dim<__half, 64>(a, false, longest_rows, workspace, di, s);
    if (a.head_dim <= 128)
        return bf16 ? attn_tc_launch_dim<__nv_bfloat16, 128>(a, true, longest_rows, workspace, di, s) : attn_tc_launch_dim<__half, 128>(a, false, longest_rows, workspace, di, s);
    return bf16 ? attn_tc_launch_dim<__nv_bfloat16, 256>(a, true, longest_rows, workspace, di, s) : attn_tc_launch_dim<__half, 256>(a, false, longest_rows, workspace, di, s);
}

size_t attn_tc_workspace(int head_dim) { return head_dim <= 64 ? TcShape<64>::WORKSPACE : head_dim <= 128 ? TcShape<128>::WORKSPACE : TcShape<256>::WORKSPACE; }

}  // namespace tb200
