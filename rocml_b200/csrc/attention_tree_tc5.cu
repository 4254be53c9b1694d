// Attention of trees of drafted tokens on the 5th-generation tensor cores: bfloat16, heads of 64, 128 and 256 (attention_tree.cu says what
// is computed and how blocks share the pages).
//
// A block holds 128 rows (a tile of nodes times the query heads of one key/value head: one TMA box gathers them, [nodes][heads][64
// dimensions] with the rows in node order) and walks its share of pages, a page of 64 keys a tile.  S = Q K^T and O += P V are tcgen05.mma with the
// accumulators in tensor memory.  Warp 0 loads (K and V in rings of STAGES pages), warp 1 issues the products, warps 2-5 are the softmax, a thread a
// row.  Every tile costs the same whatever few rows are used: 128 keys of 128 dimensions take the tensor core 1,024 cycles and
// memory, at this multiprocessor's part of the bandwidth, about 2,900, so up to 128 rows the reads decide and the rows are free.  Two blocks share a
// multiprocessor (up to heads of 128): one's products and softmax run beside the other's.
//
// Measured: 100,003 keys on 8 heads, 64 rows, 66 us = 6.2 TB/s; 32 sequences of up to 12,100 keys and trees of 9 to 33 nodes, 4 query heads a
// key/value head, 133 us for 815 MB; a block alone on its multiprocessor 0.95 us a tile, waiting for the ring of two pages.
//
// In a cluster (CLUSTER) a block has one piece and leaves its (maximum, sum, unnormalised result) where Q and the rings were; each block then joins a
// part of the dimensions of all rows, reading its peers' shared memory (a batch of eight parts at a time, none twice: peers that read one block's part
// again for what is not there took 50 us).  How much is read grows with the rows, so large tiles are joined by the second kernel.  One sequence of 709
// keys, 16 rows: 10 us, 12 with two kernels, and 5 us less of the host's time.
//
// A share may hold pieces of several sequences, one after the other: the rings and the two score buffers run on, Q and O are handed over at
// the pieces' ends (q_empty, o_free).  P is rounded to bfloat16 for its product, and the row's sum is that of the rounded weights;
// everything else is 32-bit until the result.
#include "api.h"
#include "per_device.h"
#include "sm100.cuh"
#include "tree.cuh"

using namespace sm100;
using namespace rb_tree;
using rb::ex2;

namespace {
constexpr int BM = 128, BK = 64;
constexpr float RESCALE_AT = 8.0f;       // O is rescaled when a row's maximum has grown by more than 2^8

template <int HD>
struct Sizes {
    static constexpr int HALVES = HD / 64;                       // blocks of 64 dimensions (128 bytes a row, 128-byte swizzle)
    static constexpr int Q_HALF = BM * 128, KV_HALF = BK * 128, KV_TILE = KV_HALF * HALVES;
    static constexpr int STAGES = HD == 64 ? 4 : 2;
    static constexpr int BLOCKS_PER_SM = HD <= 128 ? 2 : 1;
    static constexpr int TILE_BYTES = Q_HALF * HALVES + 2 * STAGES * KV_TILE;
    static constexpr int EXTRA = 1024 + 512 + (2 * MAX_SEQS + 1) * 4;  // alignment, barriers, the sequences' tiles and their sums
    static constexpr int SMEM_BYTES = TILE_BYTES + EXTRA;
    static_assert(BLOCKS_PER_SM * (SMEM_BYTES + 1024) <= 228 * 1024, "the blocks must fit a multiprocessor");
    static constexpr int TMEM_COLS = HD <= 128 ? 256 : 512;      // S0 [0, 64), S1 [64, 128), O [128, 128 + HD)
};

template <int STAGES>
struct Barriers {
    uint64_t q_full, q_empty, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_full[2], o_done, o_final, o_free, checked, drain;
    uint32_t tmem_slot, abort_flag, bad[3][2];
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// A wait that another role's failed wait ends too.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, const uint32_t* abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (*(volatile const uint32_t*)abort_flag != 0 || clock64() - t0 > RB_WAIT_CYCLES) return false;
    }
    return true;
}

// What the blocks of a cluster found for a tile of rows, joined: each takes a part of the dimensions, of all rows; a thread four dimensions of a row.
template <int HD>
__device__ __forceinline__ void join_cluster(const TreeArgs& a, const ClusterShare& share, int kvh, uint32_t part_o, uint32_t part_ml,
                                             __nv_bfloat16* __restrict__ out, long long o_stride) {
    constexpr int BATCH = 8;
    static_assert(HD * BM * 4 <= 2 * Sizes<HD>::STAGES * Sizes<HD>::KV_TILE, "a block's part lies where its rings were");
    const Seq s = seq_of(a, share.b);
    const int row0 = share.mt * a.rows_tile, rows = min(a.rows_tile, s.n * a.group - row0);
    const int d0 = HD / 4 * share.rank / a.cluster, d1 = HD / 4 * (share.rank + 1) / a.cluster;
    for (int i = threadIdx.x; i < (d1 - d0) * rows; i += blockDim.x) {
        const int d = d0 + i / rows, r = i - i / rows * rows;
        const int node = (row0 + r) / a.group, head = kvh * a.group + (row0 + r) % a.group;
        const float sink = (a.sinks ? a.sinks[head] : a.sink) * LOG2E;
        float top = rb::has_sink(sink) ? sink : NEG_BIG, total = rb::has_sink(sink) ? 1.f : 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < share.parts; c0 += BATCH) {
            float m[BATCH], l[BATCH], x[BATCH][4];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                m[j] = NEG_BIG;
                if (c0 + j >= share.parts) continue;
                const int c = c0 + j;
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m[j]), "=f"(l[j]) : "r"(map_to_cta(part_ml, c) + r * 8));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[j][0]), "=f"(x[j][1]), "=f"(x[j][2]), "=f"(x[j][3])
                             : "r"(map_to_cta(part_o, c) + (d * BM + r) * 16));
            }
            float top_new = top;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) top_new = fmaxf(top_new, m[j]);
            const float old = exp2f(top - top_new);
            top = top_new;
            total *= old;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] *= old;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                if (c0 + j >= share.parts) continue;         // (a part of weight zero is added all the same: it may be NaN)
                const float w = exp2f(m[j] - top);
                total = fmaf(l[j], w, total);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = fmaf(x[j][e], w, acc[e]);
            }
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        uint2 y;
        const __nv_bfloat162 lo = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv), hi = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
        y.x = *reinterpret_cast<const uint32_t*>(&lo);
        y.y = *reinterpret_cast<const uint32_t*>(&hi);
        *reinterpret_cast<uint2*>(out + (size_t)(s.q0 + node) * o_stride + (size_t)head * HD + 4 * d) = y;
    }
}

template <int HD, bool CAP, bool CLUSTER>
__global__ void __launch_bounds__(192, Sizes<HD>::BLOCKS_PER_SM)
attention_tree_tc5_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, __nv_bfloat16* __restrict__ out, long long o_stride, const TreeArgs a,
                          int* __restrict__ status) {
    using Z = Sizes<HD>;
    constexpr int HALVES = Z::HALVES, Q_HALF = Z::Q_HALF, KV_HALF = Z::KV_HALF, KV_TILE = Z::KV_TILE, STAGES = Z::STAGES;
    rb::pdl_wait();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* Qs = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* Ks = Qs + Q_HALF * HALVES;
    uint8_t* Vs = Ks + STAGES * KV_TILE;
    auto* bar = (Barriers<STAGES>*)(Vs + STAGES * KV_TILE);
    static_assert(sizeof(Barriers<STAGES>) <= 512, "barriers");
    int* pre = (int*)(Vs + STAGES * KV_TILE + 512);
    int* tl = pre + a.B + 1;
    const int kvh = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(&bar->q_full, 1);
        mbar_init(&bar->q_empty, 1);
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&bar->k_full[i], 1); mbar_init(&bar->k_empty[i], 1);
            mbar_init(&bar->v_full[i], 1); mbar_init(&bar->v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&bar->s_full[i], 1); mbar_init(&bar->p_full[i], 128); }
        mbar_init(&bar->o_done, 1);
        mbar_init(&bar->o_final, 1);
        mbar_init(&bar->o_free, 128);
        mbar_init(&bar->checked, 128);
        mbar_init(&bar->drain, 1);
        bar->abort_flag = 0;
        for (int i = 0; i < 6; ++i) bar->bad[i / 2][i % 2] = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&bar->tmem_slot, Z::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    int extra = 0;
    if (CLUSTER) __syncthreads();
    else extra = prefix_tiles(a, pre, tl);                   // (ends with a block-wide barrier)
    tc_fence_after();
    // Only now may later kernels be scheduled: products take their tensor memory before they wait for this kernel, and one that took a
    // multiprocessor's columns ahead of a block of this grid would wait for it for good.
    rb::pdl_trigger();
    const uint32_t tmem_base = bar->tmem_slot;
    Pieces<CLUSTER> pieces(a, pre, blockIdx.x, extra);
    int b, mt, p0, p1;

    if (warp == 0) {
        if (lane == 0) { tma_prefetch_desc(&map_q); tma_prefetch_desc(&map_k); tma_prefetch_desc(&map_v); }
        const int q_bytes = a.rows_tile * 128 * HALVES;
        bool ok = true;
        int it = 0, piece = 0;             // tiles and pieces so far
        // A piece's lengths and the ids of its first 32 pages are two reads one after the other: they are looked up while the piece before is loaded.
        Seq s{}, s_next{};
        int page = 0, page_next = 0, b_next = 0, mt_next = 0, p0_next = 0, p1_next = 0;
        auto look_ahead = [&]() -> bool {
            if (!pieces.next(pre, tl, b_next, mt_next, p0_next, p1_next)) return false;
            s_next = seq_of(a, b_next);
            page_next = p0_next + lane < p1_next ? a.block_table[(size_t)s_next.slot * a.max_pages + tile_of(s_next, p0_next + lane)] : 0;
            return true;
        };
        bool more = look_ahead();
        while (ok && more) {
            s = s_next; page = max(0, page_next); mt = mt_next; p0 = p0_next; p1 = p1_next;
            more = look_ahead();
            const int* table = a.block_table + (size_t)s.slot * a.max_pages;
            for (int j = p0; j < p1 && ok; ++j, ++it) {
                if (j > p0 && (j - p0) % 32 == 0) page = j + lane < p1 ? max(0, table[tile_of(s, j + lane)]) : 0;      // 32 pages' ids at a time
                const int row = (__shfl_sync(0xffffffffu, page, (j - p0) & 31) * a.nkv + kvh) * PAGE;
                const int st = it % STAGES;
                const uint32_t free_parity = ((it / STAGES) & 1) ^ 1;
                if (lane == 0) {
                    ok = mbar_wait(&bar->k_empty[st], free_parity);
                    if (ok) {
                        mbar_arrive_expect_tx(&bar->k_full[st], KV_TILE);
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) tma_load_2d(Ks + st * KV_TILE + h * KV_HALF, &map_k, h * 64, row, &bar->k_full[st]);
                        if (j == p0) {
                            ok = piece == 0 || mbar_wait(&bar->q_empty, (piece - 1) & 1);
                            if (ok) {
                                mbar_arrive_expect_tx(&bar->q_full, q_bytes);
#pragma unroll
                                for (int h = 0; h < HALVES; ++h)
                                    tma_load_3d(Qs + h * Q_HALF, &map_q, h * 64, kvh * a.group, s.q0 + mt * (a.rows_tile / a.group), &bar->q_full);
                            }
                        }
                        ok = ok && mbar_wait(&bar->v_empty[st], free_parity);
                        if (ok) {
                            mbar_arrive_expect_tx(&bar->v_full[st], KV_TILE);
#pragma unroll
                            for (int h = 0; h < HALVES; ++h) tma_load_2d(Vs + st * KV_TILE + h * KV_HALF, &map_v, h * 64, row, &bar->v_full[st]);
                        }
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            ++piece;
        }
        if (lane == 0) {
            if (!ok) { atomicExch(status, RB_ERR_TIMEOUT); atomicExch(&bar->abort_flag, 1u); }
            // the copies that are still in flight land before the block ends (a stage's last phase, bounded as every wait)
            for (int i = 0; i < STAGES; ++i) {
                const int last = it - 1 - (it - 1 - i + STAGES * 4) % STAGES;      // the last tile of stage i
                if (it > 0 && last >= 0 && !ok) {
                    mbar_wait(&bar->k_full[i], (last / STAGES) & 1, 100000000);
                    mbar_wait(&bar->v_full[i], (last / STAGES) & 1, 100000000);
                }
            }
            if (!ok && piece > 0) mbar_wait(&bar->q_full, (piece - 1) & 1, 100000000);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc_s = idesc_bf16_f32(BM, BK), idesc_o = idesc_bf16_f32_b_mn(BM, HD);
            const uint32_t q_lo = smem_desc_sw128_lo(smem_u32(Qs)), k_lo0 = smem_desc_sw128_lo(smem_u32(Ks));
            const uint32_t v_lo0 = ((smem_u32(Vs) >> 4) & 0x3FFFu) | ((uint32_t)(KV_HALF >> 4) << 16);      // MN-major: the distance of the 64-dimension blocks
            bool ok = true;
            int it = 0, piece = 0;
            // S of tile t into buffer t & 1, which P of tile t - 2 leaves when its product is done.  `done`: the last tile whose product
            // has been asked for (t - 2, at a piece's first tile t - 1): a wait for an earlier one could not tell its phase from the next but one.
            auto issue_s = [&](int t, int done, bool last) -> bool {
                const int st = t % STAGES;
                if (done >= 0 && !mbar_wait(&bar->o_done, done & 1)) return false;
                if (!mbar_wait(&bar->k_full[st], (t / STAGES) & 1)) return false;
                tc_fence_after();
                const uint32_t k_lo = k_lo0 + st * (KV_TILE >> 4), d = tmem_base + (t & 1) * BK;
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    mma_bf16_lo(d, q_lo + (k >> 2) * (Q_HALF >> 4) + (k & 3) * 2, k_lo + (k >> 2) * (KV_HALF >> 4) + (k & 3) * 2, idesc_s, k > 0 ? 1u : 0u);
                mma_commit(&bar->k_empty[st]);
                if (last) mma_commit(&bar->q_empty);
                mma_commit(&bar->s_full[t & 1]);
                return true;
            };
            while (ok && pieces.next(pre, tl, b, mt, p0, p1)) {
                const int n = p1 - p0;
                ok = mbar_wait(&bar->q_full, piece & 1);
                if (ok) { tc_fence_after(); ok = issue_s(it, it - 1, n == 1); }
                for (int j = 0; j < n && ok; ++j, ++it) {
                    if (j + 1 < n && !(ok = issue_s(it + 1, it - 1, j + 2 == n))) break;
                    const int st = it % STAGES;
                    ok = mbar_wait(&bar->p_full[it & 1], (it >> 1) & 1) && mbar_wait(&bar->v_full[st], (it / STAGES) & 1) &&
                         (j > 0 || piece == 0 || mbar_wait(&bar->o_free, (piece - 1) & 1));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t v_lo = v_lo0 + st * (KV_TILE >> 4);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)
                        mma_bf16_ts_lo(tmem_base + 2 * BK, tmem_base + (it & 1) * BK + k * 8, v_lo + k * (2048 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
                    mma_commit(&bar->v_empty[st]);
                    mma_commit(&bar->o_done);
                    if (j == n - 1) mma_commit(&bar->o_final);
                }
                ++piece;
            }
            if (!ok) {
                atomicExch(status, RB_ERR_TIMEOUT);
                atomicExch(&bar->abort_flag, 1u);
                mma_commit(&bar->drain);                 // what was issued is done before tensor memory goes back
                mbar_wait(&bar->drain, 0, 100000000);
            }
        }
    } else {
        const int quarter = warp & 3, r = quarter * 32 + lane, tid = threadIdx.x - 64;
        const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const float sl2 = CAP ? 1.f : a.scale * LOG2E;
        const rb::SoftCap capped = rb::soft_cap(a.scale, a.softcap);
        bool alive = true;
        int it = 0, piece = 0, checks = 0;      // tiles, pieces and masked tiles so far
        if constexpr (!CLUSTER)
            if (a.n_notes) note_nothing(a, pieces, pre, tl, kvh, blockIdx.x, tid, 128);
        while (alive && pieces.next(pre, tl, b, mt, p0, p1)) {
            const Seq s = seq_of(a, b);
            const int row0 = mt * a.rows_tile, rows = min(a.rows_tile, s.n * a.group - row0);
            if constexpr (!CLUSTER)
                if (a.n_notes && tid == 0) note_piece(a, pieces, s, kvh, blockIdx.x, b, mt, p0, p1);
            const bool row_here = r < rows, warp_here = quarter * 32 < rows;
            const int node = (row0 + r) / a.group, head = kvh * a.group + (row0 + r) % a.group;
            float m_used = NEG_BIG, l_sum = 0.f;
            RowBits bits;
            if (row_here) bits.load(a, s.q0 + node);
            int ahead = 0;                           // the furthest position of the tile's nodes, of which a tile has 128 at most
            if (a.window > 0) {
                for (int i = lane; i < rows / a.group; i += 32) ahead = max(ahead, a.positions[s.q0 + row0 / a.group + i]);
                ahead = __reduce_max_sync(0xffffffffu, ahead);
            }
            for (int j = p0; j < p1; ++j, ++it) {
                const int buf = it & 1, st = it % STAGES;
                const int key0 = tile_of(s, j) * BK;
                // a tile inside the context that every node sees whole needs no mask
                const bool whole_tile = key0 + BK <= s.ctx && (a.window == 0 || key0 > ahead - a.window || key0 + BK <= a.keep);
                unsigned long long seen = ~0ull;
                bool spoiled = false;
                // This wait comes before the one for V: scores of this tile say that the product of the tile before last is done, and so that the V before
                // this one in its stage has landed.  Without that the wait for V could take that one's phase for this one's.
                alive = __all_sync(0xffffffffu, wait_or_abort(&bar->s_full[buf], (it >> 1) & 1, &bar->abort_flag));
                if (!alive) break;
                tc_fence_after();
                if (!whole_tile) {
                    seen = row_here ? bits.seen(a, s.ctx, s.n, key0) : 0ull;
                    // Weights of zero still multiply what lies in V: rows past the sequence's end are stale, and a value that is not finite
                    // must not reach a row that does not see it.  Such values become zero here, and the rows that do see them NaN.
                    alive = __all_sync(0xffffffffu, wait_or_abort(&bar->v_full[st], (it / STAGES) & 1, &bar->abort_flag));
                    if (!alive) break;
                    uint8_t* Vt = Vs + st * KV_TILE;
                    constexpr int CHUNKS = HD / 8;
                    const int valid = min(BK, s.len - key0);
                    for (int i = tid; i < BK * CHUNKS; i += 128) {
                        const int vr = i / CHUNKS, ch = i % CHUNKS;
                        uint4* at = reinterpret_cast<uint4*>(Vt + (ch >> 3) * KV_HALF + vr * 128 + (((ch & 7) ^ (vr & 7)) << 4));
                        if (vr >= valid) { *at = make_uint4(0, 0, 0, 0); continue; }
                        uint4 x = *at;
                        // (an exponent of all ones carries into the sign's place)
                        const uint32_t carry = ((x.x & 0x7f807f80u) + 0x00800080u) | ((x.y & 0x7f807f80u) + 0x00800080u) |
                                               ((x.z & 0x7f807f80u) + 0x00800080u) | ((x.w & 0x7f807f80u) + 0x00800080u);
                        if (carry & 0x80008000u) {
                            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
                                if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
                            }
                            *at = make_uint4(w[0], w[1], w[2], w[3]);
                            atomicOr(&bar->bad[checks % 3][vr >> 5], 1u << (vr & 31));
                        }
                    }
                    fence_proxy_async();
                    // Three words of flags in turn: those of the next masked tile are cleared by a thread that has seen everybody arrive at the one before
                    // this, and so be done with the words of the one before that.
                    if (tid == 0) { const int next = (checks + 1) % 3; bar->bad[next][0] = 0; bar->bad[next][1] = 0; }
                    mbar_arrive(&bar->checked);
                    alive = __all_sync(0xffffffffu, wait_or_abort(&bar->checked, checks & 1, &bar->abort_flag));
                    if (!alive) break;
                    const volatile uint32_t* bad = bar->bad[checks % 3];
                    spoiled = (seen & (((unsigned long long)bad[1] << 32) | bad[0])) != 0;
                    ++checks;
                }
                if (warp_here) {
                    float sv[BK];
                    tmem_ld64(lane_base + buf * BK, sv);
                    if (CAP) {
#pragma unroll
                        for (int i = 0; i < BK; ++i) sv[i] = capped(sv[i]);
                    }
                    if (!whole_tile) {
                        const uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            sv[i] = (lo >> i) & 1 ? sv[i] : -INFINITY;
                            sv[32 + i] = (hi >> i) & 1 ? sv[32 + i] : -INFINITY;
                        }
                    }
                    float mxa[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) mxa[q] = fmaxf(sv[2 * q], sv[2 * q + 1]);
#pragma unroll
                    for (int i = 8; i < BK; i += 8) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) mxa[q] = max3(mxa[q], sv[i + 2 * q], sv[i + 2 * q + 1]);
                    }
                    const float mx = fmaxf(fmaxf(mxa[0], mxa[1]), fmaxf(mxa[2], mxa[3])) * sl2;
                    const bool grow = mx - m_used > RESCALE_AT;
                    const float m_new = grow ? mx : m_used;
                    const float alpha = ex2(m_used - m_new);
                    m_used = m_new;
                    l_sum *= alpha;
                    if (j > p0 && __any_sync(0xffffffffu, grow)) {
                        alive = __all_sync(0xffffffffu, wait_or_abort(&bar->o_done, (it - 1) & 1, &bar->abort_flag));
                        if (!alive) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD / 16; ++c) {
                            float ov[16];
                            tmem_ld16(lane_base + 2 * BK + c * 16, ov);
#pragma unroll
                            for (int i = 0; i < 16; ++i) ov[i] *= alpha;
                            tmem_st16(lane_base + 2 * BK + c * 16, ov);
                        }
                    }
                    const uint64_t sl2_2 = pack2(sl2, sl2), neg_m2 = pack2(-m_used, -m_used);
                    uint64_t lacc[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < BK / 32; ++c) {
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float x0, x1;
                            unpack2(fma2(pack2(sv[c * 32 + e], sv[c * 32 + e + 1]), sl2_2, neg_m2), x0, x1);
                            const __nv_bfloat162 h = __floats2bfloat162_rn(ex2(x0), ex2(x1));
                            const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
                            packed[e / 2] = w;
                            // (the sum is of the rounded weights, those that multiply V: a row's weights add up to one, and a row that hangs on few keys
                            // does not carry their rounding)
                            lacc[(e >> 1) & 3] = add2(lacc[(e >> 1) & 3], pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
                        }
                        tmem_st16u(lane_base + buf * BK + c * 16, packed);
                    }
                    float l0, l1;
                    unpack2(add2(add2(lacc[0], lacc[1]), add2(lacc[2], lacc[3])), l0, l1);
                    l_sum += l0 + l1;
                    if (spoiled) l_sum = __int_as_float(0x7fc00000);
                    tmem_st_wait();
                }
                tc_fence_before();
                mbar_arrive(&bar->p_full[buf]);
            }
            if (alive) alive = __all_sync(0xffffffffu, wait_or_abort(&bar->o_final, piece & 1, &bar->abort_flag));
            if (!alive) break;
            tc_fence_after();
            const bool whole = p0 == 0 && p1 == s.tiles;
            if (warp_here) {
                if (whole) {
                    const float sink = (a.sinks && row_here ? a.sinks[head] : a.sink) * LOG2E;
                    if (rb::has_sink(sink)) l_sum += exp2f(fminf(sink - m_used, 126.f));
                }
                const float f = !whole ? 1.f : l_sum == 0.f ? 0.f : 1.f / l_sum;
                // (a place's result is [HD / 4][rows][4]: a warp writes 32 rows' 16 bytes side by side)
                const size_t place = (size_t)(2 * blockIdx.x + (p0 == 0 ? 1 : 0)) * a.nkv + kvh;
                __nv_bfloat16* orow = out + (size_t)(s.q0 + node) * o_stride + (size_t)head * HD;
                // In a cluster it stays in shared memory: the rings' and Q's last reads are done, and no copy is in flight.
                const int part_rows = CLUSTER ? BM : a.rows_tile;
                float* prow = CLUSTER ? reinterpret_cast<float*>(Ks) + r * 4 : a.part_o + place * HD * a.rows_tile + r * 4;
                float* pml = CLUSTER ? reinterpret_cast<float*>(Qs) + r * 2 : a.part_ml + (place * a.rows_tile + r) * 2;
                if (!whole && row_here) *reinterpret_cast<float2*>(pml) = make_float2(m_used, l_sum);
#pragma unroll 1
                for (int c = 0; c < HD / 64; ++c) {
                    float ov[64];
                    tmem_ld64(lane_base + 2 * BK + c * 64, ov);
                    if (!row_here) continue;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const __nv_bfloat162 h = __floats2bfloat162_rn(ov[8 * i + 2 * e] * f, ov[8 * i + 2 * e + 1] * f);
                                w[e] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                            reinterpret_cast<uint4*>(orow + c * 64)[i] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) rb::store4(prow + (size_t)(c * 16 + i) * part_rows * 4, ov + 4 * i);
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(&bar->o_free);
            ++piece;
        }
        if (!alive && lane == 0) atomicExch(status, RB_ERR_TIMEOUT);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, Z::TMEM_COLS);
    }
    if (CLUSTER) {
        __syncwarp();
        const ClusterShare share(a, blockIdx.x);
        if (share.parts < 2) return;                         // (every block of the cluster agrees)
        cluster_arrive();
        cluster_wait();
        join_cluster<HD>(a, share, kvh, smem_u32(Ks), smem_u32(Qs), out, o_stride);
        cluster_arrive();                                    // (a block stays until its shared memory has been read)
        cluster_wait();
    }
}

int encode(CUtensorMap* map, const void* ptr, int dims, const cuuint64_t* size, const cuuint64_t* strides, const cuuint32_t* box) {
    const sm100::EncodeTiledFn fn = sm100::encode_fn();
    if (!fn) return RB_ERR_NO_DRIVER_FN;
    const cuuint32_t steps[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, const_cast<void*>(ptr), size, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? RB_OK : RB_ERR_BAD_SIZE;
}

template <int HD, bool CAP, bool CLUSTER>
int launch(const void* q, long long q_stride, int T, void* out, long long o_stride, const void* k, const void* v, int n_pages,
           const TreeArgs& a, int* status, cudaStream_t stream) {
    CUtensorMap mq, mk, mv;
    const cuuint64_t q_size[3] = {(cuuint64_t)HD, (cuuint64_t)a.nq, (cuuint64_t)T}, q_strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)q_stride * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(a.rows_tile / a.group)};
    const cuuint64_t c_size[2] = {(cuuint64_t)HD, (cuuint64_t)n_pages * a.nkv * PAGE}, c_strides[1] = {(cuuint64_t)HD * 2};
    const cuuint32_t c_box[2] = {64, BK};
    int rc;
    if ((rc = encode(&mq, q, 3, q_size, q_strides, q_box)) != RB_OK || (rc = encode(&mk, k, 2, c_size, c_strides, c_box)) != RB_OK ||
        (rc = encode(&mv, v, 2, c_size, c_strides, c_box)) != RB_OK)
        return rc;
    auto kernel = attention_tree_tc5_kernel<HD, CAP, CLUSTER>;
    static rb::PerDevice<int> allowed;
    int device;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const int* known;
    rc = allowed.get(device, &known, [&](int&) {
        const int bad = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sizes<HD>::SMEM_BYTES);
        return bad || !CLUSTER ? bad : (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (rc) return rc;
    if (CLUSTER)
        return (int)rb::launch_clustered(kernel, dim3(a.B * a.max_units * a.cluster, a.nkv), dim3(192), dim3(a.cluster), Sizes<HD>::SMEM_BYTES, stream, mq,
                                         mk, mv, (__nv_bfloat16*)out, o_stride, a, status);
    RB_LAUNCH((kernel), dim3(a.shares, a.nkv), dim3(192), Sizes<HD>::SMEM_BYTES, stream, mq, mk, mv, (__nv_bfloat16*)out, o_stride, a, status);
    return RB_OK;
}
}  // namespace

namespace rb_tree {
int launch_tc5(const void* q, long long q_stride, int T, void* out, long long o_stride, const void* k, const void* v, int n_pages,
               const TreeArgs& a, int* status, cudaStream_t stream) {
    if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) || q_stride % 8 || o_stride % 8) return RB_ERR_BAD_ALIGN;
    if (T <= 0 || n_pages <= 0 || !status || (long long)n_pages * a.nkv * PAGE > 0x7fffffffll) return RB_ERR_BAD_SIZE;
#define RB_TREE_ARGS q, q_stride, T, out, o_stride, k, v, n_pages, a, status, stream
#define RB_TREE_HD(HD) \
    if (a.hd == HD) { \
        if (a.cluster > 1) return a.softcap > 0.f ? launch<HD, true, true>(RB_TREE_ARGS) : launch<HD, false, true>(RB_TREE_ARGS); \
        return a.softcap > 0.f ? launch<HD, true, false>(RB_TREE_ARGS) : launch<HD, false, false>(RB_TREE_ARGS); \
    }
    RB_TREE_HD(64)
    RB_TREE_HD(128)
    RB_TREE_HD(256)
    return RB_ERR_BAD_SIZE;
#undef RB_TREE_HD
#undef RB_TREE_ARGS
}
}  // namespace rb_tree
