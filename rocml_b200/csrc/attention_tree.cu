// Attention of trees of drafted tokens over the paged cache.
//
// A sequence brings n nodes.  Its context is the c = kv_len - n positions before them; node j's key and value lie at place c + j
// of its pages.  Row (node i, query head h) attends to
//     { places p < c with p > position_i - window, or p < keep }   (window 0: the whole context)
//     and { c + j : bit j of visible_i },
// with softmax in 32 bits (base 2), an optional soft cap on the scores, an optional further term exp(sink) in the denominator.
// A row that sees nothing is zero.  visible: int32 [tokens, words], bit j % 32 of word j / 32.
//
// Rows.  The rows of a (sequence, key/value head) are its nodes times the `group` query heads that share the head, node by
// node: a tile of rows reads every key once for all of them.
//
// Shares.  What is read grows with the contexts, and contexts differ.  So for each key/value head the pages of ALL sequences (as often as
// a sequence has tiles of rows) are laid end to end, W of them, and `shares` blocks take W / shares pages each, wherever sequences begin and
// end: every block streams the same number of pages.  A (sequence, tile of rows) that lies inside one share is finished there; of
// one that is cut, each share leaves (maximum, sum, unnormalised result) in the work space and attention_tree_merge_kernel joins them.  A
// share is cut at most at its two ends, so its work space has two places: 2 c for what began earlier, 2 c + 1 for what goes on later.
//
// Clusters.  Where a sequence's tile of rows has few pages a block, the blocks of a cluster share them instead and join through each other's shared
// memory: no second kernel, no way through memory (tensor-core kernel only; kernels.py has the rule and what it was measured with).
//
// This file: the entry point, the kernel that joins pieces, and attention_tree_simple_kernel, which takes any head size up to 512 and both types
// with 32-bit multiply-adds.  attention_tree_tc5.cu: bfloat16 heads of 64, 128 and 256 on the tensor cores.
#include "api.h"
#include "per_device.h"
#include "tree.cuh"
#include <type_traits>

using namespace rb_tree;

namespace {
// ---- any head size, both types, 32-bit multiply-adds ------------------------------------------------------------------
// 128 threads, 8 RPT rows (16, or 32 where trees have more) by 64 keys a tile.  Keys and values come 64 dimensions at a time, as float32, through a ring of RING blocks of shared memory:
// a tile is its blocks of keys, then its blocks of values, and RING - 1 blocks are asked for ahead of the one in use (32-bit rows by cp.async; staged through
// registers a block waited for memory four times a tile: 10 us).  Thread (rg, kg), rg = t / 16, kg = t % 16, forms the scores of rows RPT rg .. RPT rg + RPT - 1
// against keys kg + 16 i, and the results of the same rows at dimensions 4 kg .. 4 kg + 3 of every block of 64: RPT + 4 16-byte reads of shared
// memory for 16 RPT multiply-adds in both products.  A tile of 128 dimensions takes a block about 5 us (one warp a scheduler, between barriers), which
// bounds short calls; three sequences of up to 1,337 keys, 25 us.
constexpr int SLD = 68;               // row stride of a staged [64][64] block (68 floats: 16-byte reads of 8 rows miss each other's banks)
constexpr int RING = 4;

__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool real) {
    const unsigned int at = (unsigned int)__cvta_generic_to_shared(dst);
    const int bytes = real ? 16 : 0;                   // (the rest is zeros)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(src), "r"(bytes) : "memory");
}
// [64 keys][64 dims from d0] of a page of this head; rows beyond `rows` and dimensions beyond hd are zero
template <typename T>
__device__ __forceinline__ void stage64(const T* src, int hd, int d0, int rows, float* dst) {
    const int d = (threadIdx.x & 15) * 4, r0 = threadIdx.x >> 4;
    if (sizeof(T) == 4 && hd % 4 == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + 8 * i;
            const bool real = r < rows && d0 + d < hd;
            copy_async16(dst + r * SLD + d, real ? src + (size_t)r * hd + d0 + d : src, real);
        }
        return;
    }
    float x[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + 8 * i;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
        if (r < rows) {
            if (hd % 4 == 0) {
                if (d0 + d < hd) rb::load4(src + (size_t)r * hd + d0 + d, x[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d0 + d + e < hd) x[i][e] = rb::to_f32(src[(size_t)r * hd + d0 + d + e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) rb::store4(dst + (r0 + 8 * i) * SLD + d, x[i]);
}

template <typename T, int BLOCKS, int RPT>       // BLOCKS: blocks of 64 dimensions a head, 1, 2, 4 or 8
__global__ void __launch_bounds__(128)
attention_tree_simple_kernel(const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long o_stride,
                             const T* __restrict__ k_cache, const T* __restrict__ v_cache, const TreeArgs a) {
    rb::pdl_trigger();
    rb::pdl_wait();
    constexpr int SR = 8 * RPT;
    extern __shared__ float smem[];
    float* Qs = smem;                              // [SR][64 BLOCKS]
    float* Ring = Qs + SR * 64 * BLOCKS;           // [RING][64][SLD]
    float* Ps = Ring + RING * 64 * SLD;            // [SR][SLD]
    int* pre = (int*)(Ps + SR * SLD);
    int* tl = pre + a.B + 1;
    const int kvh = blockIdx.y;
    const int extra = prefix_tiles(a, pre, tl);
    Pieces<false> pieces(a, pre, blockIdx.x, extra);
    if (a.n_notes) note_nothing(a, pieces, pre, tl, kvh, blockIdx.x, threadIdx.x, 128);
    const int rg = threadIdx.x >> 4, kg = threadIdx.x & 15;
    const float sl2 = a.scale * LOG2E;
    const rb::SoftCap capped = rb::soft_cap(a.scale, a.softcap);
    int b, mt, p0, p1;
    while (pieces.next(pre, tl, b, mt, p0, p1)) {
        const Seq s = seq_of(a, b);
        if (a.n_notes && threadIdx.x == 0) note_piece(a, pieces, s, kvh, blockIdx.x, b, mt, p0, p1);
        const int row0 = mt * a.rows_tile, rows = min(SR, s.n * a.group - row0);
        const int* table = a.block_table + (size_t)s.slot * a.max_pages;
        const int n_blocks = (p1 - p0) * 2 * BLOCKS;
        // block i of the piece: tile p0 + i / (2 BLOCKS), keys before values
        auto fetch = [&](int i) {
            if (i < n_blocks) {
                const int key0 = tile_of(s, p0 + i / (2 * BLOCKS)) * PAGE, c = i % (2 * BLOCKS);
                const size_t at = ((size_t)max(0, table[key0 / PAGE]) * a.nkv + kvh) * PAGE * a.hd;
                stage64((c < BLOCKS ? k_cache : v_cache) + at, a.hd, c % BLOCKS * 64, min(PAGE, s.len - key0), Ring + i % RING * 64 * SLD);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // the next block has landed, and the one before it is free for what comes RING - 1 blocks later
        auto arrive = [&](int i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
            __syncthreads();
            fetch(i + RING - 1);
            return Ring + i % RING * 64 * SLD;
        };
        __syncthreads();
        // the rows' queries, sixteen threads a row; 32-bit rows on 16 bytes in the first group of copies
        const bool q16 = sizeof(T) == 4 && a.hd % 4 == 0 && q_stride % 4 == 0 && ((uintptr_t)q & 15) == 0;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = rg + 8 * i, row = row0 + r, node = row / a.group, h = row - node * a.group;
            const T* src = q + (size_t)(s.q0 + (r < rows ? node : 0)) * q_stride + (size_t)(kvh * a.group + (r < rows ? h : 0)) * a.hd;
#pragma unroll
            for (int c = 0; c < BLOCKS; ++c) {
                const int d = c * 64 + 4 * kg;
                float* dst = Qs + r * 64 * BLOCKS + d;
                if (q16) {
                    const bool real = r < rows && d < a.hd;
                    copy_async16(dst, real ? src + d : src, real);
                } else {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = r < rows && d + e < a.hd ? rb::to_f32(__ldg(src + d + e)) : 0.f;
                    rb::store4(dst, x);
                }
            }
        }
#pragma unroll 1
        for (int i = 0; i < RING - 1; ++i) fetch(i);
        RowBits bits[RPT];
        int ahead = 0;                                 // the furthest position of this thread's rows
#pragma unroll
        for (int r = 0; r < RPT; ++r)
            if (RPT * rg + r < rows) {
                bits[r].load(a, s.q0 + (row0 + RPT * rg + r) / a.group);
                ahead = max(ahead, bits[r].position);
            }
        float m[RPT], l[RPT], o[BLOCKS][RPT][4];
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            m[r] = NEG_BIG;
            l[r] = 0.f;
#pragma unroll
            for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][r][e] = 0.f;
        }
        int block = 0;
        for (int j = p0; j < p1; ++j) {
            const int key0 = tile_of(s, j) * PAGE;
            // a tile inside the context that each of these rows sees whole needs no mask
            const bool whole_tile = key0 + PAGE <= s.ctx && (a.window == 0 || key0 > ahead - a.window || key0 + PAGE <= a.keep);
            float sc[RPT][4] = {};
#pragma unroll 1
            for (int c = 0; c < BLOCKS; ++c) {
                const float* Ks = arrive(block++);
#pragma unroll 4
                for (int d = 0; d < 64; d += 4) {
                    float qa[RPT][4], kb[4][4];
#pragma unroll
                    for (int r = 0; r < RPT; ++r) rb::load4(Qs + (RPT * rg + r) * 64 * BLOCKS + c * 64 + d, qa[r]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) rb::load4(Ks + (kg + 16 * i) * SLD + d, kb[i]);
#pragma unroll
                    for (int r = 0; r < RPT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) sc[r][i] = fmaf(qa[r][e], kb[i][e], sc[r][i]);
                }
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                unsigned long long seen = ~0ull;
                if (!whole_tile) seen = RPT * rg + r < rows ? bits[r].seen(a, s.ctx, s.n, key0) : 0ull;
                float mx = NEG_BIG;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[r][i] = a.softcap > 0.f ? capped(sc[r][i]) : sc[r][i] * sl2;
                    if (!((seen >> (kg + 16 * i)) & 1)) sc[r][i] = -INFINITY;
                    mx = fmaxf(mx, sc[r][i]);
                }
#pragma unroll
                for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
                const float m_new = fmaxf(m[r], mx), alpha = exp2f(m[r] - m_new);
                m[r] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2f(sc[r][i] - m_new);
                    sum += p;
                    Ps[(RPT * rg + r) * SLD + kg + 16 * i] = p;
                }
                l[r] = l[r] * alpha + sum;         // (each thread its own keys; joined at the end)
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c][r][e] *= alpha;
            }
            // What a row does not see may hold anything, NaN too: in a masked tile a weight of zero takes no part.
            auto add_values = [&](float (&oc)[RPT][4], const float* Vs, auto masked) {
#pragma unroll 4
                for (int key = 0; key < 64; key += 4) {
                    float pa[RPT][4], vb[4][4];
#pragma unroll
                    for (int r = 0; r < RPT; ++r) rb::load4(Ps + (RPT * rg + r) * SLD + key, pa[r]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) rb::load4(Vs + (key + i) * SLD + 4 * kg, vb[i]);
#pragma unroll
                    for (int r = 0; r < RPT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (!masked || pa[r][i] != 0.f) oc[r][e] = fmaf(pa[r][i], vb[i][e], oc[r][e]);
                }
            };
#pragma unroll
            for (int c = 0; c < BLOCKS; ++c) {
                const float* Vs = arrive(block++);          // (its barrier also makes Ps whole)
                if (whole_tile) add_values(o[c], Vs, std::false_type());
                else add_values(o[c], Vs, std::true_type());
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        const bool whole = p0 == 0 && p1 == s.tiles;
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
            if (RPT * rg + r >= rows) continue;
            const int row = row0 + RPT * rg + r, node = row / a.group, head = kvh * a.group + row % a.group;
            if (whole) {
                const float sink = (a.sinks ? a.sinks[head] : a.sink) * LOG2E;
                float f = 1.f, total = l[r];
                if (rb::has_sink(sink)) {
                    const float top = fmaxf(m[r], sink);
                    f = exp2f(m[r] - top);
                    total = total * f + exp2f(sink - top);
                }
                const float inv = total == 0.f ? 0.f : f / total;
                T* dst = out + (size_t)(s.q0 + node) * o_stride + (size_t)head * a.hd;
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c * 64 + 4 * kg + e < a.hd) dst[c * 64 + 4 * kg + e] = rb::from_f32<T>(o[c][r][e] * inv);
            } else {
                const size_t place = ((size_t)(2 * blockIdx.x + (p0 == 0 ? 1 : 0)) * a.nkv + kvh) * a.rows_tile + RPT * rg + r;
                if (kg == 0) { a.part_ml[place * 2] = m[r]; a.part_ml[place * 2 + 1] = l[r]; }
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c * 64 + 4 * kg + e < a.hd) a.part_o[place * a.hd + c * 64 + 4 * kg + e] = o[c][r][e];
            }
        }
    }
}

// ---- joining what several shares have of a (sequence, tile of rows) -----------------------------------------------------
// Block (x, head, entry) joins rows 8 x .. 8 x + 7 of what the entry's note names, a warp two rows: the shares' maxima and sums 32 at
// a time, a lane each, then their results, the whole head side by side and eight shares in flight.
constexpr int MERGE_ROWS = 8;
template <typename T, int VEC>              // VEC: dimensions a lane, 32 VEC >= hd
__global__ void __launch_bounds__(128)
attention_tree_merge_kernel(T* __restrict__ out, long long o_stride, const TreeArgs a) {
    rb::pdl_trigger();
    rb::pdl_wait();
    const int kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 note = *note_of(a, kvh, blockIdx.z);
    const int c0 = note.w >> 16, c1 = note.w & 0xffff;
    if (c0 == c1) return;
    for (int r = blockIdx.x * MERGE_ROWS + warp; r < min(note.z, (int)(blockIdx.x + 1) * MERGE_ROWS); r += 4) {
        const int row = note.y + r;
        const int node = row / a.group, head = kvh * a.group + row % a.group;
        auto place = [&](int c) { return ((size_t)(2 * c + (c == c0 ? 1 : 0)) * a.nkv + kvh) * a.rows_tile + r; };
        const float sink = (a.sinks ? a.sinks[head] : a.sink) * LOG2E;
        float top = rb::has_sink(sink) ? sink : NEG_BIG, total = rb::has_sink(sink) ? 1.f : 0.f;
        float acc[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        const int d0 = lane * VEC;
        for (int g = c0; g <= c1; g += 32) {
            const int n = min(32, c1 - g + 1);
            float m = NEG_BIG, l = 0.f;
            if (lane < n) {
                const float2 x = *reinterpret_cast<const float2*>(a.part_ml + place(g + lane) * 2);
                m = x.x;
                l = x.y;
            }
            const float top_new = fmaxf(top, rb::warp_max(m)), old = exp2f(top - top_new), f = exp2f(m - top_new);
            total = total * old + rb::warp_sum(lane < n ? l * f : 0.f);
            top = top_new;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] *= old;
            for (int i0 = 0; i0 < n; i0 += 8) {
                float x[8][VEC];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float* src = a.part_o + place(g + min(i0 + i, n - 1)) * a.hd + d0;
                    if constexpr (VEC % 4 == 0) {
#pragma unroll
                        for (int e = 0; e < VEC; e += 4)
                            if (i0 + i < n && d0 + e < a.hd) rb::load4(src + e, x[i] + e);
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (i0 + i < n && d0 + e < a.hd) x[i][e] = src[e];
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float w = __shfl_sync(0xffffffffu, f, min(i0 + i, 31));
                    if (i0 + i < n) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (d0 + e < a.hd) acc[e] = fmaf(w, x[i][e], acc[e]);
                    }
                }
            }
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        T* dst = out + (size_t)(note.x + node) * o_stride + (size_t)head * a.hd + d0;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (d0 + e < a.hd) dst[e] = rb::from_f32<T>(acc[e] * inv);
    }
}

// The tensor-core kernel's results: [hd / 4][rows][4] a place, a lane a row (that kernel's threads hold a row each, so what a warp writes or reads at
// once is 32 rows' 16 bytes side by side).  A block takes 32 rows.  Its eight warps are `ways` over the shares (the power of two that the number of shares asks for) times
// 8 / ways over blocks of 16 dimensions; each works relative to its own maximum, and they meet in shared memory.  All shares are
// asked for at once that way: one warp over twelve shares in turn took 14 us, eight warps over two shares left six of them idle.
constexpr int JOIN_DIMS = 16, JOIN_WARPS = 8;
__global__ void __launch_bounds__(32 * JOIN_WARPS)
attention_tree_merge_rows_kernel(__nv_bfloat16* __restrict__ out, long long o_stride, const TreeArgs a) {
    rb::pdl_trigger();
    rb::pdl_wait();
    __shared__ float part[JOIN_WARPS][JOIN_DIMS][33], tops[JOIN_WARPS][32], sums[JOIN_WARPS][32];
    __shared__ long long offset[32];
    const int kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row_blocks = (a.rows_tile + 31) / 32, r0 = blockIdx.x % row_blocks * 32;
    const int4 note = *note_of(a, kvh, blockIdx.z);
    const int c0 = note.w >> 16, c1 = note.w & 0xffff;
    if (c0 == c1 || r0 >= note.z) return;
    const int r = min(r0 + lane, note.z - 1), n = c1 - c0 + 1;
    const int ways = n > 8 ? 8 : n > 4 ? 4 : n > 2 ? 2 : 1, chunks = JOIN_WARPS / ways;        // (two shares a warp at a time)
    auto place = [&](int c) { return (size_t)(2 * c + (c == c0 ? 1 : 0)) * a.nkv + kvh; };
    const int step = gridDim.x / row_blocks * chunks * JOIN_DIMS;
    for (int base = blockIdx.x / row_blocks * chunks * JOIN_DIMS; base < a.hd; base += step) {
        const int d0 = base + warp / ways * JOIN_DIMS;
        float top = NEG_BIG, total = 0.f, acc[JOIN_DIMS];
#pragma unroll
        for (int d = 0; d < JOIN_DIMS; ++d) acc[d] = 0.f;
        if (d0 < a.hd) {
            for (int c = c0 + warp % ways; c <= c1; c += 2 * ways) {
                // two shares at a time, all of both asked for before either is used
                float2 ml[2];
                float4 x[2][JOIN_DIMS / 4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int ci = min(c + i * ways, c1);
                    ml[i] = *reinterpret_cast<const float2*>(a.part_ml + (place(ci) * a.rows_tile + r) * 2);
                    const float4* src = reinterpret_cast<const float4*>(a.part_o + (place(ci) * a.hd + d0) * a.rows_tile) + r;
#pragma unroll
                    for (int d = 0; d < JOIN_DIMS / 4; ++d) x[i][d] = src[d * a.rows_tile];
                }
                if (c + ways > c1) ml[1] = make_float2(NEG_BIG, 0.f);
                const float top_new = fmaxf(top, fmaxf(ml[0].x, ml[1].x)), old = exp2f(top - top_new);
                const float w0 = exp2f(ml[0].x - top_new), w1 = c + ways > c1 ? 0.f : exp2f(ml[1].x - top_new);
                top = top_new;
                total = fmaf(total, old, fmaf(ml[0].y, w0, ml[1].y * w1));
#pragma unroll
                for (int d = 0; d < JOIN_DIMS / 4; ++d) {
                    acc[4 * d] = fmaf(acc[4 * d], old, fmaf(x[0][d].x, w0, x[1][d].x * w1));
                    acc[4 * d + 1] = fmaf(acc[4 * d + 1], old, fmaf(x[0][d].y, w0, x[1][d].y * w1));
                    acc[4 * d + 2] = fmaf(acc[4 * d + 2], old, fmaf(x[0][d].z, w0, x[1][d].z * w1));
                    acc[4 * d + 3] = fmaf(acc[4 * d + 3], old, fmaf(x[0][d].w, w0, x[1][d].w * w1));
                }
            }
        }
        __syncthreads();
        tops[warp][lane] = top;
        sums[warp][lane] = total;
#pragma unroll
        for (int d = 0; d < JOIN_DIMS; ++d) part[warp][d][lane] = acc[d];
        __syncthreads();
        // what each way's part of a row is multiplied by, a lane a row (every block of dimensions has the same maxima and sums)
        if (warp == 0) {
            const int row = note.y + r0 + lane, node = row / a.group, head = kvh * a.group + row - node * a.group;
            const float sink = (a.sinks ? a.sinks[min(head, a.nq - 1)] : a.sink) * LOG2E;
            float m = rb::has_sink(sink) ? sink : NEG_BIG;
            for (int w = 0; w < ways; ++w) m = fmaxf(m, tops[w][lane]);
            float l = rb::has_sink(sink) ? exp2f(sink - m) : 0.f;
            for (int w = 0; w < ways; ++w) l = fmaf(sums[w][lane], exp2f(tops[w][lane] - m), l);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            for (int w = 0; w < ways; ++w) sums[w][lane] = exp2f(tops[w][lane] - m) * inv;
            offset[lane] = (long long)(note.x + node) * o_stride + (long long)head * a.hd + base;
        }
        __syncthreads();
        // two neighbouring dimensions of a row a thread and round
        for (int i = threadIdx.x; i < chunks * (JOIN_DIMS / 2) * 32; i += 32 * JOIN_WARPS) {
            const int d = i % (JOIN_DIMS / 2) * 2, rr = i / (JOIN_DIMS / 2) % 32, chunk = i / (JOIN_DIMS / 2 * 32), w0 = chunk * ways;
            if (r0 + rr >= note.z || base + chunk * JOIN_DIMS >= a.hd) continue;
            float y0 = 0.f, y1 = 0.f;
            for (int w = 0; w < ways; ++w) {
                y0 = fmaf(part[w0 + w][d][rr], sums[w][rr], y0);
                y1 = fmaf(part[w0 + w][d + 1][rr], sums[w][rr], y1);
            }
            *reinterpret_cast<__nv_bfloat162*>(out + offset[rr] + chunk * JOIN_DIMS + d) = __floats2bfloat162_rn(y0, y1);
        }
    }
}

template <typename T, int BLOCKS, int RPT>
int launch_simple(const void* q, long long q_stride, void* out, long long o_stride, const void* k, const void* v, const TreeArgs& a,
                  cudaStream_t stream) {
    const size_t smem = (8 * RPT * 64 * BLOCKS + RING * 64 * SLD + 8 * RPT * SLD) * sizeof(float) + (2 * a.B + 1) * sizeof(int);
    auto kernel = attention_tree_simple_kernel<T, BLOCKS, RPT>;
    static rb::PerDevice<int> allowed;
    int device;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const int* known;
    const int rc = allowed.get(device, &known, [&](int& x) {
        x = 1;
        return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    });
    if (rc) return rc;
    RB_LAUNCH((kernel), dim3(a.shares, a.nkv), dim3(128), smem, stream, (const T*)q, q_stride, (T*)out, o_stride, (const T*)k, (const T*)v, a);
    return RB_OK;
}

template <typename T>
int launch_any(const void* q, long long q_stride, void* out, long long o_stride, const void* k, const void* v, const TreeArgs& a,
               cudaStream_t stream) {
    if (a.rows_tile == 32) {                    // (32 rows of more than 256 dimensions do not fit a thread's registers)
        if (a.hd <= 64) return launch_simple<T, 1, 4>(q, q_stride, out, o_stride, k, v, a, stream);
        if (a.hd <= 128) return launch_simple<T, 2, 4>(q, q_stride, out, o_stride, k, v, a, stream);
        return a.hd <= 256 ? launch_simple<T, 4, 4>(q, q_stride, out, o_stride, k, v, a, stream) : RB_ERR_BAD_SIZE;
    }
    if (a.hd <= 64) return launch_simple<T, 1, 2>(q, q_stride, out, o_stride, k, v, a, stream);
    if (a.hd <= 128) return launch_simple<T, 2, 2>(q, q_stride, out, o_stride, k, v, a, stream);
    if (a.hd <= 256) return launch_simple<T, 4, 2>(q, q_stride, out, o_stride, k, v, a, stream);
    return launch_simple<T, 8, 2>(q, q_stride, out, o_stride, k, v, a, stream);
}

template <typename T>
int launch_merge(void* out, long long o_stride, const TreeArgs& a, cudaStream_t stream) {
    const dim3 grid((a.rows_tile + MERGE_ROWS - 1) / MERGE_ROWS, a.nkv, a.n_notes);
    // four dimensions a lane are read together where heads are a whole number of them
    if (a.hd <= 32) RB_LAUNCH((attention_tree_merge_kernel<T, 1>), grid, dim3(128), 0, stream, (T*)out, o_stride, a);
    else if (a.hd <= 128 && a.hd % 4 == 0) RB_LAUNCH((attention_tree_merge_kernel<T, 4>), grid, dim3(128), 0, stream, (T*)out, o_stride, a);
    else if (a.hd <= 256 && a.hd % 4 == 0) RB_LAUNCH((attention_tree_merge_kernel<T, 8>), grid, dim3(128), 0, stream, (T*)out, o_stride, a);
    else if (a.hd % 4 == 0) RB_LAUNCH((attention_tree_merge_kernel<T, 16>), grid, dim3(128), 0, stream, (T*)out, o_stride, a);
    else RB_LAUNCH((attention_tree_merge_kernel<T, 17>), grid, dim3(128), 0, stream, (T*)out, o_stride, a);
    return RB_OK;
}
}  // namespace

// rows_tile: 16 or 32 (heads of up to 256), the plain kernel; 128 / group * group, the tensor-core kernel (attention_tree_tc5.cu), which takes aligned rows only.  work (shares > 1,
// 16-byte aligned): 2 shares * nkv * rows_tile * (hd + 2) floats, then nkv * min(shares - 1, n_seqs * tiles of rows of max_nodes nodes) entries
// of four ints.
extern "C" int rb_attention_tree(const RbTreeCall* call, void* stream) {
    const RbTreeCall& x = *call;
    if (x.n_seqs <= 0 || x.max_nodes <= 0) return RB_OK;
    if (x.n_seqs > MAX_SEQS || x.nkv <= 0 || x.nq <= 0 || x.nq % x.nkv || x.hd <= 0 || x.hd > 512 || x.words <= 0 || x.max_nodes > 32 * x.words ||
        x.shares <= 0 || x.shares > 32767 || x.window < 0 || x.keep < 0 || !(x.scale > 0.f) || x.max_pages <= 0 || x.max_pages > 0x7fffffff / PAGE || (x.window > 0 && !x.positions) ||
        (x.shares > 1 && x.cluster <= 1 && !x.work) || x.nkv > 65535 || x.rows_tile <= 0)
        return RB_ERR_BAD_SIZE;
    if (x.dtype != RB_F32 && x.dtype != RB_BF16) return RB_ERR_BAD_DTYPE;
    if ((uintptr_t)x.work & 15) return RB_ERR_BAD_ALIGN;
    const int group = x.nq / x.nkv;
    const bool tc5 = x.rows_tile != 16 && x.rows_tile != 32;
    if (tc5 && (x.dtype != RB_BF16 || (x.hd != 64 && x.hd != 128 && x.hd != 256) || group > 128 || x.rows_tile != 128 / group * group)) return RB_ERR_BAD_SIZE;
    TreeArgs a{};
    a.block_table = x.block_table; a.max_pages = x.max_pages; a.seq_slot = x.seq_slot; a.cu_q = x.cu_q; a.kv_len = x.kv_len;
    a.visible = x.visible; a.words = x.words; a.positions = x.positions;
    a.B = x.n_seqs; a.nq = x.nq; a.nkv = x.nkv; a.group = group; a.hd = x.hd;
    a.scale = x.scale; a.window = x.window; a.keep = x.window <= 0 ? 0 : x.keep / PAGE < x.max_pages ? x.keep : x.max_pages * PAGE; a.sink = x.sink; a.sinks = x.sinks; a.softcap = x.softcap;
    a.shares = x.shares; a.rows_tile = x.rows_tile; a.max_nodes = x.max_nodes;
    const long long units = ((long long)x.max_nodes * group + x.rows_tile - 1) / x.rows_tile;
    if (units > 0x7fffffff / MAX_SEQS) return RB_ERR_BAD_SIZE;
    a.max_units = (int)units;
    const bool clustered = x.cluster > 1;
    if (clustered && (!tc5 || x.cluster > 16 || x.n_seqs * units * x.cluster > 0x7fffffff)) return RB_ERR_BAD_SIZE;
    a.cluster = x.cluster;
    if (x.shares > 1 && !clustered) {
        const size_t places = 2ull * x.shares * x.nkv * x.rows_tile;
        a.part_o = x.work;
        a.part_ml = x.work + places * x.hd;
        a.notes = reinterpret_cast<int4*>(a.part_ml + places * 2);
        a.notes_by_unit = x.n_seqs * units < x.shares - 1;
        a.n_notes = a.notes_by_unit ? (int)(x.n_seqs * units) : x.shares - 1;
    }
    cudaStream_t st = (cudaStream_t)stream;
    int rc;
    if (tc5) {
        rc = launch_tc5(x.q, x.q_stride, x.tokens, x.out, x.o_stride, x.k_cache, x.v_cache, x.n_pages, a, x.status, st);
    } else {
        const int align = x.dtype == RB_F32 ? 15 : 7;
        if (x.hd % 4 == 0 && (((uintptr_t)x.k_cache & align) || ((uintptr_t)x.v_cache & align))) return RB_ERR_BAD_ALIGN;
        rc = x.dtype == RB_F32 ? launch_any<float>(x.q, x.q_stride, x.out, x.o_stride, x.k_cache, x.v_cache, a, st)
                               : launch_any<__nv_bfloat16>(x.q, x.q_stride, x.out, x.o_stride, x.k_cache, x.v_cache, a, st);
    }
    if (rc != RB_OK || x.shares == 1 || clustered) return rc;
    if (tc5) {
        RB_LAUNCH((attention_tree_merge_rows_kernel), dim3((x.rows_tile + 31) / 32 * (x.hd / (a.notes_by_unit ? JOIN_DIMS : 64)), x.nkv, a.n_notes), dim3(32 * JOIN_WARPS), 0, st, (__nv_bfloat16*)x.out, x.o_stride, a);
        return RB_OK;
    }
    return x.dtype == RB_F32 ? launch_merge<float>(x.out, x.o_stride, a, st) : launch_merge<__nv_bfloat16>(x.out, x.o_stride, a, st);
}
