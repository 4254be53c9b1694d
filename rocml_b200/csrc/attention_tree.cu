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
// Shares.  What is read grows with the contexts, and contexts differ.  So for each (key/value head, row tile) the pages of ALL sequences
// are laid end to end, W of them, and `shares` blocks take W / shares pages each, wherever sequences begin and end: every block
// streams the same number of pages.  A sequence that lies inside one share is finished there; of one that is cut, each share
// leaves (maximum, sum, unnormalised result) in the work space and attention_tree_merge_kernel joins them.  A share is cut at most
// at its two ends, so its work space has two places: 2 c for a sequence that began earlier, 2 c + 1 for one that goes on later.
//
// This file: the entry point, the kernel that joins pieces, and attention_tree_simple_kernel, which takes any head size up to 512 and both types
// with 32-bit multiply-adds.  attention_tree_tc5.cu: bfloat16 heads of 64, 128 and 256 on the tensor cores.
#include "api.h"
#include "per_device.h"
#include "tree.cuh"

using namespace rb_tree;

namespace {
// ---- any head size, both types, 32-bit multiply-adds ------------------------------------------------------------------
// 128 threads, 16 rows by 64 keys a tile, keys and values staged 64 dimensions at a time as float32.  Thread (rg, kg), rg = t / 16, kg = t % 16,
// forms the scores of rows 2 rg, 2 rg + 1 against keys kg + 16 i, and the results of the same rows at dimensions 4 kg .. 4 kg + 3
// of every block of 64: six 16-byte reads of shared memory for 32 multiply-adds in both products.
constexpr int SR = 16, SLD = 68;      // rows a tile; row stride of a staged [64][64] block (68 floats: 16-byte reads of 8 rows miss each other's banks)

template <typename T>
__device__ __forceinline__ void stage64(const T* src, int hd, int d0, int rows, float* dst) {
    // [64 keys][64 dims from d0] of a page of this head; rows beyond `rows` and dimensions beyond hd are zero
    for (int i = threadIdx.x; i < 64 * 16; i += 128) {
        const int r = i >> 4, d = (i & 15) * 4;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            if (hd % 4 == 0) {
                if (d0 + d < hd) rb::load4(src + (size_t)r * hd + d0 + d, x);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d0 + d + e < hd) x[e] = rb::to_f32(src[(size_t)r * hd + d0 + d + e]);
            }
        }
        rb::store4(dst + r * SLD + d, x);
    }
}

template <typename T, int BLOCKS>       // BLOCKS: blocks of 64 dimensions a head, 1, 2, 4 or 8
__global__ void __launch_bounds__(128)
attention_tree_simple_kernel(const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long o_stride,
                             const T* __restrict__ k_cache, const T* __restrict__ v_cache, const TreeArgs a) {
    rb::pdl_trigger();
    rb::pdl_wait();
    extern __shared__ float smem[];
    float* Qs = smem;                              // [16][64 BLOCKS]
    float* Ks = Qs + SR * 64 * BLOCKS;             // [64][SLD]
    float* Vs = Ks + 64 * SLD;
    float* Ps = Vs + 64 * SLD;                     // [16][SLD]
    int* pre = (int*)(Ps + SR * SLD);
    const int tile = blockIdx.y, kvh = tile % a.nkv, mt = tile / a.nkv;
    prefix_tiles(a, mt, pre);
    Pieces pieces(pre, a.B, a.shares, blockIdx.x);
    const int rg = threadIdx.x >> 4, kg = threadIdx.x & 15;
    const float sl2 = a.scale * LOG2E;
    const rb::SoftCap capped = rb::soft_cap(a.scale, a.softcap);
    int b, p0, p1;
    while (pieces.next(pre, b, p0, p1)) {
        const Seq s = seq_of(a, b, mt);
        const int row0 = mt * a.rows_tile, rows = min(SR, s.n * a.group - row0);
        const int* table = a.block_table + (size_t)s.slot * a.max_pages;
        __syncthreads();
        for (int i = threadIdx.x; i < SR * 64 * BLOCKS; i += 128) {
            const int r = i / (64 * BLOCKS), d = i % (64 * BLOCKS);
            float x = 0.f;
            if (r < rows && d < a.hd) {
                const int node = (row0 + r) / a.group, h = (row0 + r) % a.group;
                x = rb::to_f32(q[(size_t)(s.q0 + node) * q_stride + (size_t)(kvh * a.group + h) * a.hd + d]);
            }
            Qs[i] = x;
        }
        float m[2] = {NEG_BIG, NEG_BIG}, l[2] = {0.f, 0.f}, o[BLOCKS][2][4];
#pragma unroll
        for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][r][e] = 0.f;
        for (int j = p0; j < p1; ++j) {
            const int key0 = tile_of(s, j) * PAGE, valid = min(PAGE, s.len - key0);
            const int page = max(0, table[key0 / PAGE]);
            const size_t at = ((size_t)page * a.nkv + kvh) * PAGE * a.hd;
            float sc[2][4] = {};
#pragma unroll 1
            for (int c = 0; c < BLOCKS; ++c) {
                __syncthreads();
                stage64(k_cache + at, a.hd, c * 64, valid, Ks);
                __syncthreads();
#pragma unroll 4
                for (int d = 0; d < 64; d += 4) {
                    float qa[2][4], kb[4][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) rb::load4(Qs + (2 * rg + r) * 64 * BLOCKS + c * 64 + d, qa[r]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) rb::load4(Ks + (kg + 16 * i) * SLD + d, kb[i]);
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) sc[r][i] = fmaf(qa[r][e], kb[i][e], sc[r][i]);
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = row0 + 2 * rg + r;
                const unsigned long long seen = 2 * rg + r < rows ? seen_bits(a, s.q0 + row / a.group, s.ctx, s.n, key0) : 0ull;
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
                    Ps[(2 * rg + r) * SLD + kg + 16 * i] = p;
                }
                l[r] = l[r] * alpha + sum;         // (each thread its own keys; joined at the end)
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c][r][e] *= alpha;
            }
#pragma unroll
            for (int c = 0; c < BLOCKS; ++c) {
                __syncthreads();
                stage64(v_cache + at, a.hd, c * 64, valid, Vs);
                __syncthreads();
#pragma unroll 4
                for (int key = 0; key < 64; key += 4) {
                    float pa[2][4], vb[4][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) rb::load4(Ps + (2 * rg + r) * SLD + key, pa[r]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) rb::load4(Vs + (key + i) * SLD + 4 * kg, vb[i]);
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (pa[r][i] != 0.f) {       // (what a row does not see may hold anything, NaN too)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[c][r][e] = fmaf(pa[r][i], vb[i][e], o[c][r][e]);
                            }
                }
            }
        }
        const bool whole = p0 == 0 && p1 == s.tiles;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
            if (2 * rg + r >= rows) continue;
            const int row = row0 + 2 * rg + r, node = row / a.group, head = kvh * a.group + row % a.group;
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
                const size_t place = ((size_t)(2 * blockIdx.x + (p0 == 0 ? 1 : 0)) * gridDim.y + tile) * a.rows_tile + 2 * rg + r;
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

// ---- joining what several shares have of a sequence --------------------------------------------------------------------
// A warp a row.  Grid (row tiles times quarters of a tile's rows, nkv, sequences).
template <typename T>
__global__ void __launch_bounds__(128)
attention_tree_merge_kernel(T* __restrict__ out, long long o_stride, int n_tiles_y, const TreeArgs a) {
    rb::pdl_trigger();
    rb::pdl_wait();
    __shared__ int sums[2][4];
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_tile = (a.rows_tile + 3) / 4;
    const int mt = blockIdx.x / per_tile, r = blockIdx.x % per_tile * 4 + warp, row = mt * a.rows_tile + r;
    // the tiles before this sequence, and all
    int before = 0, all = 0;
    for (int i = threadIdx.x; i < a.B; i += 128) {
        const int t = seq_of(a, i, mt).tiles;
        all += t;
        if (i < b) before += t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    if (lane == 0) { sums[0][warp] = before; sums[1][warp] = all; }
    __syncthreads();
    before = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
    const long long W = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
    const Seq s = seq_of(a, b, mt);
    if (s.tiles == 0 || r >= a.rows_tile || row >= s.n * a.group) return;
    // share of page f: the last c with c W / shares <= f
    const long long shares = min((long long)a.shares, W);
    const int c0 = (int)((((long long)before + 1) * shares - 1) / W);
    const int c1 = (int)((((long long)before + s.tiles) * shares - 1) / W);
    if (c0 == c1) return;                                     // finished where it lies
    const int tile = mt * a.nkv + kvh;
    const int node = row / a.group, head = kvh * a.group + row % a.group;
    auto place = [&](int c) { return ((size_t)(2 * c + (c == c0 ? 1 : 0)) * n_tiles_y + tile) * a.rows_tile + r; };
    float top = NEG_BIG;
    for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, a.part_ml[place(c) * 2]);
    top = rb::warp_max(top);
    const float sink = (a.sinks ? a.sinks[head] : a.sink) * LOG2E;
    if (rb::has_sink(sink)) top = fmaxf(top, sink);
    float total = 0.f;
    for (int c = c0 + lane; c <= c1; c += 32) total += a.part_ml[place(c) * 2 + 1] * exp2f(a.part_ml[place(c) * 2] - top);
    total = rb::warp_sum(total);
    if (rb::has_sink(sink)) total += exp2f(sink - top);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T* dst = out + (size_t)(s.q0 + node) * o_stride + (size_t)head * a.hd;
    for (int d0 = 0; d0 < a.hd; d0 += 128) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = c0; c <= c1; ++c) {
            const size_t pl = place(c);
            const float f = exp2f(a.part_ml[pl * 2] - top);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = d0 + lane + 32 * e;
                if (d < a.hd) acc[e] = fmaf(f, a.part_o[pl * a.hd + d], acc[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = d0 + lane + 32 * e;
            if (d < a.hd) dst[d] = rb::from_f32<T>(acc[e] * inv);
        }
    }
}

template <typename T, int BLOCKS>
int launch_simple(const void* q, long long q_stride, void* out, long long o_stride, const void* k, const void* v, int tiles, const TreeArgs& a,
                  cudaStream_t stream) {
    const size_t smem = (SR * 64 * BLOCKS + 2 * 64 * SLD + SR * SLD) * sizeof(float) + (a.B + 1) * sizeof(int);
    auto kernel = attention_tree_simple_kernel<T, BLOCKS>;
    static rb::PerDevice<int> allowed;
    int device;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const int* known;
    const int rc = allowed.get(device, &known, [&](int& x) {
        x = 1;
        return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    });
    if (rc) return rc;
    RB_LAUNCH((kernel), dim3(a.shares, tiles), dim3(128), smem, stream, (const T*)q, q_stride, (T*)out, o_stride, (const T*)k, (const T*)v, a);
    return RB_OK;
}

template <typename T>
int launch_any(const void* q, long long q_stride, void* out, long long o_stride, const void* k, const void* v, int tiles, const TreeArgs& a,
               cudaStream_t stream) {
    if (a.hd <= 64) return launch_simple<T, 1>(q, q_stride, out, o_stride, k, v, tiles, a, stream);
    if (a.hd <= 128) return launch_simple<T, 2>(q, q_stride, out, o_stride, k, v, tiles, a, stream);
    if (a.hd <= 256) return launch_simple<T, 4>(q, q_stride, out, o_stride, k, v, tiles, a, stream);
    return launch_simple<T, 8>(q, q_stride, out, o_stride, k, v, tiles, a, stream);
}

template <typename T>
int launch_merge(void* out, long long o_stride, int tiles, const TreeArgs& a, cudaStream_t stream) {
    RB_LAUNCH((attention_tree_merge_kernel<T>), dim3(tiles / a.nkv * ((a.rows_tile + 3) / 4), a.nkv, a.B), dim3(128), 0, stream, (T*)out, o_stride, tiles, a);
    return RB_OK;
}
}  // namespace

// rows_tile: 16, the plain kernel; 128 / group * group, the tensor-core kernel (attention_tree_tc5.cu), which takes aligned rows only.
extern "C" int rb_attention_tree(const void* q, long long q_stride, int T, void* out, long long o_stride, int dtype, const void* k_cache,
                                 const void* v_cache, int n_pages, const int* block_table, int max_pages, const int* seq_slot, const int* cu_q,
                                 const int* kv_len, const int* visible, int words, const int* positions, int n_seqs, int max_nodes, int nq,
                                 int nkv, int hd, float scale, int window, int keep, float sink, const float* sinks, float softcap,
                                 int shares, int rows_tile, float* part_o, float* part_ml, int* status, void* stream) {
    if (n_seqs <= 0 || max_nodes <= 0) return RB_OK;
    if (n_seqs > MAX_SEQS || nkv <= 0 || nq <= 0 || nq % nkv || hd <= 0 || hd > 512 || words <= 0 || shares <= 0 || window < 0 ||
        keep < 0 || !(scale > 0.f) || max_pages <= 0 || (window > 0 && !positions) || (shares > 1 && (!part_o || !part_ml)))
        return RB_ERR_BAD_SIZE;
    if (dtype != RB_F32 && dtype != RB_BF16) return RB_ERR_BAD_DTYPE;
    if (window == 0) keep = 0;
    const int group = nq / nkv;
    const bool tc5 = rows_tile != SR;
    if (tc5 && (dtype != RB_BF16 || (hd != 64 && hd != 128 && hd != 256) || group > 128 || rows_tile != 128 / group * group)) return RB_ERR_BAD_SIZE;
    TreeArgs a{block_table, max_pages, seq_slot, cu_q, kv_len, visible, words, positions, n_seqs, nq, nkv, group, hd,
               scale, window, keep, sink, sinks, softcap, shares, rows_tile, part_o, part_ml};
    const long long m_tiles = ((long long)max_nodes * group + rows_tile - 1) / rows_tile;
    if (m_tiles * nkv > 65535) return RB_ERR_BAD_SIZE;
    const int tiles = (int)m_tiles * nkv;
    cudaStream_t st = (cudaStream_t)stream;
    int rc;
    if (tc5) {
        rc = launch_tc5(q, q_stride, T, out, o_stride, k_cache, v_cache, n_pages, tiles, a, status, st);
    } else {
        const int align = dtype == RB_F32 ? 15 : 7;
        if (hd % 4 == 0 && (((uintptr_t)k_cache & align) || ((uintptr_t)v_cache & align))) return RB_ERR_BAD_ALIGN;
        rc = dtype == RB_F32 ? launch_any<float>(q, q_stride, out, o_stride, k_cache, v_cache, tiles, a, st)
                             : launch_any<__nv_bfloat16>(q, q_stride, out, o_stride, k_cache, v_cache, tiles, a, st);
    }
    if (rc != RB_OK || shares == 1) return rc;
    return dtype == RB_F32 ? launch_merge<float>(out, o_stride, tiles, a, st) : launch_merge<__nv_bfloat16>(out, o_stride, tiles, a, st);
}
