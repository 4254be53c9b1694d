// What the kernels of attention over trees of drafted tokens share: the call's arguments, which tiles of keys a sequence has, how blocks share
// them, and which keys of a tile a row sees (attention_tree.cu says what is computed).
#pragma once
#include "common.cuh"

namespace rb_tree {
constexpr int PAGE = RB_PAGE;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_BIG = -1e30f;
constexpr int MAX_SEQS = 1024;       // sequences a launch (the prefix sums of their pages are kept in shared memory)

struct TreeArgs {
    const int* block_table; int max_pages;
    const int* seq_slot; const int* cu_q; const int* kv_len;
    const int* visible; int words;
    const int* positions;            // needed with a window only
    int B, nq, nkv, group, hd;
    float scale; int window, keep; float sink; const float* sinks; float softcap;
    int shares, rows_tile;           // rows_tile: rows of a tile that are used, a whole number of nodes for the tensor-core kernel
    float* part_o; float* part_ml;   // [2 shares][gridDim.y tiles][rows_tile][hd], [..][2]
};

struct Seq { int slot, q0, n, ctx, len, first, kept, tiles; };   // tiles of 64 keys: [0, kept) and [first, ..]

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int b, int mt) {
    Seq s;
    s.slot = a.seq_slot[b];
    s.q0 = a.cu_q[b];
    s.n = a.cu_q[b + 1] - s.q0;
    s.len = a.kv_len[b];
    s.ctx = s.len - s.n;
    // (a sequence shorter than its nodes, or longer than its row of the table, is no sequence: nothing is read or written for it)
    const bool live = s.slot >= 0 && s.n > 0 && s.ctx >= 0 && s.len <= a.max_pages * PAGE && mt * a.rows_tile < s.n * a.group;
    const int lo = a.window > 0 ? max(0, s.ctx - a.window + 1) : 0;       // (positions are >= ctx)
    s.first = min(lo, s.ctx) / PAGE;
    s.kept = a.keep > 0 ? min((a.keep + PAGE - 1) / PAGE, s.first) : 0;
    s.tiles = live ? s.kept + (s.len - 1) / PAGE - s.first + 1 : 0;
    return s;
}
__device__ __forceinline__ int tile_of(const Seq& s, int j) { return j < s.kept ? j : s.first + (j - s.kept); }

// pre[b] = tiles of the sequences before b, pre[B] = all of them.  Every thread of the block calls this.
__device__ __forceinline__ void prefix_tiles(const TreeArgs& a, int mt, int* pre) {
    for (int b = threadIdx.x; b < a.B; b += blockDim.x) pre[b + 1] = seq_of(a, b, mt).tiles;
    if (threadIdx.x == 0) pre[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        int carry = 0;
        for (int b0 = 0; b0 < a.B; b0 += 32) {
            const int b = b0 + threadIdx.x;
            int v = b < a.B ? pre[b + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if ((int)threadIdx.x >= o) v += u;
            }
            if (b < a.B) pre[b + 1] = carry + v;
            carry += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
}

// Walks the pieces of sequences that one share holds.
struct Pieces {
    int f, end, b;
    __device__ Pieces(const int* pre, int B, int shares, int c) {
        const long long W = pre[B];
        if (shares > W) shares = max(1, (int)W);           // (no share between two others is empty: the joining kernel counts on it)
        f = c < shares ? (int)(c * W / shares) : 0;
        end = c < shares ? (int)((c + 1) * W / shares) : 0;
        int lo = 0, hi = B - 1;
        while (lo < hi) {                      // the last b with pre[b] <= f (the one that holds page f)
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= f) lo = mid; else hi = mid - 1;
        }
        b = lo;
    }
    // the next piece: tiles [p0, p1) of sequence `seq`; false: none is left
    __device__ bool next(const int* pre, int& seq, int& p0, int& p1) {
        if (f >= end) return false;
        while (pre[b + 1] <= f) ++b;
        seq = b;
        p0 = f - pre[b];
        p1 = min(pre[b + 1], end) - pre[b];
        f += p1 - p0;
        return true;
    }
};

// Bits [a, b) of 64 (a and b may lie outside).
__device__ __forceinline__ unsigned long long range_bits(int a, int b) {
    a = max(a, 0);
    b = min(b, 64);
    if (a >= b) return 0ull;
    const unsigned long long upto = b == 64 ? ~0ull : (1ull << b) - 1ull;
    return upto & ~((1ull << a) - 1ull);
}
// Which of the 64 keys from key0 on row `t` (a node of a sequence with context ctx and n nodes) sees.
__device__ __forceinline__ unsigned long long seen_bits(const TreeArgs& a, int t, int ctx, int n, int key0) {
    unsigned long long m = range_bits(0, ctx - key0);
    if (a.window > 0 && m) {
        const int lo = a.positions[t] - a.window + 1;
        m &= range_bits(lo - key0, 64) | range_bits(0, a.keep - key0);
    }
    const int off = key0 - ctx;                       // the node at the tile's first key
    if (off + 64 > 0 && off < n) {
        const int* row = a.visible + (size_t)t * a.words;
        const int w0 = off >> 5;                      // (rounds down below zero too)
        const int sh = off & 31;
        unsigned int w[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) w[i] = (w0 + i >= 0 && w0 + i < a.words) ? (unsigned int)row[w0 + i] : 0u;
        const unsigned int lo = __funnelshift_r(w[0], w[1], sh), hi = __funnelshift_r(w[1], w[2], sh);
        m |= (((unsigned long long)hi << 32) | lo) & range_bits(-off, n - off);
    }
    return m;
}

// attention_tree_tc5.cu: bfloat16, head sizes 64, 128 and 256; rows_tile = 128 / group * group.
int launch_tc5(const void* q, long long q_stride, int T, void* out, long long o_stride, const void* k, const void* v, int n_pages, int tiles,
               const TreeArgs& a, int* status, cudaStream_t stream);
}  // namespace rb_tree
