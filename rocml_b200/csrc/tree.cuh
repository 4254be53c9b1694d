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
    int max_nodes, max_units;        // nodes and tiles of rows of the largest tree
    int cluster;                     // > 1: a (sequence, tile of rows) is shared by the blocks of a cluster, which join what they found themselves
    int4* notes; int n_notes, notes_by_unit;      // see note_of
    float* part_o; float* part_ml;   // [2 shares][nkv][rows_tile][hd], [..][2]
};

struct Seq { int slot, q0, n, ctx, len, first, kept, tiles, units; };   // tiles of 64 keys: [0, kept) and [first, ..]; units: tiles of rows

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int b) {
    Seq s;
    s.slot = a.seq_slot[b];
    s.q0 = a.cu_q[b];
    s.n = a.cu_q[b + 1] - s.q0;
    s.len = a.kv_len[b];
    s.ctx = s.len - s.n;
    // (a sequence shorter than its nodes, or longer than its row of the table, is no sequence: nothing is read or written for it)
    const bool live = s.slot >= 0 && s.n > 0 && s.n <= a.max_nodes && s.ctx >= 0 && s.len <= a.max_pages * PAGE;
    const int lo = a.window > 0 ? max(0, s.ctx - a.window + 1) : 0;       // (positions are >= ctx)
    s.first = min(lo, s.ctx) / PAGE;
    s.kept = a.keep > 0 ? min((a.keep + PAGE - 1) / PAGE, s.first) : 0;
    s.tiles = live ? s.kept + (s.len - 1) / PAGE - s.first + 1 : 0;
    s.units = live ? (s.n * a.group + a.rows_tile - 1) / a.rows_tile : 0;
    return s;
}
__device__ __forceinline__ int tile_of(const Seq& s, int j) { return j < s.kept ? j : s.first + (j - s.kept); }

// What a block pays for beginning and ending a (sequence, tile of rows), and for the masked tiles at its ends, in tiles of keys: each counts as so
// many tiles more when the work is shared out, a third of a share at most.  (Eight sequences of 900 to 9,000 keys under a window of 4,096, 12
// tiles a block: blocks with two pieces took 28 us where those with one took 20.)
constexpr int MAX_EXTRA = 4;

// The work of a key/value head, laid end to end: pre[b] = tiles of keys times tiles of rows of the sequences before b, pre[B] = of all of them, with
// `extra` (returned) more of keys each; tl[b] = tiles of keys of sequence b, with as many more (0: nothing to do).  Every thread of the block calls
// this.
__device__ __forceinline__ int prefix_tiles(const TreeArgs& a, int* pre, int* tl) {
    for (int b = threadIdx.x; b < a.B; b += blockDim.x) {
        const Seq s = seq_of(a, b);
        pre[b + 1] = s.tiles * s.units;
        tl[b] = s.units;
    }
    if (threadIdx.x == 0) pre[0] = 0;
    __syncthreads();
    if (a.B > 1) {
        if (threadIdx.x < 32) {
            int pairs = 0, units = 0;                      // of the sequences before b0
            for (int b0 = 0; b0 < a.B; b0 += 32) {
                const int b = b0 + threadIdx.x;
                int v = b < a.B ? pre[b + 1] : 0, u = b < a.B ? tl[b] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v2 = __shfl_up_sync(0xffffffffu, v, o), u2 = __shfl_up_sync(0xffffffffu, u, o);
                    if ((int)threadIdx.x >= o) { v += v2; u += u2; }
                }
                if (b < a.B) { pre[b + 1] = pairs + v; tl[b] = units + u; }
                pairs += __shfl_sync(0xffffffffu, v, 31);
                units += __shfl_sync(0xffffffffu, u, 31);
            }
        }
        __syncthreads();
    }
    const int extra = min(MAX_EXTRA, pre[a.B] / (3 * a.shares));
    __syncthreads();
    for (int b = threadIdx.x; b < a.B; b += blockDim.x) {
        const int t = seq_of(a, b).tiles;
        pre[b + 1] += extra * tl[b];
        tl[b] = t > 0 ? t + extra : 0;
    }
    __syncthreads();
    return extra;
}
// The sequence that holds pair f (f < pre[B]).
__device__ __forceinline__ int sequence_of(const int* pre, int B, int f) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {                      // the last b with pre[b] <= f
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= f) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// How the blocks of a cluster share a (sequence, tile of rows): `per` tiles of keys each, the last of `parts` blocks what is left, others nothing.
struct ClusterShare {
    int b, mt, rank, tiles, per, parts;
    __device__ ClusterShare(const TreeArgs& a, int block) {
        const int unit = block / a.cluster;
        rank = block - unit * a.cluster;
        b = unit / a.max_units;
        mt = unit - b * a.max_units;
        const Seq s = seq_of(a, b);
        tiles = mt < s.units ? s.tiles : 0;
        per = max(1, (tiles + a.cluster - 1) / a.cluster);
        parts = (tiles + per - 1) / per;
    }
};

// Walks the pieces that one share holds: of a sequence's tiles of rows one after the other, each over all its tiles of keys.
template <bool CLUSTER>
struct Pieces;
template <>
struct Pieces<false> {
    int f, end, b, W, shares, extra, begin;      // begin: where the last piece's (sequence, tile of rows) begins
    __device__ Pieces(const TreeArgs& a, const int* pre, int c, int more) : extra(more) {
        W = pre[a.B];
        shares = max(1, min(a.shares, W));           // (no share between two others is empty: joining counts on it)
        // (64-bit divisions take half a microsecond)
        const bool small = W < 0x7fffffff / (shares + 1);
        f = c >= shares ? 0 : small ? c * W / shares : (int)((long long)c * W / shares);
        end = c >= shares ? 0 : small ? (c + 1) * W / shares : (int)((c + 1ll) * W / shares);
        b = sequence_of(pre, a.B, f);
    }
    // the next piece: tiles of keys [p0, p1) for tile of rows mt of sequence `seq`; false: none is left
    __device__ bool next(const int* pre, const int* tl, int& seq, int& mt, int& p0, int& p1) {
        for (;;) {
            if (f >= end) return false;
            while (pre[b + 1] <= f) ++b;
            const int t = tl[b], off = f - pre[b];
            mt = off / t;
            p0 = off - mt * t;
            begin = f - p0;
            const int stop = min(t, p0 + end - f);
            f += stop - p0;
            if (p0 >= t - extra) continue;            // nothing but what is counted on top
            seq = b;
            p1 = min(stop, t - extra);
            return true;
        }
    }
    // the share that holds pair g: the last c with c W / shares <= g
    __device__ int share_of(int g) const { return (int)(((g + 1ll) * shares - 1) / W); }
};
// A cluster's block has one piece at most.
template <>
struct Pieces<true> {
    int b, mt, f, end;
    __device__ Pieces(const TreeArgs& a, const int*, int block, int) {
        const ClusterShare c(a, block);
        b = c.b;
        mt = c.mt;
        f = c.rank < c.parts ? c.rank * c.per : 0;
        end = c.rank < c.parts ? min(f + c.per, c.tiles) : 0;
    }
    __device__ bool next(const int*, const int*, int& seq, int& tile_of_rows, int& p0, int& p1) {
        if (f >= end) return false;
        seq = b;
        tile_of_rows = mt;
        p0 = f;
        p1 = f = end;
        return true;
    }
};

// What the joining kernel is told, one entry a (sequence, tile of rows) where those are fewer than the shares, else one a share (for what begins in it
// and goes on in the next): {first token, first row, rows, first share << 16 | last share}; equal shares: nothing to join.
__device__ __forceinline__ int4* note_of(const TreeArgs& a, int kvh, int entry) { return a.notes + (size_t)kvh * a.n_notes + entry; }
// One thread of a block calls this for every piece.
__device__ __forceinline__ void note_piece(const TreeArgs& a, const Pieces<false>& p, const Seq& s, int kvh, int c, int b, int mt, int p0, int p1) {
    if (p0 != 0) return;
    const int last = p1 == s.tiles ? c : p.share_of(p.begin + s.tiles - 1);
    const int row0 = mt * a.rows_tile;
    const int4 note = make_int4(s.q0, row0, min(a.rows_tile, s.n * a.group - row0), (c << 16) | last);
    if (a.notes_by_unit) *note_of(a, kvh, b * a.max_units + mt) = note;
    else if (last != c) *note_of(a, kvh, c) = note;
}
// Every thread of a block calls this once: entries that no piece will fill.
__device__ __forceinline__ void note_nothing(const TreeArgs& a, const Pieces<false>& p, const int* pre, const int* tl, int kvh, int c, int tid, int threads) {
    const int4 none = make_int4(0, 0, 0, 0);
    if (a.notes_by_unit) {
        if (c == 0)
            for (int u = tid; u < a.n_notes; u += threads) {
                const int b = u / a.max_units;
                if (tl[b] == 0 || (u % a.max_units) * tl[b] >= pre[b + 1] - pre[b]) *note_of(a, kvh, u) = none;
            }
        return;
    }
    // by shares: this one has an entry if its end cuts the tiles of what began in it
    if (tid == 0 && c < a.n_notes) {
        bool cuts = false;
        if (c + 1 < p.shares && p.f < p.end) {
            const int b = sequence_of(pre, a.B, p.end), into = (p.end - pre[b]) % tl[b];
            cuts = into != 0 && into < tl[b] - p.extra && p.end - into >= p.f;
        }
        if (!cuts) *note_of(a, kvh, c) = none;
    }
}

// Bits [a, b) of 64 (a and b may lie outside).
__device__ __forceinline__ unsigned long long range_bits(int a, int b) {
    a = max(a, 0);
    b = min(b, 64);
    if (a >= b) return 0ull;
    const unsigned long long upto = b == 64 ? ~0ull : (1ull << b) - 1ull;
    return upto & ~((1ull << a) - 1ull);
}
// A row's words of bits, and its position, read once a piece.
constexpr int MAX_WORDS = 8;
struct RowBits {
    unsigned int w[MAX_WORDS];
    int position;
    __device__ void load(const TreeArgs& a, int t) {
#pragma unroll
        for (int i = 0; i < MAX_WORDS; ++i) w[i] = i < a.words ? (unsigned int)a.visible[(size_t)t * a.words + i] : 0u;
        position = a.window > 0 ? a.positions[t] : 0;
    }
    // Which of the 64 keys from key0 on the row (a node of a sequence with context ctx and n nodes) sees.
    __device__ unsigned long long seen(const TreeArgs& a, int ctx, int n, int key0) const {
        unsigned long long m = range_bits(0, ctx - key0);
        if (a.window > 0 && m) {
            const int lo = position - a.window + 1;
            m &= range_bits(lo - key0, 64) | range_bits(0, a.keep - key0);
        }
        const int off = key0 - ctx;                       // the node at the tile's first key
        if (off + 64 > 0 && off < n) {
            const int w0 = off >> 5, sh = off & 31;       // (rounds down below zero too)
            unsigned int x[3] = {0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < MAX_WORDS; ++i) {
#pragma unroll
                for (int j = 0; j < 3; ++j) x[j] = i == w0 + j ? w[i] : x[j];
            }
            const unsigned int lo = __funnelshift_r(x[0], x[1], sh), hi = __funnelshift_r(x[1], x[2], sh);
            m |= (((unsigned long long)hi << 32) | lo) & range_bits(-off, n - off);
        }
        return m;
    }
};

// attention_tree_tc5.cu: bfloat16, head sizes 64, 128 and 256; rows_tile = 128 / group * group.
int launch_tc5(const void* q, long long q_stride, int T, void* out, long long o_stride, const void* k, const void* v, int n_pages,
               const TreeArgs& a, int* status, cudaStream_t stream);
}  // namespace rb_tree
