// Which drafted nodes a sampler's tokens confirm, and their keys and values moved behind the context.
//
// Node i is like its parent's draw when token[i] == sampled[parent[i]] and no earlier child of that parent has the same token; node
// 0 always is.  It is confirmed when it and all its ancestors are: with the rows of bits that the attention reads
// (ancestors and the node itself) that is (visible_i & ~like) == 0, without a walk from node to node.  The confirmed nodes form one
// path, and a node's place on it is its depth, popcount(visible_i) - 1.
//
// Their keys and values lie at places c + node and belong at c + depth.  A thread owns 16 bytes of one head of one layer for the whole
// path.  Nodes come after their parents, so depth <= node: writing place c + d destroys nothing that a deeper node is still read
// from (its node is larger than d), and a batch of loads ahead of its stores is in order.  Eight loads are in flight a thread; the
// path's rows once in and once out bound the kernel (32 sequences of 7 nodes, 36 layers of 8 heads: 57 MB in 13.5 us).  Every block of a sequence finds the path again (microseconds less than
// a launch of its own would take); the first writes it down.
#include "common.cuh"
#include "api.h"

namespace {
constexpr int MAX_NODES = 256, WORDS = MAX_NODES / 32, THREADS = 256, BATCH = 8;

template <typename Vec>
__global__ void __launch_bounds__(THREADS)
tree_accept_kernel(const int* __restrict__ tokens, const int* __restrict__ parents, const int* __restrict__ visible, int words,
                   const int* __restrict__ sampled, const int* __restrict__ cu_q, int* __restrict__ path, int path_ld,
                   int* __restrict__ counts, int* __restrict__ next_token, const int* __restrict__ seq_slot, const int* __restrict__ kv_len,
                   const int* __restrict__ block_table, int max_pages, Vec* k, Vec* v, int units, int nkv, long long n_pages,
                   int vecs) {
    rb::pdl_trigger();
    rb::pdl_wait();
    __shared__ int first[MAX_NODES], way[MAX_NODES];
    __shared__ unsigned int like_bits[WORDS];
    __shared__ int count;
    __shared__ int2 pages[MAX_NODES];
    const int b = blockIdx.y, tid = threadIdx.x;
    const int slot = seq_slot ? seq_slot[b] : 0, q0 = cu_q[b];
    const int n = min(min(cu_q[b + 1] - q0, words * 32), path_ld);
    if (slot < 0) return;                                // (a sequence without nodes has a path of none)
    first[tid] = MAX_NODES;
    way[tid] = -1;
    if (tid == 0) count = 0;
    __syncthreads();
    int up = -1;
    bool like = false;
    if (tid < n) {
        up = parents[q0 + tid];
        like = up >= 0 && up < tid && tokens[q0 + tid] == sampled[q0 + up];
        if (like) atomicMin(&first[up], tid);
    }
    __syncthreads();
    like = tid < n && (tid == 0 || (like && first[up] == tid));
    const unsigned int ballot = __ballot_sync(0xffffffffu, like);
    if ((tid & 31) == 0) like_bits[tid >> 5] = ballot;
    __syncthreads();
    if (tid < n) {
        bool kept = like;
        int depth = -1;
        for (int w = 0; w * 32 < n; ++w) {
            unsigned int bits = (unsigned int)visible[(size_t)(q0 + tid) * words + w];
            if (n - w * 32 < 32) bits &= (1u << (n - w * 32)) - 1u;
            kept = kept && (bits & ~like_bits[w]) == 0;
            depth += __popc(bits);
        }
        if (kept && depth >= 0 && depth <= tid) {
            way[depth] = tid;
            atomicAdd(&count, 1);
        }
    }
    __syncthreads();
    const int n_path = count;
    if (blockIdx.x == 0) {
        for (int i = tid; i < path_ld; i += THREADS) path[(size_t)b * path_ld + i] = i < n_path ? way[i] : -1;
        if (tid == 0) {
            counts[b] = n_path;
            next_token[b] = n_path > 0 && way[n_path - 1] >= 0 ? sampled[q0 + way[n_path - 1]] : -1;
        }
    }
    if (!k) return;
    const int len = kv_len[b], ctx = len - (cu_q[b + 1] - q0);
    if (ctx < 0 || len > max_pages * RB_PAGE) return;
    // where the path's nodes lie and belong, as rows of a layer's first head (-1: nothing to move; a node that is where it belongs stays)
    if (tid < n_path) {
        const int* table = block_table + (size_t)slot * max_pages;
        const int node = way[tid], src = ctx + node, dst = ctx + tid;
        int from = -1, to = -1;
        if (node > tid) { from = table[src / RB_PAGE]; to = table[dst / RB_PAGE]; }
        first[tid] = from >= 0 && to >= 0 ? src % RB_PAGE : -1;
        pages[tid] = make_int2(from, to);
    }
    __syncthreads();
    // this thread's 16 bytes: unit (keys or values, layer, head) and place inside the head's row
    for (long long at = (long long)blockIdx.x * THREADS + tid; at < (v ? 2ll : 1ll) * units * vecs; at += (long long)gridDim.x * THREADS) {
        const int unit = (int)(at / vecs), col = (int)(at % vecs);
        const int lh = unit < units ? unit : unit - units, layer = lh / nkv, head = lh % nkv;
        Vec* base = (unit < units ? k : v) + (((size_t)layer * n_pages) * nkv + head) * RB_PAGE * vecs + col;
        const size_t page_step = (size_t)nkv * RB_PAGE * vecs;
        for (int d0 = 0; d0 < n_path; d0 += BATCH) {
            Vec x[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
                if (d0 + i < n_path && first[d0 + i] >= 0) x[i] = base[pages[d0 + i].x * page_step + first[d0 + i] * vecs];
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
                if (d0 + i < n_path && first[d0 + i] >= 0) base[pages[d0 + i].y * page_step + (ctx + d0 + i) % RB_PAGE * vecs] = x[i];
        }
    }
}

template <typename Vec>
int launch_accept(const RbAcceptCall& c, cudaStream_t stream) {
    const int vecs = c.row_bytes / (int)sizeof(Vec);
    const long long threads = c.k ? (c.v ? 2ll : 1ll) * c.layers * c.nkv * vecs : 1;
    const long long blocks = (threads + THREADS - 1) / THREADS;
    // about one wave of blocks over all sequences: each finds the path once, whatever it moves
    const long long wave = (5 * 148 + c.n_seqs - 1) / c.n_seqs;
    const unsigned x_blocks = (unsigned)(blocks < wave ? blocks : wave);
    RB_LAUNCH((tree_accept_kernel<Vec>), dim3(x_blocks, c.n_seqs), dim3(THREADS), 0, stream, c.tokens, c.parents, c.visible, c.words, c.sampled, c.cu_q,
              c.path, c.path_ld, c.counts, c.next_token, c.seq_slot, c.kv_len, c.block_table, c.max_pages, (Vec*)c.k, (Vec*)c.v, c.layers * c.nkv, c.nkv,
              c.n_pages, vecs);
    return RB_OK;
}
}  // namespace

// k, v: [layers, n_pages, nkv, 64, row_bytes]; v null: one tensor serves as both; both null: nothing is moved.
extern "C" int rb_tree_accept(const RbAcceptCall* call, void* stream) {
    const RbAcceptCall& c = *call;
    if (c.n_seqs <= 0) return RB_OK;
    if (c.words <= 0 || c.words > WORDS || c.path_ld <= 0 || c.path_ld > MAX_NODES || c.n_seqs > 65535) return RB_ERR_BAD_SIZE;
    if ((c.v && !c.k) || (c.k && c.k == c.v)) return RB_ERR_BAD_SIZE;          // (one tensor for both is moved once)
    if (c.k && (!c.seq_slot || !c.kv_len || !c.block_table || c.layers <= 0 || c.nkv <= 0 || c.row_bytes <= 0 || c.max_pages <= 0)) return RB_ERR_BAD_SIZE;
    cudaStream_t st = (cudaStream_t)stream;
    if (!c.k || (c.row_bytes % 16 == 0 && !(((uintptr_t)c.k | (uintptr_t)c.v) & 15))) return launch_accept<uint4>(c, st);
    if (c.element_bytes == 4 && c.row_bytes % 4 == 0) return launch_accept<uint32_t>(c, st);
    if (c.element_bytes == 2 && c.row_bytes % 2 == 0) return launch_accept<uint16_t>(c, st);
    return RB_ERR_BAD_DTYPE;
}
