// Log probabilities of given tokens, the rows' entropy and their most likely tokens, in one pass over the logits.
//
// With c >= 0 chosen near the row's maximum, in base 2:   s = sum 2^(x log2 e - c),   t = sum (x log2 e - c) 2^(x log2 e - c),
//     log sum exp = (c + log2 s) ln 2,   log p(token) = x - log sum exp,   entropy = (log2 s - t / s) ln 2.
// Each thread carries (c, s, t) of its own elements with c its running maximum; triples are joined pairwise.  Sums are 32-bit, the last
// line is 64-bit (c may be large beside what is left of it).
//
// The k most likely, largest first, equal ones by their index.  Beside its triple a thread keeps its largest element (and that
// element's chunk).  All of the k largest elements belong to the k threads whose largest elements lead: any other thread is
// behind k elements already.  So one pass over the row is enough; afterwards only those k threads' elements (k / threads of the
// row) are read again.  Keys are 64-bit whole numbers that order like (value, -index), sorted in registers of a warp, 32 at a time.
//
// A row is read by one block or by the blocks of a cluster, which meet in the first one's shared memory.
#include "common.cuh"
#include "api.h"
#include "per_device.h"
#include "sm100.cuh"

namespace {
constexpr float LOG2E = 1.4426950408889634f;
// Back from base 2 with the very factor that the logits were multiplied by: a 32-bit log2 e is 2^-25 off, which times a logit of 30 would be seen.
constexpr double FROM_LOG2 = 1.0 / (double)LOG2E;
constexpr float NEG_BIG = -1e30f;
constexpr int THREADS = 512, WARPS = THREADS / 32, MAX_TOP = 32;
typedef unsigned long long Key;

// Orders like (x, -index); larger first.  Zero is below every key of an element.
__device__ __forceinline__ Key key_of(float x, int index) {
    const unsigned int u = __float_as_uint(x + 0.f);            // (-0 counts as 0)
    const unsigned int o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((Key)o << 32) | (0xffffffffu - (unsigned int)index);
}
__device__ __forceinline__ float key_value(Key k) {
    const unsigned int o = (unsigned int)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_index(Key k) { return (int)(0xffffffffu - (unsigned int)k); }

__device__ __forceinline__ Key exchange(Key v, int step, bool larger) {
    const Key u = __shfl_xor_sync(0xffffffffu, v, step);
    return larger ? (u > v ? u : v) : (u < v ? u : v);
}
// A warp's 32 keys, lane 0 the largest.
__device__ __forceinline__ Key warp_sort(Key v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1)
            v = exchange(v, step, ((lane & step) == 0) == ((lane & size) == 0 || size == 32));
    return v;
}
// The 32 largest of two sorted runs of 32 (`other` given with its lanes reversed), sorted.
__device__ __forceinline__ Key warp_merge(Key v, Key other_reversed) {
    const int lane = threadIdx.x & 31;
    v = v > other_reversed ? v : other_reversed;
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) v = exchange(v, step, (lane & step) == 0);
    return v;
}

// The larger one, NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

struct Sum { float c, s, t; };
__device__ __forceinline__ Sum join(Sum a, Sum b) {
    const float c = fmaxf(a.c, b.c);
    const float fa = rb::ex2(a.c - c), fb = rb::ex2(b.c - c);
    // (x log2 e - c) = (x log2 e - a.c) + (a.c - c); an empty side (s = 0) brings nothing
    const float ta = a.s > 0.f ? fa * fmaf(a.c - c, a.s, a.t) : fa * a.s, tb = b.s > 0.f ? fb * fmaf(b.c - c, b.s, b.t) : fb * b.s;
    return Sum{c, fmaf(fa, a.s, fb * b.s), ta + tb};
}

template <typename T> struct Chunk;                  // 32 bytes
template <> struct Chunk<float> { static constexpr int E = 8; };
template <> struct Chunk<__nv_bfloat16> { static constexpr int E = 16; };

// The chunk whose first element is `i0` (which may lie before the row, or end after it: -inf there).
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int i0, int V, float* x) {
    constexpr int E = Chunk<T>::E;
    if (i0 >= 0 && i0 + E <= V) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + i0)), b = __ldg(reinterpret_cast<const uint4*>(row + i0) + 1);
        const unsigned int w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (E == 8) x[i] = __uint_as_float(w[i]);
            else { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = i0 + e >= 0 && i0 + e < V ? rb::to_f32(row[i0 + e]) : -INFINITY;
    }
}

struct Shared {
    Key lists[WARPS][32];
    Sum sums[WARPS];
    Key best[32];             // this block's k most likely, sorted
    Sum sum;
};

// The 32 largest of all warps' sorted lists, sorted, in warp 0 (every thread calls this; `v`: the warp's list).
__device__ __forceinline__ Key block_merge(Shared& sh, Key v) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    sh.lists[warp][lane] = v;
#pragma unroll
    for (int half = WARPS / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            v = warp_merge(v, sh.lists[warp + half][31 - lane]);
            sh.lists[warp][lane] = v;
        }
    }
    return v;
}

// The warps' triples joined, by warp 0.
__device__ __forceinline__ void sum_up(Shared& sh) {
    const int lane = threadIdx.x & 31;
    Sum v = lane < WARPS ? sh.sums[lane] : Sum{NEG_BIG, 0.f, 0.f};
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
        Sum other{__shfl_xor_sync(0xffffffffu, v.c, o), __shfl_xor_sync(0xffffffffu, v.s, o), __shfl_xor_sync(0xffffffffu, v.t, o)};
        v = join(v, other);
    }
    if (lane == 0) sh.sum = v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(const T* __restrict__ logits, long long ld, int V, const int* __restrict__ ids, int m, float* __restrict__ logprobs,
                      float* __restrict__ entropy, float* __restrict__ top_logprobs, int* __restrict__ top_ids, int top, int blocks) {
    constexpr int E = Chunk<T>::E;
    rb::pdl_trigger();
    rb::pdl_wait();
    __shared__ Shared sh;
    const int r = blockIdx.x / blocks, part = blockIdx.x % blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* row = logits + (size_t)r * ld;
    // chunks start on 32 bytes: the first may begin before the row
    const int before = (int)(((uintptr_t)row & 31) / sizeof(T));
    const int n_chunks = (V + before + E - 1) / E;
    const int lo = (int)((long long)n_chunks * part / blocks), hi = (int)((long long)n_chunks * (part + 1) / blocks);

    Sum mine{NEG_BIG, 0.f, 0.f};
    float best = -INFINITY;
    int best_chunk = lo + (int)threadIdx.x < hi ? lo + (int)threadIdx.x : -1;
    for (int c = lo + threadIdx.x; c < hi; c += THREADS) {
        float x[E];
        load_chunk(row, c * E - before, V, x);
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < E; ++e) mx = fmaxf(mx, x[e]);
        if (mx > best) { best = mx; best_chunk = c; }
        const float c_new = fmaxf(mine.c, mx * LOG2E);
        const float f = rb::ex2(mine.c - c_new);
        mine.t = mine.s > 0.f ? f * fmaf(mine.c - c_new, mine.s, mine.t) : f * mine.s;
        mine.s *= f;
        mine.c = c_new;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = max_nan(fmaf(x[e], LOG2E, -c_new), -1000.f);       // (-inf: 2^-1000 is 0, and so is 0 times -1000)
            const float p = rb::ex2(d);
            mine.s += p;
            mine.t = fmaf(d, p, mine.t);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sum other{__shfl_xor_sync(0xffffffffu, mine.c, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.t, o)};
        mine = join(mine, other);
    }
    if (lane == 0) sh.sums[warp] = mine;
    __syncthreads();
    if (warp == 0) sum_up(sh);
    if (top > 0) {
        // the threads whose largest elements lead (by value, then chunk: chunks of different threads differ)
        Key v = block_merge(sh, warp_sort(best_chunk >= 0 ? key_of(best, best_chunk) : 0ull));
        if (warp == 0) sh.best[lane] = v;
        __syncthreads();
        const Key last = sh.best[top - 1];
        const float least = last ? key_value(last) : -INFINITY;
        Key found = 0ull;
        for (int j = warp; j < top; j += WARPS) {
            const Key lead = sh.best[j];
            if (!lead) break;
            const int c0 = lo + (key_index(lead) - lo) % THREADS;
            for (int cb = c0; cb < hi; cb += 32 * THREADS) {
                const int c = cb + lane * THREADS, i0 = c * E - before;
                float x[E];
                if (c < hi) load_chunk(row, i0, V, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    // (what is not ahead of the k-th found so far is not sorted in: rows of many equal values end quickly)
                    const bool may = c < hi && i0 + e >= 0 && i0 + e < V && x[e] >= least;
                    if (!__any_sync(0xffffffffu, may)) continue;
                    Key key = may ? key_of(x[e], i0 + e) : 0ull;
                    if (!__any_sync(0xffffffffu, key > __shfl_sync(0xffffffffu, found, top - 1))) continue;
                    key = warp_sort(key);
                    found = warp_merge(found, __shfl_sync(0xffffffffu, key, 31 - lane));
                }
            }
        }
        v = block_merge(sh, found);
        if (warp == 0) sh.best[lane] = v;
    }
    __syncthreads();
    if (blocks > 1) {
        // the first block of the cluster reads what the others found, a warp a block
        sm100::cluster_arrive();
        sm100::cluster_wait();
        if (part == 0) {
            Sum v{NEG_BIG, 0.f, 0.f};
            Key k = 0ull;
            if (warp < blocks) {
                const uint32_t at = sm100::map_to_cta(sm100::smem_u32(&sh.sum), warp);
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v.c) : "r"(at));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v.s) : "r"(at + 4));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v.t) : "r"(at + 8));
                if (top > 0)
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(sm100::map_to_cta(sm100::smem_u32(&sh.best[lane]), warp)));
            }
            if (lane == 0) sh.sums[warp] = v;
            if (top > 0) k = block_merge(sh, k);
            __syncthreads();
            if (warp == 0) {
                sum_up(sh);
                if (top > 0) sh.best[lane] = k;
            }
            __syncthreads();
        }
        sm100::cluster_arrive();
        sm100::cluster_wait();
        if (part != 0) return;
    }
    const Sum all = sh.sum;
    const float log_s = log2f(all.s);
    const double lse = ((double)all.c + (double)log_s) * FROM_LOG2;
    const bool nothing = all.s == 0.f;                   // every logit -inf: nothing has a probability
    if (entropy && threadIdx.x == 0) entropy[r] = nothing ? 0.f : (float)((double)(log_s - all.t / all.s) * FROM_LOG2);
    for (int j = threadIdx.x; j < m; j += THREADS) {
        const int id = ids[(size_t)r * m + j];
        logprobs[(size_t)r * m + j] = id < 0 || id >= V || nothing ? -INFINITY : (float)((double)rb::to_f32(row[id]) - lse);
    }
    if ((int)threadIdx.x < top) {
        const Key k = sh.best[threadIdx.x];
        if (top_ids) top_ids[(size_t)r * top + threadIdx.x] = k ? key_index(k) : -1;
        if (top_logprobs) top_logprobs[(size_t)r * top + threadIdx.x] = !k || nothing ? -INFINITY : (float)((double)key_value(k) - lse);
    }
}
}  // namespace

// logits [n, V] (row stride ld elements); ids int32 [n, m]; logprobs float32 [n, m]; entropy float32 [n] or null; top_logprobs float32 and
// top_ids int32 [n, top], top <= 32.  blocks: 1, 2, 4, 8 or 16 blocks a row.
extern "C" int rb_token_logprobs(const void* logits, int dtype, long long ld, int n, int V, const int* ids, int m, float* logprobs,
                                 float* entropy, float* top_logprobs, int* top_ids, int top, int blocks, void* stream) {
    if (n <= 0) return RB_OK;
    if (V <= 0 || V > (1 << 30) || m < 0 || top < 0 || top > MAX_TOP || top > V || (m > 0 && (!ids || !logprobs)) || blocks < 1 || blocks > 16 ||
        (blocks & (blocks - 1)) || (long long)n * blocks > 0x7fffffffll)
        return RB_ERR_BAD_SIZE;
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto kernel, auto* x, rb::PerDevice<int>& allowed) -> int {
        if (blocks == 1) {
            RB_LAUNCH((kernel), dim3(n), dim3(THREADS), 0, st, x, ld, V, ids, m, logprobs, entropy, top_logprobs, top_ids, top, blocks);
            return RB_OK;
        }
        int device;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return (int)e;
        const int* known;
        const int rc = allowed.get(device, &known, [&](int&) { return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
        if (rc) return rc;
        e = rb::launch_clustered(kernel, dim3(n * blocks), dim3(THREADS), dim3(blocks), 0, st, x, ld, V, ids, m, logprobs, entropy, top_logprobs,
                                 top_ids, top, blocks);
        return (int)e;
    };
    static rb::PerDevice<int> allowed_f32, allowed_bf16;
    if (dtype == RB_F32) return ((uintptr_t)logits & 3) ? RB_ERR_BAD_ALIGN : go(token_logprobs_kernel<float>, (const float*)logits, allowed_f32);
    if (dtype == RB_BF16) return ((uintptr_t)logits & 1) ? RB_ERR_BAD_ALIGN : go(token_logprobs_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits, allowed_bf16);
    return RB_ERR_BAD_DTYPE;
}
