// Log probabilities of given tokens, the rows' entropy and their most likely tokens, in one pass over the logits.
//
// With m the row's maximum, d = (x - m) log2 e, and n elements that are the maximum:   s = sum of 2^d over the others,   t = sum d 2^d,
//     log p(token) = (x - m) - log(n + s),   entropy = log(n + s) - t / ((n + s) log2 e).
// Each thread carries (m, n, s, t) of its own elements with m its running maximum; a warp raises its own to their maximum and adds them up.  Tokens are often nearly certain, and then
// both results hang on s alone, which a one beside it would swallow: hence n apart, and log1p(s) where n is one.  All sums are 32-bit, a chunk's terms
// added among themselves first (three hundred small terms, one by one, on top of a sum that already holds a large one would each be rounded at its size).
//
// The k most likely, largest first, equal ones by their index.  Beside its sums a thread keeps its largest element (and that
// element's chunk).  All of the k largest elements belong to the k threads whose largest elements lead: any other thread is
// behind k elements already.  So one pass over the row is enough; afterwards only those k threads' elements (k / threads of the
// row) are read again, all at once.  Keys are 64-bit whole numbers that order like (value, -index); places are found by counting the keys ahead.
//
// A row is read by one block or by the blocks of a cluster, which meet in the first one's shared memory.
//
// Memory bounds it where there are rows enough (2,047 rows of 151,936: 192 us, 6.5 TB/s); one row with 20 alternatives takes 7.8 us, 4.7 without.
// The ones counted apart cost 1 % of 32-bit rows; packed arithmetic and packed maxima give it back, and 5 % more, to bf16 ones, which the arithmetic bounds.
#include "common.cuh"
#include "api.h"
#include "per_device.h"
#include "sm100.cuh"

namespace {
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -3.402823466e38f;          // (a row may be all of the type's lowest value)
constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_TOP = 32, MAX_BLOCKS = 16;
constexpr int UNROLL = 4;          // chunks of 32 bytes that a thread has asked for at once
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

// Two 32-bit values in one instruction.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void unpair(Pair v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ Pair pair_add(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair pair_mul(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

struct __align__(16) Sum { float m, n, s, t; };
// The same sums relative to a maximum that is larger.
__device__ __forceinline__ void raise_maximum(Sum& a, float m) {
    const float by = max_nan((a.m - m) * LOG2E, -1000.f), f = rb::ex2(by), s = a.n + a.s;
    a = Sum{m, 0.f, f * s, f * fmaf(by, s, a.t)};
}
// A warp's sums joined, in every lane: its maximum first, so that each is raised once and the rest is adding up.
__device__ __forceinline__ Sum warp_sum(Sum v) {
    const unsigned int u = __float_as_uint(v.m + 0.f), top = __reduce_max_sync(0xffffffffu, (u & 0x80000000u) ? ~u : u | 0x80000000u);
    const float m = __uint_as_float((top & 0x80000000u) ? top & 0x7fffffffu : ~top);
    if (v.m < m) raise_maximum(v, m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.n += __shfl_xor_sync(0xffffffffu, v.n, o);
        v.s += __shfl_xor_sync(0xffffffffu, v.s, o);
        v.t += __shfl_xor_sync(0xffffffffu, v.t, o);
    }
    return v;
}

template <typename T> struct Chunk;                  // 32 bytes
// (sixteen values a chunk take more registers: three blocks a multiprocessor instead of four, or they spill)
template <> struct Chunk<float> { static constexpr int E = 8, BLOCKS_PER_SM = 4; };
template <> struct Chunk<__nv_bfloat16> { static constexpr int E = 16, BLOCKS_PER_SM = 3; };

// Eight words as they lie in memory -> E values.
template <typename T>
__device__ __forceinline__ void unpack_chunk(const uint4& a, const uint4& b, float* x) {
    const unsigned int w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (Chunk<T>::E == 8) x[i] = __uint_as_float(w[i]);
        else { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
}
template <int E>
__device__ __forceinline__ float largest(const float* x) {
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) mx = fmaxf(mx, x[e]);
    return mx;
}
// The largest of eight words' values, as they lie in memory.
template <typename T>
__device__ __forceinline__ float largest_packed(const uint4& a, const uint4& b) {
    if constexpr (Chunk<T>::E == 8) {
        float x[8];
        unpack_chunk<T>(a, b, x);
        return largest<8>(x);
    } else {
        auto two = [](unsigned int w) { return *reinterpret_cast<__nv_bfloat162*>(&w); };
        const __nv_bfloat162 m = __hmax2(__hmax2(__hmax2(two(a.x), two(a.y)), __hmax2(two(a.z), two(a.w))),
                                         __hmax2(__hmax2(two(b.x), two(b.y)), __hmax2(two(b.z), two(b.w))));
        return fmaxf(__low2float(m), __high2float(m));
    }
}
// The chunk whose first element is `i0` (which may lie before the row, or end after it: -inf there).
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int i0, int V, float* x) {
    constexpr int E = Chunk<T>::E;
    if (i0 >= 0 && i0 + E <= V) {
        const uint4* at = reinterpret_cast<const uint4*>(row + i0);
        unpack_chunk<T>(__ldg(at), __ldg(at + 1), x);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = i0 + e >= 0 && i0 + e < V ? rb::to_f32(row[i0 + e]) : -INFINITY;
    }
}

struct Shared {
    Key lists[MAX_BLOCKS][32];          // (as many as warps, or blocks of a cluster)
    Sum sums[MAX_BLOCKS];
    Key best[32];             // this block's k most likely, sorted
    Key leads[THREADS];       // largest elements of threads (by chunk), then candidates
    Sum sum;
    unsigned int least[WARPS];
    int n_leads, n_found;
};

// The 32 largest of the `lists` sorted lists (a power of two of them, at most 16; a warp brings its own in `v` where `mine`), sorted, in warp 0.  Every
// thread calls this.
__device__ __forceinline__ Key block_merge(Shared& sh, Key v, int lists = WARPS, bool mine = true) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (mine) {
        __syncthreads();
        sh.lists[warp][lane] = v;
    }
    for (int half = lists / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            v = warp_merge(sh.lists[warp][lane], sh.lists[warp + half][31 - lane]);
            sh.lists[warp][lane] = v;
        }
    }
    return v;
}

// `n` sums joined (at most 16), by warp 0.
__device__ __forceinline__ void sum_up(Shared& sh, int n) {
    const int lane = threadIdx.x & 31;
    const Sum v = warp_sum(lane < n ? sh.sums[lane] : Sum{LOWEST, 0.f, 0.f, 0.f});
    if (lane == 0) sh.sum = v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, Chunk<T>::BLOCKS_PER_SM)
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

    Sum mine{LOWEST, 0.f, 0.f, 0.f};
    float best = -INFINITY;
    int best_chunk = lo + (int)threadIdx.x < hi ? lo + (int)threadIdx.x : -1;
    auto add_chunk = [&](const float* x) {
        float s2[2] = {0.f, 0.f}, n2[2] = {0.f, 0.f}, t2[2];
        Pair t = 0ull;
        const Pair less_m = pair(-mine.m, -mine.m), log2e = pair(LOG2E, LOG2E);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float d[2], p[2];
            unpair(pair_mul(pair_add(pair(x[e], x[e + 1]), less_m), log2e), d[0], d[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                d[i] = max_nan(d[i], -1000.f);             // (-inf: 2^-1000 is 0, and so is 0 times -1000)
                p[i] = rb::ex2(d[i]);
                if (d[i] == 0.f) n2[i] += 1.f;
                else s2[i] += p[i];
            }
            t = pair_fma(pair(d[0], d[1]), pair(p[0], p[1]), t);
        }
        unpair(t, t2[0], t2[1]);
        mine.n += n2[0] + n2[1];
        mine.s += s2[0] + s2[1];
        mine.t += t2[0] + t2[1];
    };
    auto new_maximum = [&](float mx) {
        if (mx > mine.m) raise_maximum(mine, mx);
    };
    // whole chunks, UNROLL of them at a time; the row's first and last chunk, which it may share with its neighbours, one by one
    const int inner_lo = max(lo, before > 0 ? 1 : 0), inner_hi = min(hi, (int)(((long long)V + before) / E));
    int c = lo + threadIdx.x;
    if (c < hi && c < inner_lo) {
        float x[E];
        load_chunk(row, c * E - before, V, x);
        best = largest<E>(x);
        new_maximum(best);
        add_chunk(x);
        c += THREADS;
    }
    for (; c < inner_hi; c += UNROLL * THREADS) {
        uint4 raw[UNROLL][2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint4* at = reinterpret_cast<const uint4*>(row + ((long long)min(c + u * THREADS, inner_hi - 1) * E - before));
            raw[u][0] = __ldg(at);
            raw[u][1] = __ldg(at + 1);
        }
        float mx[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            mx[u] = largest_packed<T>(raw[u][0], raw[u][1]);
            if (c + u * THREADS < inner_hi && mx[u] > best) { best = mx[u]; best_chunk = c + u * THREADS; }
        }
        float all = mx[0];
#pragma unroll
        for (int u = 1; u < UNROLL; ++u) all = fmaxf(all, mx[u]);
        new_maximum(all);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float x[E];
            unpack_chunk<T>(raw[u][0], raw[u][1], x);
            if (c + u * THREADS < inner_hi) add_chunk(x);
        }
    }
    if (inner_hi < hi && hi - 1 >= inner_lo && (hi - 1 - lo) % THREADS == (int)threadIdx.x) {
        float x[E];
        load_chunk(row, (hi - 1) * E - before, V, x);
        const float mx = largest<E>(x);
        if (mx > best) { best = mx; best_chunk = hi - 1; }
        new_maximum(mx);
        add_chunk(x);
    }
    mine = warp_sum(mine);
    if (lane == 0) sh.sums[warp] = mine;
    __syncthreads();
    if (warp == 0) sum_up(sh, WARPS);
    if (top > 0) {
        // 1. A bound that at least `top` threads' largest elements reach: the least of the warps' j-th largest, j = top / WARPS rounded up.  The
        //    threads that reach it (some fifty for a top of 20) are put in a list.
        const unsigned int mine_top = best_chunk >= 0 ? (unsigned int)(key_of(best, best_chunk) >> 32) : 0u;
        unsigned int left = mine_top, jth = 0u;
        for (int j = 0; j < top; j += WARPS) {
            jth = __reduce_max_sync(0xffffffffu, left);
            if (lane == __ffs(__ballot_sync(0xffffffffu, left == jth)) - 1) left = 0u;
        }
        if (threadIdx.x == 0) sh.n_leads = sh.n_found = 0;
        if (lane == 0) sh.least[warp] = jth;
        if (threadIdx.x < 32) sh.best[threadIdx.x] = 0ull;
        __syncthreads();
        unsigned int bound = sh.least[0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) bound = min(bound, sh.least[w]);
        if (best_chunk >= 0 && mine_top >= bound) sh.leads[atomicAdd(&sh.n_leads, 1)] = key_of(best, best_chunk);
        __syncthreads();
        // 2. The `top` first of them, by how many are ahead of each (by value, then chunk: chunks of different threads differ).
        const int n_leads = sh.n_leads;
        if ((int)threadIdx.x < n_leads) {
            const Key k = sh.leads[threadIdx.x];
            int ahead = 0;
            for (int i = 0; i < n_leads; ++i) ahead += sh.leads[i] > k;
            if (ahead < top) sh.best[ahead] = k;
        }
        __syncthreads();
        // 3. Their elements again, a chunk a thread, all chunks of all of them at once; what reaches the last one's value is a candidate.
        const int n_top = min(top, n_leads), share = (hi - lo + THREADS - 1) / THREADS;
        const float least = n_top == top ? key_value(sh.best[top - 1]) : -INFINITY;
        for (int i0 = threadIdx.x; i0 < n_top * share; i0 += 2 * THREADS) {
            float x[2][E];
            int c2[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = i0 + u * THREADS;
                c2[u] = i < n_top * share ? lo + (key_index(sh.best[i / share]) - lo) % THREADS + i % share * THREADS : hi;
                if (c2[u] < hi) load_chunk(row, c2[u] * E - before, V, x[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (c2[u] >= hi) continue;
                const int first = c2[u] * E - before;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (x[u][e] >= least && first + e >= 0 && first + e < V) {
                        const int at = atomicAdd(&sh.n_found, 1);
                        if (at < THREADS) sh.leads[at] = key_of(x[u][e], first + e);
                    }
                }
            }
        }
        __syncthreads();
        const int n_found = sh.n_found;
        if (n_found <= THREADS) {
            // 4. The first `top` candidates, counted the same way.
            const Key k = (int)threadIdx.x < n_found ? sh.leads[threadIdx.x] : 0ull;
            int ahead = 0;
            for (int i = 0; i < n_found; ++i) ahead += sh.leads[i] > k;
            if (threadIdx.x < 32) sh.best[threadIdx.x] = 0ull;
            __syncthreads();
            if (k && ahead < 32) sh.best[ahead] = k;
        } else {
            // Too many equal values: the same elements sorted in by warps.  (What is not ahead of the top-th found so far is not sorted in: rows
            // of many equal values end quickly.)
            Key found = 0ull;
            for (int j = warp; j < n_top; j += WARPS) {
                const int c0 = lo + (key_index(sh.best[j]) - lo) % THREADS;
                for (int cb = c0; cb < hi; cb += 32 * THREADS) {
                    const int c1 = cb + lane * THREADS, first = c1 * E - before;
                    float x[E];
                    if (c1 < hi) load_chunk(row, first, V, x);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const bool may = c1 < hi && first + e >= 0 && first + e < V && x[e] >= least;
                        if (!__any_sync(0xffffffffu, may)) continue;
                        Key key = may ? key_of(x[e], first + e) : 0ull;
                        if (!__any_sync(0xffffffffu, key > __shfl_sync(0xffffffffu, found, top - 1))) continue;
                        key = warp_sort(key);
                        found = warp_merge(found, __shfl_sync(0xffffffffu, key, 31 - lane));
                    }
                }
            }
            found = block_merge(sh, found);
            if (warp == 0) sh.best[lane] = found;
        }
    }
    __syncthreads();
    if (blocks > 1) {
        // the first block of the cluster reads what the others found, a warp up to two of them
        sm100::cluster_arrive();
        sm100::cluster_wait();
        if (part == 0) {
            Sum v[2];
            Key k[2] = {0ull, 0ull};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int p = warp + i * WARPS;
                if (p >= blocks) continue;
                const uint32_t at = sm100::map_to_cta(sm100::smem_u32(&sh.sum), p);
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(v[i].m), "=f"(v[i].n), "=f"(v[i].s), "=f"(v[i].t) : "r"(at));
                if (top > 0)
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k[i]) : "r"(sm100::map_to_cta(sm100::smem_u32(&sh.best[lane]), p)));
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int p = warp + i * WARPS;
                if (p >= blocks) continue;
                if (lane == 0) sh.sums[p] = v[i];
                sh.lists[p][lane] = k[i];
            }
            Key all_best = 0ull;
            if (top > 0) all_best = block_merge(sh, 0ull, blocks, false);
            __syncthreads();
            if (warp == 0) {
                sum_up(sh, blocks);
                if (top > 0) sh.best[lane] = all_best;
            }
            __syncthreads();
        }
        sm100::cluster_arrive();
        sm100::cluster_wait();
        if (part != 0) return;
    }
    const Sum all = sh.sum;
    const float total = all.n + all.s, log_s = all.n == 1.f && all.s < 1.f ? log1pf(all.s) : logf(total);
    auto logprob = [&](float x) { return (float)(((double)x - (double)all.m) - (double)log_s); };
    const bool nothing = total == 0.f;                   // every logit -inf: nothing has a probability
    if (entropy && threadIdx.x == 0) entropy[r] = nothing ? 0.f : (float)((double)log_s - (double)all.t / ((double)total * (double)LOG2E));
    for (int j = threadIdx.x; j < m; j += THREADS) {
        const int id = ids[(size_t)r * m + j];
        logprobs[(size_t)r * m + j] = id < 0 || id >= V || nothing ? -INFINITY : logprob(rb::to_f32(row[id]));
    }
    if ((int)threadIdx.x < top) {
        const Key k = sh.best[threadIdx.x];
        if (top_ids) top_ids[(size_t)r * top + threadIdx.x] = k ? key_index(k) : -1;
        // (too few candidates: the row holds NaN, which is nobody's candidate and has spoiled the sums)
        if (top_logprobs) top_logprobs[(size_t)r * top + threadIdx.x] = nothing ? -INFINITY : k ? logprob(key_value(k)) : total;
    }
}
}  // namespace

// logits [n, V] (row stride ld elements); ids int32 [n, m]; logprobs float32 [n, m]; entropy float32 [n] or null; top_logprobs float32 and
// top_ids int32 [n, top], top <= 32.  blocks: 1, 2, 4, 8 or 16 blocks a row.
extern "C" int rb_token_logprobs(const RbLogprobsCall* call, void* stream) {
    const RbLogprobsCall& c = *call;
    if (c.n <= 0) return RB_OK;
    if (c.vocab <= 0 || c.vocab > (1 << 30) || c.m < 0 || c.top < 0 || c.top > MAX_TOP || c.top > c.vocab || (c.m > 0 && (!c.ids || !c.logprobs)) ||
        c.blocks < 1 || c.blocks > MAX_BLOCKS || (c.blocks & (c.blocks - 1)) || (long long)c.n * c.blocks > 0x7fffffffll)
        return RB_ERR_BAD_SIZE;
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto kernel, auto* x, rb::PerDevice<int>& allowed) -> int {
        if (c.blocks == 1) {
            RB_LAUNCH((kernel), dim3(c.n), dim3(THREADS), 0, st, x, c.ld, c.vocab, c.ids, c.m, c.logprobs, c.entropy, c.top_logprobs, c.top_ids, c.top,
                      c.blocks);
            return RB_OK;
        }
        int device;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return (int)e;
        const int* known;
        const int rc = allowed.get(device, &known, [&](int&) { return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
        if (rc) return rc;
        e = rb::launch_clustered(kernel, dim3(c.n * c.blocks), dim3(THREADS), dim3(c.blocks), 0, st, x, c.ld, c.vocab, c.ids, c.m, c.logprobs, c.entropy,
                                 c.top_logprobs, c.top_ids, c.top, c.blocks);
        return (int)e;
    };
    static rb::PerDevice<int> allowed_f32, allowed_bf16;
    if (c.dtype == RB_F32)
        return ((uintptr_t)c.logits & 3) ? RB_ERR_BAD_ALIGN : go(token_logprobs_kernel<float>, (const float*)c.logits, allowed_f32);
    if (c.dtype == RB_BF16)
        return ((uintptr_t)c.logits & 1) ? RB_ERR_BAD_ALIGN : go(token_logprobs_kernel<__nv_bfloat16>, (const __nv_bfloat16*)c.logits, allowed_bf16);
    return RB_ERR_BAD_DTYPE;
}
