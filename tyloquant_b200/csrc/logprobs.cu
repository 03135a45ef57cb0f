// Log probabilities of given tokens, with entropy, rank and the best alternatives: one pass over the logits.
#include <cuda_fp16.h>

#include "select.cuh"
#include "tc05.cuh"

namespace mfqb {

constexpr int kLpTop = 32, kLpGroups = 64, kLpList = 1024, kLpBatch = 4, kLpCtas = 8;
constexpr int kLpVocab = 1 << 20, kLpBrief = 8192, kLpSplit = 128 << 10, kLpSlice = 10000;

struct LogprobArgs {
    const char* logits;
    int64_t stride;   // bytes
    const int* tokens;
    int vocab, top;
    float *logprob, *entropy, *top_logprobs;
    int *rank, *top_tokens;
};

// Sums of some of a row's logits: exp(z - top), the same times z - top, and how many come before the given token.
struct LogprobSum {
    float top, sum, moment;
    int before;
};
template <int THREADS>
struct LogprobShared {
    union {   // the search for a cut is over when the list is made
        CutShared cut;
        unsigned long long list[kLpList];
    };
    LogprobSum warp[THREADS / 32], all;
    float group[kLpGroups], bound;
    int hot[THREADS], hots, count;
    unsigned long long best[kLpTop], gathered[kLpCtas][kLpTop];   // 0: none
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLpLowest = -3.402823466e38f, kLpNone = -150.f;   // exp(-150) is 0 in float32; its product with this too, where minus infinity's would be NaN

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float one_if_ge(float a, float b) {
    float r;
    asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ unsigned long long lp_key(float z, int token) { return (unsigned long long)ordered_f32(z) << 32 | (0xFFFFFFFFu - (unsigned)token); }

// 16 bytes of logits as float32.
template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void widen(const uint4& v, float* z) {
        z[0] = __uint_as_float(v.x); z[1] = __uint_as_float(v.y); z[2] = __uint_as_float(v.z); z[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ float lowest() { return -INFINITY; }
};
template <>
struct LpVec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ __nv_bfloat16 lowest() { return __ushort_as_bfloat16(0xFF80); }
    static __device__ __forceinline__ void widen(const uint4& v, float* z) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            z[2 * i] = __uint_as_float(w[i] << 16);
            z[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <>
struct LpVec<__half> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ __half lowest() { return __ushort_as_half(0xFC00); }
    static __device__ __forceinline__ void widen(const uint4& v, float* z) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            z[2 * i] = f.x;
            z[2 * i + 1] = f.y;
        }
    }
};
__device__ __forceinline__ float lp_float(float x) { return x; }
__device__ __forceinline__ float lp_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float lp_float(__half x) { return __half2float(x); }

__device__ __forceinline__ LogprobSum lp_join(LogprobSum a, LogprobSum b) {
    LogprobSum r;
    r.top = fmaxf(a.top, b.top);
    const float da = fmaxf(a.top - r.top, kLpNone), db = fmaxf(b.top - r.top, kLpNone);
    const float fa = exp2_approx(da * kLog2e), fb = exp2_approx(db * kLog2e);
    r.sum = a.sum * fa + b.sum * fb;
    r.moment = (a.moment + da * a.sum) * fa + (b.moment + db * b.sum) * fb;
    r.before = a.before + b.before;
    return r;
}

__device__ __forceinline__ LogprobSum lp_shuffle_join(LogprobSum a, int o) {
    LogprobSum b;
    b.top = __shfl_xor_sync(0xffffffffu, a.top, o);
    b.sum = __shfl_xor_sync(0xffffffffu, a.sum, o);
    b.moment = __shfl_xor_sync(0xffffffffu, a.moment, o);
    b.before = __shfl_xor_sync(0xffffffffu, a.before, o);
    return lp_join(a, b);
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();   // the aligned form wants the warp together, whatever its lanes did before
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared variable in another CTA of the cluster, and a load from there.
__device__ __forceinline__ uint32_t remote_smem(const void* p, unsigned rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t remote_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long remote_u64(uint32_t addr) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}

// A cluster per row, a slice of the row per CTA.  A thread takes every 256th vector of 16 bytes and keeps a running maximum with its sums.  The k
// best: a bound that at least k logits reach comes from the maxima of 64 groups of threads (the k-th largest of them), and only the
// vectors of threads whose own maximum reaches it are read again, a warp for each of those threads.  Where too many logits reach the
// bound (equal ones, or all in a few threads' vectors) the cut is searched by counting instead.
// Sums are float32, a thread's own of some hundred terms each, joined in a tree: a log sum is off by some 1e-7 (the sum is 1 and more, so a log probability
// below 6e-8 in size comes out as 0, and one of -1e-6 is off by a tenth of itself), an entropy likewise.  Many rows: bound by memory and by issue (1024 rows of 128256 in float32,
// five alternatives: 92 us, 5.7 TB/s, 12.6 instructions a logit; with checks of the ends of a row in the loop 19 instructions and 111 us).  One row: a chain of trips (7.5 us,
// with twenty alternatives 8.8: the logits, the hot threads' vectors again, the cluster's lists).
template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int kN = LpVec<T>::kN, kLpThreads = THREADS, kLpWarps = THREADS / 32;
    __shared__ LogprobShared<THREADS> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = cluster_rank(), ctas = cluster_size();
    const int64_t row = blockIdx.x / ctas;
    chained_wait();
    const T* z = reinterpret_cast<const T*>(a.logits + row * a.stride);
    // Vectors start at 16-byte boundaries; vector v holds logits v * kN - skew ..; those outside the row count as minus infinity.
    const int skew = (int)(((uintptr_t)z & 15) / sizeof(T)), vectors = (skew + a.vocab + kN - 1) / kN;
    const int first = (int)((int64_t)vectors * rank / ctas), last = (int)((int64_t)vectors * (rank + 1) / ctas);
    auto fetch = [&](int v) -> uint4 {
        const int at = v * kN - skew;
        if (at >= 0 && at + kN <= a.vocab) return __ldcg(reinterpret_cast<const uint4*>(z + at));
        alignas(16) T x[kN];
#pragma unroll
        for (int e = 0; e < kN; ++e) x[e] = at + e >= 0 && at + e < a.vocab ? z[at + e] : LpVec<T>::lowest();
        return *reinterpret_cast<const uint4*>(x);
    };
    auto load = [&](int v, float* x) { LpVec<T>::widen(fetch(v), x); };
    const int token = __ldcg(a.tokens + row);
    const bool there = (unsigned)token < (unsigned)a.vocab;
    // A logit comes before the token's own if it is larger, or equal with a lower number.
    const float zt = there ? lp_float(z[token]) + 0.f : INFINITY;
    const float above = unordered_f32(ordered_f32(zt) + 1u);
    // Of the CTA's vectors, those that lie wholly in the row are shared out over the threads; the row's ends go to two of them.
    const bool head = first == 0 && skew > 0 && first < last, tail = last == vectors && (skew + a.vocab) % kN && !(head && last == 1) && first < last;
    const int in0 = first + head, in1 = last - tail;
    float high_of = kLpLowest, most = -INFINITY;   // what the sums are of; the largest of all
    uint64_t sum = 0ull, moment = 0ull, before = 0ull;   // of the even and the odd ones of a vector
    const int token_at = there ? (token + skew) / kN : -1;   // the token's vector; its own equals before the token are added below
    auto take = [&](const auto& x, int v0, int step) {   // vectors v0, v0 + step ..
        constexpr int kVectors = sizeof(x) / sizeof(x[0]);
        float high = -INFINITY;
#pragma unroll
        for (int u = 0; u < kVectors; ++u)
#pragma unroll
            for (int e = 0; e < kN; ++e) high = fmaxf(high, x[u][e]);
        most = fmaxf(most, high);
        if (high > high_of) {
            const float d = fmaxf(high_of - high, kLpNone), f = exp2_approx(d * kLog2e);
            moment = fma_f32x2(fma_f32x2(pair_f32(d, d), sum, moment), pair_f32(f, f), 0ull);
            sum = fma_f32x2(sum, pair_f32(f, f), 0ull);
            high_of = high;
        }
        const uint64_t down = pair_f32(-high_of, -high_of), log2e = pair_f32(kLog2e, kLog2e);
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            const float line = v0 + u * step < token_at ? zt : above;
#pragma unroll
            for (int e = 0; e < kN; e += 2) {
                const float2 d = split_f32(add_f32x2(pair_f32(x[u][e], x[u][e + 1]), down));
                const uint64_t dd = pair_f32(max_nan(d.x, kLpNone), max_nan(d.y, kLpNone));
                const float2 y = split_f32(fma_f32x2(dd, log2e, 0ull));
                const uint64_t p = pair_f32(exp2_approx(y.x), exp2_approx(y.y));
                sum = add_f32x2(sum, p);
                moment = fma_f32x2(p, dd, moment);
                before = add_f32x2(before, pair_f32(one_if_ge(x[u][e], line), one_if_ge(x[u][e + 1], line)));   // at most vocab of them
            }
        }
    };
    {
        const uint4* at = reinterpret_cast<const uint4*>(z - skew) + in0 + tid;   // may point behind the row where there is nothing to read
        const int mine = in0 + tid < in1 ? (in1 - in0 - tid + kLpThreads - 1) / kLpThreads : 0, batches = mine / kLpBatch;
        uint4 next[kLpBatch];
        auto ask = [&](int from) {
#pragma unroll
            for (int u = 0; u < kLpBatch; ++u) next[u] = __ldcg(at + (from + u) * kLpThreads);
        };
        if (batches) ask(0);
        for (int i = 0; i < batches; ++i) {
            float x[kLpBatch][kN];
#pragma unroll
            for (int u = 0; u < kLpBatch; ++u) LpVec<T>::widen(next[u], x[u]);
            if (i + 1 < batches) ask((i + 1) * kLpBatch);   // on its way while this one is worked on
            take(x, in0 + tid + i * kLpBatch * kLpThreads, kLpThreads);
        }
        const int left = mine - batches * kLpBatch;
#pragma unroll
        for (int u = 0; u < kLpBatch - 1; ++u)
            if (u < left) next[u] = __ldcg(at + (batches * kLpBatch + u) * kLpThreads);
#pragma unroll
        for (int u = 0; u < kLpBatch - 1; ++u)
            if (u < left) {
                float x[1][kN];
                LpVec<T>::widen(next[u], x[0]);
                take(x, in0 + tid + (batches * kLpBatch + u) * kLpThreads, kLpThreads);
            }
        const int end = tid == 0 && head ? 0 : tid == 1 && tail ? vectors - 1 : -1;
        if (end >= 0) {
            float x[1][kN];
            load(end, x[0]);
            take(x, end, 0);
        }
    }
    LogprobSum s;
    {
        const float2 x = split_f32(sum), y = split_f32(moment), n = split_f32(before);
        s = LogprobSum{high_of, x.x + x.y, y.x + y.y, (int)n.x + (int)n.y};
    }
    if (zt == -INFINITY && tid == 0 && head && token_at > 0) s.before -= skew;   // minus infinities that are not the row's
    if (tid == 0 && token_at >= first && token_at < last)
        for (int i = max(0, token_at * kN - skew); i < token; ++i) s.before += lp_float(z[i]) == zt;
    // ---- the CTA's sums
    LogprobSum joint = s;
    for (int o = 16; o > 0; o >>= 1) joint = lp_shuffle_join(joint, o);
    if (lane == 0) sh.warp[warp] = joint;
    if (a.top > 0) {
        float group = most;   // of neighbouring threads
        for (int o = kLpThreads / kLpGroups / 2; o > 0; o >>= 1) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, o));
        if (tid % (kLpThreads / kLpGroups) == 0) sh.group[tid / (kLpThreads / kLpGroups)] = group;
        if (tid == 0) sh.hots = sh.count = 0;
    }
    __syncthreads();
    if (warp == 0) {
        LogprobSum x = sh.warp[lane & (kLpWarps - 1)];
        for (int o = kLpWarps / 2; o > 0; o >>= 1) x = lp_shuffle_join(x, o);
        if (lane == 0) sh.all = x;
    }
    if (a.top > 0) {
        // ---- the bound: the group maxima in order, equal ones by group
        if (tid < kLpGroups) {
            const float g = sh.group[tid];
            int larger = 0;
            for (int j = 0; j < kLpGroups; ++j) larger += sh.group[j] > g || (sh.group[j] == g && j < tid);
            if (larger == a.top - 1) sh.bound = g;
        }
        __syncthreads();
        const float bound = sh.bound;
        if (most >= bound && (in0 + tid < in1 || (tid == 0 && head) || (tid == 1 && tail))) sh.hot[atomicAdd(&sh.hots, 1)] = tid;
        __syncthreads();
        const int hots = sh.hots;
        for (int h = warp; h < hots; h += kLpWarps) {
            const int thread = sh.hot[h], end = thread == 0 && head ? 0 : thread == 1 && tail ? vectors - 1 : -1;
            const int count = (in0 + thread < in1 ? (in1 - in0 - thread + kLpThreads - 1) / kLpThreads : 0) + (end >= 0);
            for (int i = lane; i < count; i += 32) {
                const int v = end >= 0 && i == count - 1 ? end : in0 + thread + i * kLpThreads;
                float x[kN];
                load(v, x);
                const int at = v * kN - skew;
#pragma unroll
                for (int e = 0; e < kN; ++e)
                    if (x[e] >= bound && at + e >= 0 && at + e < a.vocab) {
                        const int i = atomicAdd(&sh.count, 1);
                        if (i < kLpList) sh.list[i] = lp_key(x[e], at + e);
                    }
            }
        }
        __syncthreads();
        int n = sh.count;
        if (n > kLpList) {
            auto each = [&](auto f) {
                for (int v = first + tid; v < last; v += kLpThreads) {
                    float x[kN];
                    load(v, x);
                    const int at = v * kN - skew;
#pragma unroll
                    for (int e = 0; e < kN; ++e)
                        if (at + e >= 0 && at + e < a.vocab) f(ordered_f32(x[e]), at + e);
                }
            };
            unsigned low = 0xFFFFFFFFu, high = 0u;
            each([&](unsigned k, int) {
                low = min(low, k);
                high = max(high, k);
            });
            const Cut cut = select_cut<kLpThreads>(a.top, low, high, 0xFFFFFFFFu, a.vocab, sh.cut, each);
            __syncthreads();
            if (tid == 0) sh.count = 0;
            __syncthreads();
            each([&](unsigned k, int token) {
                if (!cut.in(k, token)) return;
                const int i = atomicAdd(&sh.count, 1);   // a.top of them; the bounds are for logits that change meanwhile
                if (i < kLpList) sh.list[i] = (unsigned long long)k << 32 | (0xFFFFFFFFu - (unsigned)token);
            });
            __syncthreads();
            n = min(sh.count, kLpList);
        }
        // ---- the list in order: every key counts those above it
        const int keep = min(n, a.top);
        for (int i = tid; i < n; i += kLpThreads) {
            const unsigned long long key = sh.list[i];
            int larger = 0;
            for (int j = 0; j < n; ++j) larger += sh.list[j] > key;
            if (larger < keep) sh.best[larger] = key;
        }
        if (tid >= keep && tid < kLpTop) sh.best[tid] = 0ull;
    }
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    if (rank == 0) {
        LogprobSum x = sh.all;
        const unsigned long long* best = sh.best;
        if (ctas > 1) {   // lane c has CTA c's sums, every warp the same; all lists are brought here at once
            const uint32_t at = remote_smem(&sh.all, lane % ctas);
            x = LogprobSum{__uint_as_float(remote_u32(at)), __uint_as_float(remote_u32(at + 4)), __uint_as_float(remote_u32(at + 8)), (int)remote_u32(at + 12)};
            if (a.top > 0) {
                for (int i = tid; i < (int)ctas * kLpTop; i += kLpThreads) sh.gathered[i / kLpTop][i % kLpTop] = remote_u64(remote_smem(&sh.best[i % kLpTop], i / kLpTop));
                if (tid == 0) sh.count = 0;
            }
            for (int o = ctas / 2; o > 0; o >>= 1) x = lp_shuffle_join(x, o);
            if (a.top > 0) {
                __syncthreads();
                // In order, the lists have at least `top` keys up to here; what lies below the smallest of these is not among the best.
                unsigned long long line = sh.gathered[lane % ctas][(a.top + ctas - 1) / ctas - 1];
                for (int o = ctas / 2; o > 0; o >>= 1) line = min(line, __shfl_xor_sync(0xffffffffu, line, o));
                for (int i = tid; i < (int)ctas * kLpTop; i += kLpThreads) {
                    const unsigned long long key = sh.gathered[i / kLpTop][i % kLpTop];
                    if (key && key >= line) sh.list[atomicAdd(&sh.count, 1)] = key;   // at most eight lists of 32
                }
                __syncthreads();
                const int n = sh.count;
                for (int i = tid; i < n; i += kLpThreads) {
                    const unsigned long long key = sh.list[i];
                    int larger = 0;
                    for (int j = 0; j < n; ++j) larger += sh.list[j] > key;
                    if (larger < a.top) sh.best[larger] = key;
                }
                __syncthreads();
            }
        }
        // a NaN, plus infinity, or nothing above minus infinity leaves no log sum
        const bool good = x.sum > 0.f && x.sum < INFINITY && x.top < INFINITY;
        const float log_sum = logf(x.sum);
        if (tid == 0) {
            a.logprob[row] = !there ? 0.f : good ? (zt - x.top) - log_sum : NAN;
            a.entropy[row] = good ? log_sum - x.moment / x.sum : NAN;
            a.rank[row] = good && there ? x.before + 1 : 0;
        }
        if (tid < a.top) {
            const unsigned long long key = best[tid];
            a.top_logprobs[row * a.top + tid] = good ? (unordered_f32((unsigned)(key >> 32)) - x.top) - log_sum : NAN;
            a.top_tokens[row * a.top + tid] = good ? (int)(0xFFFFFFFFu - (unsigned)key) : -1;
        }
    }
    if (ctas > 1) cluster_sync();   // no CTA leaves while its lists are read
}

template <typename T>
static void launch_logprobs(const LogprobArgs& a, int rows, cudaStream_t s) {
    // CTAs of a row.  Joining them costs some 1 to 2 us, which rows of up to 128 KB do not earn: 30, 230 rows of 32768 in float32 6.4, 11.8 us with one and 6.9, 12.3 with two, of
    // 40000 7.9, 14.3 and 7.5, 13.1; of 50257 in bfloat16 8.0, 13.8 and 8.0, 14.2, of 80000 10.3, 19.0 and 9.0, 17.9 (one row gains from 80 KB on: 64000 in bfloat16 8.0
    // and 7.5).  Above that two, four: as long as all are on the SMs at once (300 rows of 128256: 35.5 with one, 43 with two).  Eight where a slice keeps 10000 logits and
    // an SM has two of them at most: 30 rows of 64000 7.8 with four, 8.9 with eight, of 100000 10.5 and 9.7, of 262144 17.7 and 14.0; 70 rows of 128256 14.5 and 16.2;
    // one row of 128256 14.4, 10.5, 8.5 and 7.5 with one, two, four, eight (five alternatives; twenty: 18.2, 12.6, 9.8, 8.8).
    int ctas = 1;
    const int64_t bytes = (int64_t)a.vocab * sizeof(T);
    if (bytes > kLpSplit)
        while (ctas < kLpCtas && (int64_t)rows * ctas * 2 <= (ctas < 4 ? 4 : 2) * 148 && (ctas < 4 || a.vocab / kLpCtas >= kLpSlice)) ctas *= 2;
    // Four CTAs on an SM read more at a time (1024 rows of 128256 in float32 92 us, 108 with three; in bfloat16 60 with either), three have more registers (300 rows 35.3 us, 37.6 with
    // four; in bfloat16 27.7 and 34.4).
    const bool four = (int64_t)rows * ctas > 3 * 148;
    // Many short rows are a chain each, of which more run at once in CTAs of 128 threads, eight on an SM: 4000 rows of 1000 in float32
    // 22 us, 33.6 in CTAs of 256; 2000 of 8000 21.6 and 27.7; 1500 of 32001 47 and 43 (600 of 16000 13.7 and 14.9, in bfloat16 14.6 and 14.0).
    const bool brief = four && ctas == 1 && a.vocab <= kLpBrief;
    const int threads = brief ? 128 : 256;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * ctas);
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    MFQB_CUDA(cudaLaunchKernelEx(&cfg, brief ? logprobs_kernel<T, 128, 8> : four ? logprobs_kernel<T, 256, 4> : logprobs_kernel<T, 256, 3>, a));
}

}  // namespace mfqb

using namespace mfqb;

extern "C" {
#pragma GCC visibility push(default)

int mfqb_token_logprobs(const void* logits, int dtype, int rows, int vocab, int64_t row_stride, const int32_t* tokens, int top, float* logprob, float* entropy,
                        int32_t* rank, float* top_logprobs, int32_t* top_tokens, mfqb_stream_t stream) {
    return guarded([&] {
        if (!logits || !tokens || !logprob || !entropy || !rank) fail(MFQB_ERR_ARG, "mfqb_token_logprobs: null argument");
        if (dtype != MFQB_F32 && dtype != MFQB_BF16 && dtype != MFQB_F16) fail(MFQB_ERR_ARG, "mfqb_token_logprobs: bad type of logits %d", dtype);
        const int size = dtype == MFQB_F32 ? 4 : 2;
        if ((uintptr_t)logits & (size - 1)) fail(MFQB_ERR_ARG, "mfqb_token_logprobs: logits must be aligned to their type");
        if (rows < 1 || rows > (1 << 24)) fail(MFQB_ERR_ARG, "mfqb_token_logprobs: 1 to %d rows, got %d", 1 << 24, rows);
        if (vocab < 1 || vocab > kLpVocab) fail(MFQB_ERR_UNSUPPORTED, "mfqb_token_logprobs: a vocabulary of 1 to %d tokens, got %d", kLpVocab, vocab);
        if (row_stride < vocab && rows > 1) fail(MFQB_ERR_ARG, "mfqb_token_logprobs: rows of %d logits every %lld", vocab, (long long)row_stride);
        if (top < 0 || top > kLpTop || top > vocab) fail(MFQB_ERR_UNSUPPORTED, "mfqb_token_logprobs: 0 to min(%d, vocab) alternatives, got %d", kLpTop, top);
        if (top && (!top_logprobs || !top_tokens)) fail(MFQB_ERR_ARG, "mfqb_token_logprobs: null argument");
        LogprobArgs a{static_cast<const char*>(logits), row_stride * size, tokens, vocab, top, logprob, entropy, top_logprobs, rank, top_tokens};
        if (dtype == MFQB_F32) launch_logprobs<float>(a, rows, stream);
        else if (dtype == MFQB_BF16) launch_logprobs<__nv_bfloat16>(a, rows, stream);
        else launch_logprobs<__half>(a, rows, stream);
    });
}

#pragma GCC visibility pop
}  // extern "C"
