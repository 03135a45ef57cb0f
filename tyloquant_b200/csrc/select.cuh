// Selection of the largest of many float32 values inside a CTA, with ties by order: what the eviction and the log probabilities share.
#pragma once
#include "paged.h"

namespace mfqb {

// Values in the order of unsigned numbers: -0 as 0, a NaN as minus infinity.
__device__ __forceinline__ unsigned ordered_f32(float x) {
    const unsigned b = __float_as_uint(x == x ? x + 0.f : -INFINITY);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered_f32(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }

// Sum over the threads up to and with this one; every thread calls it.  sums: THREADS / 32 + 1 ints of shared memory, the last one becomes the total.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* sums) {
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();   // the sums of an earlier call have been read
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    int before = lane < kWarps ? sums[lane] : 0;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    if (threadIdx.x == 31) sums[kWarps] = before;
    return v + (warp ? __shfl_sync(0xffffffffu, before, warp - 1) : 0);
}

// What is in: keys above `key`, and the first `ties` of those that equal it.
struct Cut {
    unsigned key;
    int ties;
};
constexpr int kCutBins = 2048;
struct CutShared {
    int bins[kCutBins], sums[33], at, left, inside;
    unsigned low, high;
};

// The cut that lets `want` of the keys in (1 <= want <= how many there are).  each(f) calls f(key) for this thread's share of the keys, the same
// ones every time.  Bins divide the range from the smallest to the largest key: float32 values that span orders of magnitude lie in
// many of them (by the first bits of the keys they would meet in a few counters, whose additions wait for one another), and three rounds
// of 11 bits are enough for any range; a round ends the search when all of its last bin is in.
template <int THREADS, class Each>
__device__ Cut select_cut(int want, CutShared& sh, Each each) {
    static_assert(kCutBins % THREADS == 0, "bins of a thread");
    constexpr int kOwn = kCutBins / THREADS;
    unsigned low = 0xFFFFFFFFu, high = 0u;
    each([&](unsigned k) {
        low = min(low, k);
        high = max(high, k);
    });
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.low = 0xFFFFFFFFu;
        sh.high = 0u;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        atomicMin(&sh.low, low);
        atomicMax(&sh.high, high);
    }
    __syncthreads();
    unsigned base = sh.low, range = sh.high - sh.low;   // keys base .. base + range
    for (;;) {
        const int shift = max(0, 21 - __clz(range | 1u));   // range >> shift is below 2048
        for (int b = threadIdx.x; b < kCutBins; b += THREADS) sh.bins[b] = 0;
        __syncthreads();
        each([&](unsigned k) {
            if (k - base <= range) atomicAdd(&sh.bins[(k - base) >> shift], 1);
        });
        __syncthreads();
        int own[kOwn], mine = 0;   // this thread's bins, from the last one down
#pragma unroll
        for (int j = 0; j < kOwn; ++j) mine += own[j] = sh.bins[kCutBins - 1 - ((int)threadIdx.x * kOwn + j)];
        int upto = block_scan<THREADS>(mine, sh.sums);
        if (upto >= want && upto - mine < want) {
            int before = upto - mine;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                if (before < want && before + own[j] >= want) {
                    sh.at = kCutBins - 1 - ((int)threadIdx.x * kOwn + j);
                    sh.left = want - before;
                    sh.inside = own[j];
                }
                before += own[j];
            }
        }
        __syncthreads();
        want = sh.left;
        const int inside = sh.inside;
        base += (unsigned)sh.at << shift;
        __syncthreads();
        if (want == inside) return Cut{base - 1u, 0};   // no key of a value is 0
        if (shift == 0) return Cut{base, want};
        range = (1u << shift) - 1u;
    }
}

}  // namespace mfqb
