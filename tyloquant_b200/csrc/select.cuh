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

// What is in: keys above `key`, and of those that equal it the ones at places up to `last`.
struct Cut {
    unsigned key;
    int last;
    __device__ __forceinline__ bool in(unsigned k, int place) const { return k > key || (k == key && place <= last); }
};
constexpr int kCutBins = 2048, kCutFew = 64;
constexpr unsigned kCutZero = 0x80000000u;   // ordered_f32(0)
struct CutShared {
    alignas(16) int bins[kCutBins];
    alignas(16) unsigned long long few[kCutFew];
    int sums[33], at, left, inside;
    unsigned low[32], high[32], above[32];
    Cut cut;
};

// The cut that lets `want` of the keys in, equal ones by place (1 <= want <= how many there are).  each(f) calls f(key, place) for this
// thread's share of the keys, the same ones every time, at places 0 .. places - 1; a key 0 is none.  low and high are the smallest and the
// largest of the thread's (all ones and 0 where there are none).  Bins divide the range from the smallest to the largest key: float32 values
// that span orders of magnitude lie in many of them (by the first bits of the keys they would meet in a few counters, whose additions
// wait for one another), and three rounds of 11 bits are enough for any range, a fourth where the first one splits at zero.  Weights are mostly positive with some zeros, far below the
// others in this order: the first round's first bin has all that is not above zero, the others divide the rest.  A round ends the search when all of its last bin is in, or
// when that holds so few keys that they are better counted against each other.  The next one goes by what the keys of the bin span; where
// they are equal, by their places.
template <int THREADS, class Each>
__device__ Cut select_cut(int want, unsigned low, unsigned high, unsigned above, int places, CutShared& sh, Each each) {
    static_assert(kCutBins % (4 * THREADS) == 0 && 2 * kCutFew <= THREADS, "bins of a thread");
    constexpr int kOwn = kCutBins / THREADS, kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31;
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    above = __reduce_min_sync(0xffffffffu, above);
    if (lane == 0) {
        sh.low[threadIdx.x >> 5] = low;
        sh.high[threadIdx.x >> 5] = high;
        sh.above[threadIdx.x >> 5] = above;
    }
    __syncthreads();
    unsigned base = __reduce_min_sync(0xffffffffu, sh.low[lane % kWarps]);
    above = __reduce_min_sync(0xffffffffu, sh.above[lane % kWarps]);   // the smallest one above zero
    unsigned range = __reduce_max_sync(0xffffffffu, sh.high[lane % kWarps]) - base;   // keys base .. base + range
    bool split = base <= kCutZero && above != 0xFFFFFFFFu;   // the first round
    unsigned tied = 0;   // the key whose places are being sorted out, the first one the largest
    // At most four rounds by key (three, and one that splits at zero) and three by place.  The count is also what ends the search when keys change while it is under way.
    for (int round = 0; round < 7; ++round) {
        // range >> shift is below 2048, or, of what is above zero, below 2047
        const int shift = split ? max(0, 21 - __clz((base + range - above) | 1u)) + ((base + range - above) >> max(0, 21 - __clz((base + range - above) | 1u)) == 2047u)
                                : max(0, 21 - __clz(range | 1u));
        int4* own_bins = reinterpret_cast<int4*>(sh.bins + kCutBins - kOwn * ((int)threadIdx.x + 1));   // from the last one down
#pragma unroll
        for (int j = 0; j < kOwn / 4; ++j) own_bins[j] = make_int4(0, 0, 0, 0);
        __syncthreads();
        if (split) {
            each([&](unsigned k, int) {
                if (k) atomicAdd(&sh.bins[k >= above ? min((k - above) >> shift, 2046u) + 1 : 0u], 1);
            });
        } else if (!tied) {
            each([&](unsigned k, int) {
                if (k - base <= range) atomicAdd(&sh.bins[(k - base) >> shift], 1);
            });
        } else {
            each([&](unsigned k, int place) {
                const unsigned x = ~(unsigned)place - base;
                if (k == tied && x <= range) atomicAdd(&sh.bins[x >> shift], 1);
            });
        }
        __syncthreads();
        int own[kOwn], mine = 0;
#pragma unroll
        for (int j = 0; j < kOwn / 4; ++j) {
            const int4 x = own_bins[j];
            own[kOwn - 4 * j - 1] = x.x; own[kOwn - 4 * j - 2] = x.y; own[kOwn - 4 * j - 3] = x.z; own[kOwn - 4 * j - 4] = x.w;
            mine += x.x + x.y + x.z + x.w;
        }
        const int upto = block_scan<THREADS>(mine, sh.sums);
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
        if (split && sh.at == 0) {
            range = kCutZero - base;
        } else {
            base = split ? above + ((unsigned)(sh.at - 1) << shift) : base + ((unsigned)sh.at << shift);
            range = (1u << shift) - 1u;
        }
        split = false;
        if (want == inside) return tied ? Cut{tied, (int)~base} : Cut{base - 1u, -1};   // no key of a value is 0
        if (inside <= kCutFew) {
            __syncthreads();
            if (threadIdx.x == 0) sh.at = 0;
            __syncthreads();
            each([&](unsigned k, int place) {
                if (tied ? k == tied && ~(unsigned)place - base <= range : k - base <= range) {
                    const int i = atomicAdd(&sh.at, 1);
                    if (i < kCutFew) sh.few[i] = (unsigned long long)k << 32 | ~(unsigned)place;
                }
            });
            __syncthreads();
            // Two or four threads count for a key.
            const int each_key = inside <= THREADS / 4 ? 4 : 2, at = threadIdx.x / each_key, from = threadIdx.x % each_key;
            int larger = 0;
            const unsigned long long x = sh.few[min(at, kCutFew - 1)];
            if (at < inside)
                for (int i = from; i < inside; i += each_key) larger += sh.few[i] > x;
            larger += __shfl_xor_sync(0xffffffffu, larger, 1);
            if (each_key == 4) larger += __shfl_xor_sync(0xffffffffu, larger, 2);
            if (at < inside && larger == want - 1) sh.cut = Cut{(unsigned)(x >> 32), (int)~(unsigned)x};
            __syncthreads();
            return sh.cut;
        }
        if (!tied) {   // what the bin's keys really span: equal ones are found so at once
            low = 0xFFFFFFFFu;
            high = 0u;
            each([&](unsigned k, int) {
                if (k - base <= range) {
                    low = min(low, k);
                    high = max(high, k);
                }
            });
            low = __reduce_min_sync(0xffffffffu, low);
            high = __reduce_max_sync(0xffffffffu, high);
            if (lane == 0) {
                sh.low[threadIdx.x >> 5] = low;
                sh.high[threadIdx.x >> 5] = high;
            }
            __syncthreads();
            base = __reduce_min_sync(0xffffffffu, sh.low[lane % kWarps]);
            range = __reduce_max_sync(0xffffffffu, sh.high[lane % kWarps]) - base;
            if (range == 0) {
                tied = base;
                base = ~(unsigned)(places - 1);
                range = (unsigned)(places - 1);
            }
        }
        __syncthreads();
    }
    return Cut{0xFFFFFFFFu, -1};
}

}  // namespace mfqb
