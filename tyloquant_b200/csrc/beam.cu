// Beam selection: the k best continuations of a group of beams by score + log softmax(logits), one pass over the logits.
#include <mutex>

#include "paged.h"

namespace mfqb {

constexpr int kBeamMax = 128, kBeamKeep = 128, kBeamProduct = 8192;   // beams of a group, candidates kept, one times the other
constexpr int kSliceThreads = 256, kSliceEach = 32, kSlice = kSliceThreads * kSliceEach;
constexpr size_t kMergeSmem = 200 * 1024;        // of the merging kernel
constexpr int kSlicesMax = 128;                  // slices of a row: lists that the 32 lanes of a warp merge, four each

// A slice's record: its largest logit, the sum of exp(logit - largest) and its k best keys, best first.
struct SliceSum {
    double sum;
    float top;
    float pad;
};

// Larger key = better candidate of a beam: logit (a NaN as minus infinity, -0 as 0), then the lower token.
__device__ __forceinline__ unsigned long long beam_key(float x, unsigned token) {
    const float y = x == x ? x + 0.f : -INFINITY;
    const unsigned b = __float_as_uint(y);
    const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

// Float32 values in the order of unsigned numbers, for values that are no NaN.
__device__ __forceinline__ unsigned order_f32(float v) {
    const unsigned b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_f32(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }

constexpr int kListMax = 1024;   // candidates of a slice that are ranked by counting
constexpr int kThreadMost = 8;   // of a thread's 32

// CTA (slice, row).  A thread keeps its 32 logits in registers: element (j * 256 + thread) * 4 + e of the slice whatever the row's
// alignment, so that equal rows have equal sums to the last bit and ties between beams are ties.
//
// Candidates are the elements that reach a bound which at least k of them do: the j-th largest thread maximum of a warp, j = ceil(k / c), in the
// c-th best of the eight warps, for the better of c = 8 and 4 (some 35 candidates for k = 16; with c = 8 alone some 100).  They go into a list,
// and a candidate's place is the number of larger ones in it.  The j-th largest is found by j rounds of a warp's maximum up to k = 32, by a
// sort beyond (a sort for k = 16 was a quarter of a CTA's time); the k-th largest of all 256 maxima, found by counting, took as long as
// everything else.  Where too many elements reach the bound for the list (most of
// the slice is masked) a second list leaves out equal ones that cannot be among the best, or, where that does not help, the k-th largest is found by
// bisection, bit by bit of its value, then of its place.
//
// 16 groups of 8 beams, 128256 tokens, k = 16: 17 us of 24 (73 in all with counting); all but 100 tokens masked: 64 in all (k = 64: 87), and 200 (627) where
// a short list meant k rounds of the largest.
__global__ void __launch_bounds__(kSliceThreads, 4) beam_slice_kernel(const float* logits, const int* done, int vocab, int k, int slices, bool wide, SliceSum* sums,
                                                                      unsigned long long* keys) {
    chained_wait();
    __shared__ unsigned long long s_list[kListMax];
    __shared__ float s_top[8], s_low[16];
    __shared__ double s_sum[8];
    __shared__ int s_count, s_part[2][8];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, slice = blockIdx.x;
    const int64_t row = blockIdx.y;
    if (done && __ldcg(done + row)) return;
    const int base = slice * kSlice;
    const float* src = logits + row * vocab + base;
    const int n = min(kSlice, vocab - base);
    float x[kSliceEach];   // minus infinity behind the end
    if (wide && n == kSlice) {
#pragma unroll
        for (int j = 0; j < kSliceEach / 4; ++j) {
            const float4 v = __ldcs(reinterpret_cast<const float4*>(src) + j * kSliceThreads + t);
            x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kSliceEach; ++j) {
            const int i = ((j >> 2) * kSliceThreads + t) * 4 + (j & 3);
            x[j] = i < n ? __ldcs(src + i) : -INFINITY;
        }
    }
    if (t == 0) s_count = 0;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSliceEach; j += 2) top = fmaxf(fmaxf(top, x[j]), x[j + 1]);
    // the warp's largest thread maximum, its ceil(k / 8)-th and its ceil(k / 4)-th
    const int j8 = (k + 7) / 8, j4 = (k + 3) / 4;
    float high, low8, low4;
    if (j4 <= 8) {
        unsigned mine = order_f32(top), best = 0u, first = 0u, eighth = 0u;
        for (int j = 1; j <= j4; ++j) {   // lanes that are equal leave together: the value found is at most the j-th
            best = __reduce_max_sync(0xffffffffu, mine);
            if (j == 1) first = best;
            if (j == j8) eighth = best;
            if (mine == best) mine = 0u;
        }
        high = from_order_f32(first);
        low8 = eighth ? from_order_f32(eighth) : -INFINITY;   // 0: no lane was left
        low4 = best ? from_order_f32(best) : -INFINITY;
    } else {
        float v = top;   // in descending order
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
            for (int o = size >> 1; o > 0; o >>= 1) {
                const float u = __shfl_xor_sync(0xffffffffu, v, o);
                v = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(v, u) : fminf(v, u);
            }
        high = __shfl_sync(0xffffffffu, v, 0);
        low8 = __shfl_sync(0xffffffffu, v, j8 - 1);
        low4 = __shfl_sync(0xffffffffu, v, j4 - 1);
    }
    if (lane == 0) {
        s_top[warp] = high;
        s_low[warp] = low8;
        s_low[8 + warp] = low4;
    }
    __syncthreads();
    float bound;
    {   // the least of the warps' first value, the fourth of their second
        const float mine = s_low[8 + (lane & 7)];
        float least = s_low[0];
        int above = 0;
        top = s_top[0];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float v = s_low[8 + w];
            top = fmaxf(top, s_top[w]);
            least = fminf(least, s_low[w]);
            above += v > mine || (v == mine && w < (lane & 7));
        }
        bound = fmaxf(least, __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, above == 3)) - 1));
    }
    unsigned take = 0;
    float part = 0.f;
    if (top > -INFINITY && top < INFINITY && (bound > -INFINITY || n == kSlice)) {
        // exp(x - top), the exponent in two terms (log2(e) in one float32 is off by 2^-26); NaN where there is a NaN
        uint64_t sum = 0ull;
        const uint64_t minus_top = pair_f32(-top, -top), hi = pair_f32(1.44269502f, 1.44269502f), lo = pair_f32(1.9259629e-8f, 1.9259629e-8f);
#pragma unroll
        for (int j = 0; j < kSliceEach; j += 2) {
            const uint64_t d = add_f32x2(pair_f32(x[j], x[j + 1]), minus_top);
            const float2 e = split_f32(fma_f32x2(d, lo, fma_f32x2(d, hi, 0ull)));
            sum = add_f32x2(sum, pair_f32(exp2_approx(e.x), exp2_approx(e.y)));
            take |= (unsigned)(x[j] >= bound) << j | (unsigned)(x[j + 1] >= bound) << (j + 1);
        }
        const float2 both = split_f32(sum);
        part = both.x + both.y;
        if (bound == -INFINITY) take = 0xFFFFFFFFu;   // a NaN too, as minus infinity
    } else {   // the same for what is out of the ordinary; a NaN counts as minus infinity among the candidates
#pragma unroll
        for (int j = 0; j < kSliceEach; ++j) {
            const int i = ((j >> 2) * kSliceThreads + t) * 4 + (j & 3);
            if (i >= n) continue;
            const float d = x[j] - top;
            if (x[j] != -INFINITY) part += exp2f(fmaf(d, 1.9259629e-8f, d * 1.44269502f));   // infinity - infinity: NaN
            if (x[j] >= bound || bound == -INFINITY) take |= 1u << j;
        }
    }
    double sum = part;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    if (take) {
        // The order in the list does not matter.  Many of one thread's mean a slice with many equal ones: no list of these.
        int at = atomicAdd(&s_count, __popc(take) > kThreadMost ? kListMax + 1 : __popc(take));
        if (__popc(take) > kThreadMost) at = kListMax;
#pragma unroll 1
        for (unsigned left = take; left && at < kListMax; left &= left - 1, ++at) {   // read again: few, and a loop over registers would have to be unrolled
            const int j = __ffs(left) - 1, i = ((j >> 2) * kSliceThreads + t) * 4 + (j & 3);
            s_list[at] = beam_key(__ldcg(src + i), (unsigned)(base + i));
        }
    }
    __syncthreads();
    if (t == 0) {
        sum = s_sum[0];
        for (int w = 1; w < 8; ++w) sum += s_sum[w];
        sums[row * slices + slice] = SliceSum{sum, top, 0.f};
    }
    int have = s_count;
    if (have > kListMax) {
        auto place_of = [&](int j) { return ((j >> 2) * kSliceThreads + t) * 4 + (j & 3); };
        int counts = 0;
        auto count_all = [&](int c) {   // over the CTA
            c = __reduce_add_sync(0xffffffffu, c);
            int* part_of = s_part[counts++ & 1];
            if (lane == 0) part_of[warp] = c;
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) all += part_of[w];
            return all;
        };
        unsigned o[kSliceEach];   // the candidates in the order of unsigned numbers, else 0
        const unsigned least_o = order_f32(bound + 0.f);
        int c = 0;
#pragma unroll
        for (int j = 0; j < kSliceEach; ++j) {
            const int i = place_of(j);
            const float y = i < n ? __ldcg(src + i) : -INFINITY;
            o[j] = i < n && (y >= bound || bound == -INFINITY) ? order_f32(y == y ? y + 0.f : -INFINITY) : 0u;
            c += o[j] > least_o || i < min(k, n);
            if (i < min(k, n) && !o[j]) c += kSlice;
        }
        // The usual case: what is masked has one value, and the bound is that.  Where the slice's first k elements reach it, no other that equals
        // it is among the k best.
        const int few = count_all(c);
        unsigned least = least_o;
        int upto = k - 1;   // taken: what is above `least`, and what equals it up to this place
        if (few > kListMax) {
            least = 0u;   // the k-th largest
#pragma unroll 1
            for (unsigned bit = 1u << 31; bit; bit >>= 1) {
                c = 0;
#pragma unroll
                for (int j = 0; j < kSliceEach; ++j) c += o[j] >= (least | bit);
                if (count_all(c) >= k) least |= bit;
            }
            c = 0;
#pragma unroll
            for (int j = 0; j < kSliceEach; ++j) c += o[j] > least;
            const int equal = k - count_all(c);   // of the elements that equal it, the first so many
            upto = 0;
#pragma unroll 1
            for (int bit = kSlice / 2; bit; bit >>= 1) {
                c = 0;
#pragma unroll
                for (int j = 0; j < kSliceEach; ++j) c += o[j] == least && place_of(j) < (upto | bit);
                if (count_all(c) < equal) upto |= bit;
            }
        }
        if (t == 0) s_count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSliceEach; ++j)
            if (o[j] > least || (o[j] == least && place_of(j) <= upto))
                s_list[atomicAdd(&s_count, 1)] = (unsigned long long)o[j] << 32 | (0xFFFFFFFFu - (unsigned)(base + place_of(j)));
        __syncthreads();
        have = s_count;
    }
    unsigned long long* out = keys + (row * slices + slice) * k;
    for (int i0 = 0; i0 < have; i0 += kSliceThreads / 4) {   // four threads a candidate
        const int i = i0 + (t >> 2);
        const unsigned long long key = i < have ? s_list[i] : 0ull;
        int rank = 0;
#pragma unroll 4
        for (int j = t & 3; j < have; j += 4) rank += s_list[j] > key;
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if ((t & 3) == 0 && i < have && rank < k) out[rank] = key;
    }
    for (int i = have + t; i < k; i += kSliceThreads) out[i] = 0ull;   // a short slice
}

// The largest of 32 pairs (high, low word), the same in all lanes.
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
    const unsigned hi = (unsigned)(v >> 32), top = __reduce_max_sync(0xffffffffu, hi);
    return (unsigned long long)top << 32 | __reduce_max_sync(0xffffffffu, hi == top ? (unsigned)v : 0u);
}
// Doubles in the order of unsigned numbers (a NaN as minus infinity, -0 as 0).
__device__ __forceinline__ unsigned long long order_f64(double v) {
    v = v == v ? v + 0.0 : -INFINITY;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double from_order_f64(unsigned long long o) { return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o)); }

// A warp merges `lists` sorted lists into their k best: lane l has the lists l, l + 32, .. (NL of them), get(list, i) is entry i of one, 0 behind its
// end, and put(i, list, at, key) is called by the lane that has the i-th best key: entry `at` of `list`.  Equal keys: the lower list.  A
// list's next entry is asked for when the one before it comes to its head.  Returns how many there were.
template <int NL, typename Get, typename Put>
__device__ __forceinline__ int merge_lists(int lane, int k, Get get, Put put) {
    int at[NL];
    unsigned long long head[NL], next[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        at[j] = 0;
        head[j] = get(lane + 32 * j, 0);
        next[j] = get(lane + 32 * j, 1);
    }
    for (int i = 0; i < k; ++i) {
        unsigned long long mine = head[0];
#pragma unroll
        for (int j = 1; j < NL; ++j) mine = max(mine, head[j]);
        const unsigned long long best = warp_max(mine);
        if (!best) return i;
        unsigned from = 1u << 20;
#pragma unroll
        for (int j = NL - 1; j >= 0; --j)
            if (head[j] == best) from = lane + 32 * j;
        from = NL == 1 ? (unsigned)(__ffs(__ballot_sync(0xffffffffu, mine == best)) - 1) : __reduce_min_sync(0xffffffffu, from);
#pragma unroll
        for (int j = 0; j < NL; ++j)
            if (from == (unsigned)(lane + 32 * j)) {
                put(i, (int)from, at[j], best);
                head[j] = next[j];
                next[j] = get((int)from, ++at[j] + 1);
            }
    }
    return k;
}

// CTA per group.  A warp merges the lists of a beam's slices into the beam's k best, `at_once` beams at a time, then one warp the beams' lists
// into the group's.  The lists come into shared memory first where they fit (staged): every one of the k rounds waits for the entry behind
// the one that it takes.
template <int NL>
__global__ void __launch_bounds__(1024) beam_merge_kernel(const float* scores, const int* done, int eos, int beams, int k, int slices, int at_once, bool staged,
                                                          const SliceSum* sums, const unsigned long long* keys, float* out_scores, int* out_rows, int* out_tokens) {
    chained_wait();
    extern __shared__ unsigned long long s_best[];   // the beams' results [beams][k]: keys, then scores; then [at_once][slices][k] where staged
    unsigned long long* s_value = s_best + beams * k;
    __shared__ unsigned char s_done[kBeamMax];
    const int group = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < at_once) {
        for (int b = warp; b < beams; b += at_once) {
            const int64_t row = (int64_t)group * beams + b;
            const bool over = done && __ldcg(done + row);
            const double score = __ldcg(scores + row);
            if (lane == 0) s_done[b] = over;
            if (over) {
                if (lane == 0) s_value[b * k] = order_f64(score);
                continue;
            }
            SliceSum part[NL];
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                part[j].top = -INFINITY;
                part[j].sum = 0.0;
                if (lane + 32 * j < slices) part[j] = sums[row * slices + lane + 32 * j];
                top = fmaxf(top, part[j].top);
            }
            const unsigned long long *src = keys + row * slices * k, *mine = src;
            if (staged) {
                unsigned long long* dst = s_value + (size_t)beams * k + (size_t)warp * slices * k;
#pragma unroll 4
                for (int i = lane; i < slices * k; i += 32) dst[i] = __ldcg(src + i);
                mine = dst;
            }
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < NL; ++j)   // NaN where the row holds a NaN, an infinity or nothing above minus infinity
                if (lane + 32 * j < slices) sum += part[j].sum * exp((double)part[j].top - (double)top);
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const double lse = (double)top + log(sum);
            __syncwarp();
            merge_lists<NL>(
                lane, k, [&](int list, int i) { return list < slices && i < k ? mine[list * k + i] : 0ull; },
                [&](int i, int, int, unsigned long long key) { s_best[b * k + i] = key; });
            __syncwarp();
            for (int i = lane; i < k; i += 32) s_value[b * k + i] = order_f64(score + ((double)key_logit(s_best[b * k + i]) - lse));
        }
    }
    __syncthreads();
    if (warp) return;
    const int64_t o = (int64_t)group * k;
    auto get = [&](int b, int i) { return b < beams && i < (s_done[b] ? 1 : k) ? s_value[b * k + i] : 0ull; };
    auto put = [&](int i, int b, int at, unsigned long long value) {
        out_scores[o + i] = (float)from_order_f64(value);
        out_rows[o + i] = (int)((int64_t)group * beams + b);
        out_tokens[o + i] = s_done[b] ? eos : (int)(0xFFFFFFFFu - (unsigned)s_best[b * k + at]);
    };
    const int have = beams <= 32 ? merge_lists<1>(lane, k, get, put) : merge_lists<4>(lane, k, get, put);
    for (int i = have + lane; i < k; i += 32) {   // all lists are exhausted
        out_scores[o + i] = -INFINITY;
        out_rows[o + i] = -1;
        out_tokens[o + i] = -1;
    }
}

struct BeamWork {
    SliceSum* sums;                  // [rows][slices]
    unsigned long long* keys;        // [rows][slices][k]
};
static int beam_slices(int vocab) { return (vocab + kSlice - 1) / kSlice; }
static uint64_t beam_work_bytes(int64_t rows, int vocab, int k) { return (uint64_t)rows * beam_slices(vocab) * (sizeof(SliceSum) + 8ull * k); }
static BeamWork beam_work(void* work, int64_t rows, int vocab, int k) {
    BeamWork w;
    w.sums = static_cast<SliceSum*>(work);
    w.keys = reinterpret_cast<unsigned long long*>(w.sums + rows * beam_slices(vocab));
    return w;
}
static void check_beams(int groups, int beams, int vocab, int k, const char* who) {
    if (groups < 1 || beams < 1 || beams > kBeamMax || (int64_t)groups * beams > 65535)
        fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d beams in each group, at most 65535 in all, got %d groups of %d", who, kBeamMax, groups, beams);
    if (vocab < 1 || vocab > kSlicesMax * kSlice) fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d tokens, got %d", who, kSlicesMax * kSlice, vocab);
    if (k < 1 || k > kBeamKeep || k > vocab) fail(MFQB_ERR_ARG, "%s: k must be in [1, min(%d, vocab)], got %d", who, kBeamKeep, k);
    if (beams * k > kBeamProduct) fail(MFQB_ERR_UNSUPPORTED, "%s: beams times k must be at most %d, got %d beams and k = %d", who, kBeamProduct, beams, k);
}

}  // namespace mfqb

using namespace mfqb;

extern "C" {
#pragma GCC visibility push(default)

int mfqb_beam_select_work(int groups, int beams, int vocab, int k, uint64_t* bytes) {
    return guarded([&] {
        check_beams(groups, beams, vocab, k, "mfqb_beam_select_work");
        if (!bytes) fail(MFQB_ERR_ARG, "mfqb_beam_select_work: null argument");
        *bytes = beam_work_bytes((int64_t)groups * beams, vocab, k);
    });
}

int mfqb_beam_select(const float* logits, int groups, int beams, int vocab, const float* scores, const int32_t* done, int eos, int k,
                     float* out_scores, int32_t* out_rows, int32_t* out_tokens, void* work, uint64_t work_bytes, mfqb_stream_t stream) {
    return guarded([&] {
        check_beams(groups, beams, vocab, k, "mfqb_beam_select");
        if (!logits || !scores || !out_scores || !out_rows || !out_tokens || !work) fail(MFQB_ERR_ARG, "mfqb_beam_select: null argument");
        const int64_t rows = (int64_t)groups * beams;
        if (((uintptr_t)work & 15) || work_bytes < beam_work_bytes(rows, vocab, k))
            fail(MFQB_ERR_ARG, "mfqb_beam_select: work must be 16-byte aligned and hold %llu bytes, got %llu", (unsigned long long)beam_work_bytes(rows, vocab, k),
                 (unsigned long long)work_bytes);
        const BeamWork w = beam_work(work, rows, vocab, k);
        const bool wide = vocab % 4 == 0 && ((uintptr_t)logits & 15) == 0;
        const int slices = beam_slices(vocab);
        launch_chained(beam_slice_kernel, dim3(slices, (unsigned)rows), dim3(kSliceThreads), 0, stream, logits, static_cast<const int*>(done), vocab, k, slices, wide,
                       w.sums, w.keys);
        // Beams merged at once: as many as find room for their lists beside the results.
        const size_t each = (size_t)slices * k * 8, results = (size_t)beams * k * 16;
        const bool staged = results + each <= kMergeSmem;
        const int at_once = staged ? (int)std::min<size_t>({32, (size_t)beams, (kMergeSmem - results) / each}) : std::min(32, beams);
        const size_t smem = results + (staged ? at_once * each : 0);
        if (smem > 40 * 1024) {
            int device = 0;
            MFQB_CUDA(cudaGetDevice(&device));
            static std::once_flag once[64];
            std::call_once(once[device], [] {
                for (auto* f : {beam_merge_kernel<1>, beam_merge_kernel<4>})
                    MFQB_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMergeSmem));
            });
        }
        launch_chained(slices <= 32 ? beam_merge_kernel<1> : beam_merge_kernel<4>, dim3(groups), dim3(1024), smem, stream, scores, static_cast<const int*>(done), eos,
                       beams, k, slices, at_once, staged, static_cast<const SliceSum*>(w.sums), static_cast<const unsigned long long*>(w.keys), out_scores,
                       static_cast<int*>(out_rows), static_cast<int*>(out_tokens));
    });
}

#pragma GCC visibility pop
}  // extern "C"
