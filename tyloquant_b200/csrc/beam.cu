// Beam selection: the k best continuations of a group of beams by score + log softmax(logits), one pass over the logits.
#include "paged.h"

namespace mfqb {

constexpr int kBeamMax = 128, kBeamKeep = 128;   // beams of a group, candidates kept
constexpr int kSliceThreads = 256, kSliceEach = 32, kSlice = kSliceThreads * kSliceEach;
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

// CTA (slice, row).  A thread keeps its 32 logits in registers: element (j * 256 + thread) * 4 + e of the slice whatever the row's
// alignment, so that equal rows have equal sums to the last bit and ties between beams are ties.  Of the k best candidates every
// one is at least the k-th largest of the threads' own best: what reaches that bound (at most 32 k, mostly some k) goes
// into a list, and a candidate's place is the number of larger ones in it.
__global__ void __launch_bounds__(kSliceThreads) beam_slice_kernel(const float* __restrict__ logits, const int* __restrict__ done, int vocab, int k, int slices,
                                                                   bool wide, SliceSum* __restrict__ sums, unsigned long long* __restrict__ keys) {
    chained_wait();
    extern __shared__ unsigned long long s_list[];   // [kSliceEach * k]
    __shared__ unsigned long long s_best[kSliceThreads];
    __shared__ float s_top[8];
    __shared__ double s_sum[8];
    __shared__ int s_count;
    __shared__ unsigned long long s_bound;
    const int t = threadIdx.x, slice = blockIdx.x;
    const int64_t row = blockIdx.y;
    if (done && done[row]) return;
    const int base = slice * kSlice;
    const float* src = logits + row * vocab + base;
    const int n = min(kSlice, vocab - base);
    float x[kSliceEach];
#pragma unroll
    for (int j = 0; j < kSliceEach / 4; ++j) {
        const int i = (j * kSliceThreads + t) * 4;
        if (wide && i + 4 <= n) {
            const float4 v = __ldcs(reinterpret_cast<const float4*>(src + i));
            x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * j + e] = i + e < n ? __ldcs(src + i + e) : -INFINITY;
        }
    }
    unsigned long long best = 0ull;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSliceEach; ++j) {
        const int i = ((j >> 2) * kSliceThreads + t) * 4 + (j & 3);
        if (i < n) {
            best = max(best, beam_key(x[j], (unsigned)(base + i)));
            top = fmaxf(top, x[j]);
        }
    }
    s_best[t] = best;
    if (t == 0) s_count = 0;
    if (t == 0) s_bound = 1ull;
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((t & 31) == 0) s_top[t >> 5] = top;
    __syncthreads();
    top = s_top[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, s_top[w]);
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < kSliceEach; ++j) {
        const int i = ((j >> 2) * kSliceThreads + t) * 4 + (j & 3);
        if (i < n && x[j] != -INFINITY) part += expf(x[j] - top);
    }
    double sum = part;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((t & 31) == 0) s_sum[t >> 5] = sum;
    int above = 0;
    for (int j = 0; j < kSliceThreads; ++j) above += s_best[j] > best;
    if (above == k - 1 && best) s_bound = best;   // keys differ, so one thread at most
    __syncthreads();
    if (t == 0) {
        sum = s_sum[0];
        for (int w = 1; w < 8; ++w) sum += s_sum[w];
        sums[row * slices + slice] = SliceSum{sum, top, 0.f};
    }
    const unsigned long long bound = s_bound;
    if (best >= bound) {
#pragma unroll
        for (int j = 0; j < kSliceEach; ++j) {
            const int i = ((j >> 2) * kSliceThreads + t) * 4 + (j & 3);
            if (i < n) {
                const unsigned long long key = beam_key(x[j], (unsigned)(base + i));
                if (key >= bound) s_list[atomicAdd(&s_count, 1)] = key;   // the order in the list does not matter
            }
        }
    }
    __syncthreads();
    const int have = s_count;
    unsigned long long* out = keys + (row * slices + slice) * k;
    for (int i = t; i < have; i += kSliceThreads) {
        const unsigned long long key = s_list[i];
        int rank = 0;
        for (int j = 0; j < have; ++j) rank += s_list[j] > key;
        if (rank < k) out[rank] = key;
    }
    for (int i = have + t; i < k; i += kSliceThreads) out[i] = 0ull;   // a short slice
}

// CTA per group.  A warp merges the lists of a beam's slices into the beam's k best, then one warp the beams' lists into the group's.
__global__ void __launch_bounds__(1024) beam_merge_kernel(const float* __restrict__ scores, const int* __restrict__ done, int eos, int beams, int k, int slices,
                                                          const SliceSum* __restrict__ sums, const unsigned long long* __restrict__ keys,
                                                          unsigned long long* __restrict__ beam_keys, float* __restrict__ out_scores,
                                                          int* __restrict__ out_rows, int* __restrict__ out_tokens) {
    chained_wait();
    __shared__ double s_lse[kBeamMax], s_score[kBeamMax];
    __shared__ unsigned char s_done[kBeamMax];
    const int group = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = warp; b < beams; b += 32) {
        const int64_t row = (int64_t)group * beams + b;
        const bool over = done && done[row];
        if (lane == 0) {
            s_done[b] = over;
            s_score[b] = scores[row];
        }
        if (over) continue;
        float top = -INFINITY;
        for (int s = lane; s < slices; s += 32) top = fmaxf(top, sums[row * slices + s].top);
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        double sum = 0.0;
        for (int s = lane; s < slices; s += 32) {
            const SliceSum v = sums[row * slices + s];
            sum += v.sum * exp((double)v.top - (double)top);   // NaN where the row holds a NaN, an infinity or nothing above minus infinity
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_lse[b] = (double)top + log(sum);
        const unsigned long long* src = keys + row * slices * k;
        unsigned long long* dst = beam_keys + row * k;
        int at[4] = {0, 0, 0, 0};   // next entry of this lane's lists
        unsigned long long head[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) head[j] = lane + 32 * j < slices ? src[(int64_t)(lane + 32 * j) * k] : 0ull;
        for (int i = 0; i < k; ++i) {
            unsigned long long m = max(max(head[0], head[1]), max(head[2], head[3]));
            for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) dst[i] = m;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (m && head[j] == m) head[j] = ++at[j] < k ? src[(int64_t)(lane + 32 * j) * k + at[j]] : 0ull;
        }
    }
    __syncthreads();
    if (warp) return;
    // beams lane, lane + 32, ...: head candidate, its score in 64 bits
    int at[4] = {0, 0, 0, 0};
    double head[4];
    auto fetch = [&](int j) {
        const int b = lane + 32 * j;
        if (b >= beams || at[j] >= (s_done[b] ? 1 : k)) {
            at[j] = 1 << 20;   // exhausted
            return;
        }
        double v = s_score[b];
        if (!s_done[b]) v += (double)key_logit(beam_keys[((int64_t)group * beams + b) * k + at[j]]) - s_lse[b];
        head[j] = v == v ? v : -INFINITY;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) fetch(j);
    for (int i = 0; i < k; ++i) {
        double best = 0.0;
        int from = 1 << 20;   // the beam
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at[j] < (1 << 20) && (from == (1 << 20) || head[j] > best)) {
                best = head[j];
                from = lane + 32 * j;
            }
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, best, o);
            const int f = __shfl_xor_sync(0xffffffffu, from, o);
            if (f != (1 << 20) && (from == (1 << 20) || v > best || (v == best && f < from))) {
                best = v;
                from = f;
            }
        }
        const int64_t o = (int64_t)group * k + i;
        if (from == (1 << 20)) {   // all lists are exhausted
            if (lane == 0) {
                out_scores[o] = -INFINITY;
                out_rows[o] = -1;
                out_tokens[o] = -1;
            }
            continue;
        }
        if (lane == (from & 31)) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j == from >> 5) {
                    const int64_t row = (int64_t)group * beams + from;
                    out_scores[o] = (float)best;
                    out_rows[o] = (int)row;
                    out_tokens[o] = s_done[from] ? eos : (int)(0xFFFFFFFFu - (unsigned)beam_keys[row * k + at[j]]);
                    ++at[j];
                    fetch(j);
                }
        }
    }
}

struct BeamWork {
    SliceSum* sums;                  // [rows][slices]
    unsigned long long* keys;        // [rows][slices][k]
    unsigned long long* beam_keys;   // [rows][k]
};
static int beam_slices(int vocab) { return (vocab + kSlice - 1) / kSlice; }
static uint64_t beam_work_bytes(int64_t rows, int vocab, int k) { return (uint64_t)rows * beam_slices(vocab) * (sizeof(SliceSum) + 8ull * k) + (uint64_t)rows * k * 8ull; }
static BeamWork beam_work(void* work, int64_t rows, int vocab, int k) {
    BeamWork w;
    w.sums = static_cast<SliceSum*>(work);
    w.keys = reinterpret_cast<unsigned long long*>(w.sums + rows * beam_slices(vocab));
    w.beam_keys = w.keys + rows * beam_slices(vocab) * k;
    return w;
}
static void check_beams(int groups, int beams, int vocab, int k, const char* who) {
    if (groups < 1 || beams < 1 || beams > kBeamMax || (int64_t)groups * beams > 65535)
        fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d beams in each group, at most 65535 in all, got %d groups of %d", who, kBeamMax, groups, beams);
    if (vocab < 1 || vocab > kSlicesMax * kSlice) fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d tokens, got %d", who, kSlicesMax * kSlice, vocab);
    if (k < 1 || k > kBeamKeep || k > vocab) fail(MFQB_ERR_ARG, "%s: k must be in [1, min(%d, vocab)], got %d", who, kBeamKeep, k);
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
        launch_chained(beam_slice_kernel, dim3(beam_slices(vocab), (unsigned)rows), dim3(kSliceThreads), (size_t)kSliceEach * k * 8, stream, logits,
                       static_cast<const int*>(done), vocab, k, beam_slices(vocab), wide, w.sums, w.keys);
        launch_chained(beam_merge_kernel, dim3(groups), dim3(1024), 0, stream, scores, static_cast<const int*>(done), eos, beams, k, beam_slices(vocab),
                       static_cast<const SliceSum*>(w.sums), static_cast<const unsigned long long*>(w.keys), w.beam_keys, out_scores,
                       static_cast<int*>(out_rows), static_cast<int*>(out_tokens));
    });
}

#pragma GCC visibility pop
}  // extern "C"
