// How much every position was looked at: the sums of the attention's weights over the nodes and over the heads that share a kv head, added to
// one float32 per layer, sequence, kv head and position.
//
// weight(row, position) = exp2(scale' s - m) / l with the row's final maximum m and sum l, which tree_attn_kernel and tree_merge_kernel leave.  A
// position belongs to one thread, which adds the rows in their order: no atomics, a call repeats bit for bit.
#include "tree_attn.cuh"

namespace mfqb {

constexpr int kScoreRows = 64;                     // up to so many rows the attention may keep its scores
constexpr uint64_t kScoreBytes = 512ull << 20;     // as long as they take at most this
constexpr int kWeighRows = 256;                    // rows of a pass over the keys
constexpr int kWeighRing = 4, kWeighThreads = 320;

int64_t tree_score_stride(const mfqb_cache& c, int q_heads, int nodes) {
    const int64_t m_rows = (int64_t)nodes * (q_heads / c.kv_heads), stride = ((int64_t)c.width * c.page + kTile - 1) / kTile * kTile;
    return m_rows <= kScoreRows && 4ull * c.rows * c.kv_heads * m_rows * stride <= kScoreBytes ? stride : 0;
}
uint64_t tree_weigh_bytes(const mfqb_cache& c, int q_heads, int nodes) {
    const uint64_t rows = (uint64_t)c.rows * c.kv_heads * nodes * (q_heads / c.kv_heads);
    return rows * 8 + 4 * rows * tree_score_stride(c, q_heads, nodes);
}

// From the scores that the attention has kept.  CTA (stretch of positions, kv head, sequence), four positions a thread.
__global__ void __launch_bounds__(128) weigh_scores_kernel(const __grid_constant__ TreeArgs a, float* weights) {
    chained_wait();
    __shared__ float2 s_ml[kScoreRows];
    const int kvh = blockIdx.y, r = blockIdx.z, m_rows = a.nodes * a.group;
    const int64_t item = (int64_t)r * a.kv_heads + kvh;
    if ((int)threadIdx.x < m_rows) s_ml[threadIdx.x] = __ldcg(a.row_ml + item * m_rows + threadIdx.x);
    __syncthreads();
    const TreeSeq seq = tree_seq(a, r);
    const float* scores = a.scores + item * m_rows * a.score_stride;
    float* to = weights + item * a.width * a.page;
    for (int pos = (blockIdx.x * 128 + threadIdx.x) * 4; pos < seq.end; pos += gridDim.x * 512) {   // four positions lie in one page
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int row = 0; row < m_rows; ++row) {
            const float2 ml = s_ml[row];
            const float4 s = __ldcg(reinterpret_cast<const float4*>(scores + row * a.score_stride + pos));
            const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += v[e] == -INFINITY ? 0.f : exp2_approx(fmaf(v[e], a.scale_log2, -ml.x)) * ml.y;
        }
        const int page = __ldcg(a.table + (int64_t)r * a.width + pos / a.page);
        const bool good = (unsigned)page < (unsigned)a.pages;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (pos + e >= seq.end) break;
            if (pos + e >= seq.len) to[pos + e] = good ? sum[e] : 0.f;
            else if (good) to[pos + e] += sum[e];
        }
    }
}

struct WeighShared {
    uint64_t k_full[kWeighRing], k_empty[kWeighRing], q_full, s_full[2], s_empty[2], all;
    int64_t scan[kWeighThreads / 32], first, last, off;
    int row0, failed;
    int bad;                         // the last head (its number in the CTA, from 1 on) with a row whose weights are no numbers
    uint32_t tmem;
    unsigned good[8];
    unsigned long long masks[kTreeNodes];
    float4 ml[kWeighRows / 2];   // of two rows: minus their maxima, the factors
};
constexpr size_t kWeighSmem = (size_t)kWeighRing * kTileBytes + (size_t)kWeighRows * kHeadDim * 2 + sizeof(WeighShared);
static_assert(kWeighSmem <= 227 * 1024, "shared memory of an SM");

// A CTA's tiles in order: sequence, kv head, tile of 128 positions.
struct WeighWalk {
    int r, kvh, t;
    int64_t left;
    bool fresh;   // the tile is the first of its head here
    TreeSeq seq;
    __device__ __forceinline__ void start(const TreeArgs& a, const WeighShared& sh) {
        left = sh.last - sh.first;
        fresh = true;
        if (left <= 0) return;
        r = sh.row0;
        seq = tree_seq(a, r);
        kvh = (int)quotient(sh.off, seq.tiles);
        t = (int)(sh.off - (int64_t)kvh * seq.tiles);
    }
    __device__ __forceinline__ void next(const TreeArgs& a) {
        fresh = false;
        if (--left <= 0) return;
        if (++t < seq.tiles) return;
        t = 0;
        fresh = true;
        if (++kvh < a.kv_heads) return;
        kvh = 0;
        seq = tree_seq(a, ++r);
    }
};

// From the keys, by rows row0 .. row0 + rows of Q: S^T = K Q^T puts a position into each lane of tensor memory, so that the sum over the rows stays in
// a thread.  One warp asks for the pages' keys, one issues tcgen05.mma, two groups of four warps take the tiles in turns.
__global__ void __launch_bounds__(kWeighThreads, 1) tree_weigh_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap kmap, float* weights, int row0, int rows) {
    extern __shared__ __align__(1024) unsigned char ring[];
    unsigned char* q_tile = ring + (size_t)kWeighRing * kTileBytes;   // two halves of 64 dims, kWeighRows rows of 128 bytes each
    constexpr int kQHalf = kWeighRows * 128;
    WeighShared& sh = *reinterpret_cast<WeighShared*>(q_tile + 2 * kQHalf);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (smem_u32(ring) & 1023u) {   // not the case with no static shared memory
        if (tid == 0) atomicExch(a.error, MFQB_ERR_CUDA);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < kWeighRing; ++i) { mbar_init(&sh.k_full[i], 1); mbar_init(&sh.k_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.s_full[i], 1); mbar_init(&sh.s_empty[i], 4); }
        mbar_init(&sh.q_full, 8);
        mbar_init(&sh.all, 8);
        sh.failed = sh.bad = 0;
        sh.first = sh.last = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(&sh.tmem, 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    chained_wait();
    {   // this CTA's tiles: thread t holds the sequences kEach * t ..
        constexpr int kEach = (kCacheRows + kWeighThreads - 1) / kWeighThreads;
        int64_t tiles_of[kEach], mine = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            tiles_of[j] = kEach * tid + j < a.rows ? (int64_t)tree_seq(a, kEach * tid + j).tiles * a.kv_heads : 0;
            mine += tiles_of[j];
        }
        int64_t upto = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) sh.scan[warp] = upto;
        __syncthreads();
        int64_t total = 0;
        for (int i = 0; i < kWeighThreads / 32; ++i) {
            if (i < warp) upto += sh.scan[i];
            total += sh.scan[i];
        }
        const int64_t quota = quotient(total + gridDim.x - 1, gridDim.x), first = blockIdx.x * quota, last = min(total, first + quota);
        int64_t begin = upto - mine;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int64_t end = begin + tiles_of[j];
            if (first < last && begin <= first && first < end) {
                sh.row0 = kEach * tid + j;
                sh.off = first - begin;
                sh.first = first;
                sh.last = last;
            }
            begin = end;
        }
        __syncthreads();
    }
    WeighWalk w;
    w.start(a, sh);
    const int m_rows = a.nodes * a.group;
    if (warp == 0) {
        const int box = min(a.page, kTile), boxes = kTile / box;
        uint32_t j = 0;
        bool ok = true;
        for (; w.left > 0; w.next(a), ++j) {
            const int pos = w.t * kTile + lane * box;
            int page = -1;
            if (lane < boxes && pos < w.seq.end) page = __ldcg(a.table + (int64_t)w.r * a.width + pos / a.page);
            if ((unsigned)page >= (unsigned)a.pages) page = -1;
            const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
            const uint32_t stage = j % kWeighRing;
            ok = warp_wait(&sh.k_empty[stage], ((j / kWeighRing) & 1u) ^ 1u);
            if (!ok) break;
            if (lane == 0) {
                unsigned good = 0;   // groups of 16 positions with a page
                for (int g = 0; g < 8; ++g) good |= ((have >> (g * 16 / box)) & 1u) << g;
                sh.good[j & 7] = good;   // read behind the product's barrier, at most two tiles later than the next one is asked for
                mbar_arrive_expect_tx(&sh.k_full[stage], (uint32_t)__popc(have) * (uint32_t)box * 256u);
            }
            __syncwarp();
            if (page >= 0) {
                unsigned char* dst = ring + (size_t)stage * kTileBytes + lane * box * 128;
                const int y = pos & (a.page - 1);
                tma_load_4d(dst, &kmap, 0, y, w.kvh, page, &sh.k_full[stage]);
                tma_load_4d(dst + kHalfBytes, &kmap, 64, y, w.kvh, page, &sh.k_full[stage]);
            }
            __syncwarp();
        }
        if (!ok) sh.failed = 1;
        for (uint32_t i = 1; i <= min(j, (uint32_t)kWeighRing); ++i)   // no copy outlives the CTA
            if (!warp_wait(&sh.k_full[(j - i) % kWeighRing], ((j - i) / kWeighRing) & 1u)) sh.failed = 1;
    } else if (warp == 1) {
        const uint32_t idesc = __shfl_sync(0xffffffffu, instr_desc_bf16(kTile, (rows + 15) / 16 * 16, false), 0);
        const uint32_t q_addr = smem_u32(q_tile), ring_addr = smem_u32(ring);
        uint32_t j = 0, items = 0;
        bool ok = true;
        for (; w.left > 0; w.next(a), ++j) {
            const uint32_t stage = j % kWeighRing, g = j & 1u;
            ok = (!w.fresh || warp_wait(&sh.q_full, items & 1u)) && warp_wait(&sh.k_full[stage], (j / kWeighRing) & 1u) &&
                 warp_wait(&sh.s_empty[g], ((j >> 1) & 1u) ^ 1u);
            if (!ok) break;
            items += w.fresh;
            tc_fence_after_sync();
            const uint32_t k = __shfl_sync(0xffffffffu, ring_addr + stage * kTileBytes, 0), q = __shfl_sync(0xffffffffu, q_addr, 0);
            const uint32_t d = __shfl_sync(0xffffffffu, tmem + g * kWeighRows, 0);
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    tc_mma_f16_ss(d, smem_desc_sw128(k + (s >> 2) * kHalfBytes + (s & 3) * 32), smem_desc_sw128(q + (s >> 2) * kQHalf + (s & 3) * 32), idesc, s > 0);
                tc_commit(&sh.s_full[g]);
                tc_commit(&sh.k_empty[stage]);
            }
            __syncwarp();
        }
        if (!ok) sh.failed = 1;
    } else {
        const int g = (warp - 2) >> 2, quarter = warp & 3, t = tid - 64;
        const uint32_t col = tmem + ((uint32_t)(quarter * 32) << 16) + g * kWeighRows;
        const uint64_t scale2 = pair_f32(a.scale_log2, a.scale_log2);
        uint32_t j = 0, alls = 0;
        int items = 0;
        bool ok = true;
        auto all_sync = [&]() {
            warp_arrive(&sh.all);
            ok = ok && warp_wait(&sh.all, alls++ & 1u);
        };
        for (; ok && w.left > 0; w.next(a), ++j) {
            if (w.fresh) {   // all tiles of the head before have been summed, and their products read the rows that change now
                all_sync();
                if (!ok) break;
                ++items;
                const int c = t & 15, padded = (rows + 15) / 16 * 16;
                for (int r0 = t >> 4; r0 < padded; r0 += 128) {   // rows behind the last one repeat it
                    uint4 v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (r0 + 16 * u < padded) v[u] = __ldcg(reinterpret_cast<const uint4*>(a.q + a.row_at(w.r, w.kvh, min(row0 + r0 + 16 * u, m_rows - 1))) + c);
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int rr = r0 + 16 * u;
                        if (rr < padded) *reinterpret_cast<uint4*>(q_tile + (c >> 3) * kQHalf + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[u];
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&sh.q_full);
                if (t < kWeighRows) {   // rows behind the last one have its maximum and count for nothing
                    const float2 ml = __ldcg(a.row_ml + ((int64_t)w.r * a.kv_heads + w.kvh) * m_rows + min(row0 + t, row0 + rows - 1));
                    float* to = reinterpret_cast<float*>(&sh.ml[t >> 1]) + (t & 1);
                    to[0] = -ml.x;
                    to[2] = t < rows ? ml.y : 0.f;
                    if (t < rows && !(fabsf(ml.x) < INFINITY && ml.y < INFINITY)) sh.bad = items;   // NaN too
                }
                if (t < kTreeNodes) sh.masks[t] = t < a.nodes ? __ldcg(a.masks + (int64_t)w.r * a.nodes + t) : 0ull;
                all_sync();
                if (!ok) break;
            }
            if ((int)(j & 1u) != g) continue;
            const int at = quarter * 32 + lane, pos = w.t * kTile + at, node = pos - w.seq.len;
            float* to = weights + ((int64_t)w.r * a.kv_heads + w.kvh) * a.width * a.page + pos;
            const bool adds = pos < w.seq.end && (node < 0 || row0 > 0);   // to what is there
            const float before = adds ? *to : 0.f;
            ok = warp_wait(&sh.s_full[g], (j >> 1) & 1u);
            if (!ok) break;
            tc_fence_after_sync();
            const unsigned good = sh.good[j & 7];
            const bool page = (good >> (at >> 4)) & 1u;
            uint64_t sum2[2] = {0ull, 0ull};
            // Sixteen rows at a time, the next ones' scores on their way; columns behind the last row are products with it too.
            auto rows_of = [&](auto each) {
                const int chunks = (rows + 15) / 16;
                uint32_t s[2][16];
                tmem_ld16_async(col, s[0]);
#pragma unroll 1
                for (int c = 0; c < chunks; c += 2) {
                    tmem_wait_ld16(s[0]);
                    if (c + 1 < chunks) tmem_ld16_async(col + 16 * (c + 1), s[1]);
                    each(16 * c, s[0]);
                    if (c + 1 < chunks) {
                        tmem_wait_ld16(s[1]);
                        if (c + 2 < chunks) tmem_ld16_async(col + 16 * (c + 2), s[0]);
                        each(16 * (c + 1), s[1]);
                    }
                }
            };
            if (w.t * kTile + kTile <= w.seq.len && good == 0xFFu && sh.bad != items) {
                rows_of([&](int c, const uint32_t* s) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float4 ml = sh.ml[(c + e) >> 1];
                        const float2 x = split_f32(fma_f32x2(pair_f32(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, pair_f32(ml.x, ml.y)));
                        sum2[(e >> 1) & 1] = fma_f32x2(pair_f32(exp2_approx(x.x), exp2_approx(x.y)), pair_f32(ml.z, ml.w), sum2[(e >> 1) & 1]);
                    }
                });
            } else {   // a row counts where it sees the position and its score is above minus infinity
                unsigned long long seen = ~0ull;   // by which nodes the position is
                if (!page || node >= a.nodes) {
                    seen = 0ull;
                } else if (node >= 0) {
                    seen = 0ull;
                    for (int i = 0; i < a.nodes; ++i) seen |= ((sh.masks[i] >> node) & 1ull) << i;
                }
                rows_of([&](int c, const uint32_t* s) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float4 ml = sh.ml[(c + e) >> 1];
                        float p[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const float x = __uint_as_float(s[e + u]);
                            const bool on = ((seen >> a.node_of(min(row0 + c + e + u, m_rows - 1))) & 1ull) && x != -INFINITY && c + e + u < rows;
                            p[u] = on ? exp2_approx(fmaf(x, a.scale_log2, u ? ml.y : ml.x)) * (u ? ml.w : ml.z) : 0.f;
                        }
                        sum2[(e >> 1) & 1] = add_f32x2(pair_f32(p[0], p[1]), sum2[(e >> 1) & 1]);
                    }
                });
            }
            const float2 half = split_f32(add_f32x2(sum2[0], sum2[1]));
            const float sum = half.x + half.y;
            tc_fence_before_sync();
            warp_arrive(&sh.s_empty[g]);
            if (adds) {
                if (page) *to = before + sum;
            } else if (pos < w.seq.end) {
                *to = sum;
            }
        }
        if (!ok) sh.failed = 1;
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_free(tmem, 512);
        if (lane == 0 && sh.failed) atomicExch(a.error, MFQB_ERR_TIMEOUT);
    }
}

void launch_tree_weigh(const mfqb_cache& c, const TreeArgs& a, float* weights, cudaStream_t s) {
    const int m_rows = a.nodes * a.group;
    const int64_t cap = (int64_t)c.width * c.page, items = (int64_t)c.rows * c.kv_heads;
    if (a.scores) {
        // as many CTAs as fill the SMs several times, none for positions that the table cannot hold
        const int64_t each = std::min((cap + 511) / 512, std::max<int64_t>(1, 8 * kTreeSms / items));
        launch_chained(weigh_scores_kernel, dim3((unsigned)each, c.kv_heads, c.rows), dim3(128), 0, s, a, weights);
        return;
    }
    int device = 0;
    MFQB_CUDA(cudaGetDevice(&device));
    static std::once_flag once[64];
    std::call_once(once[device], [] { MFQB_CUDA(cudaFuncSetAttribute(tree_weigh_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kWeighSmem)); });
    const CUtensorMap kmap = page_map(a.k, c);
    const unsigned ctas = (unsigned)std::min<int64_t>(kTreeSms, items * ((cap + kTile - 1) / kTile));
    for (int row0 = 0; row0 < m_rows; row0 += kWeighRows)
        launch_chained(tree_weigh_kernel, dim3(ctas), dim3(kWeighThreads), kWeighSmem, s, a, kmap, weights, row0, std::min(kWeighRows, m_rows - row0));
}

}  // namespace mfqb
