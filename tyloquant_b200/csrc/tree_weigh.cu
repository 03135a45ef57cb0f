// How much every position was looked at: the sums of the attention's weights over the nodes and over the heads that share a kv head, added to
// one float32 per layer, sequence, kv head and position.
//
// weight(row, position) = exp2(scale' s - m) / l with the row's final maximum m and sum l, which tree_attn_kernel and tree_merge_kernel leave.  A
// position belongs to one thread, which adds the rows in their order: no atomics, a call repeats bit for bit.
#include "tree_attn.cuh"

namespace mfqb {

constexpr uint64_t kScoreBytes = 512ull << 20;     // as long as they take at most this
constexpr int kWeighRows = 256;                    // rows of a pass over the keys
constexpr int kWeighRing = 4, kWeighGroups = 4, kWeighThreads = 64 + 128 * kWeighGroups;   // a loader, an issuer, groups of four warps that sum

// Scores are four bytes a row and position, written and read once: up to 32 rows that is less than the 256 bytes of a key, which the other form reads again; up
// to 64 it saves a launch (kept: 1 to 3 us of the attention's time, the sums beside its merge).
int64_t tree_score_stride(const mfqb_cache& c, int q_heads, int nodes) {
    const int64_t m_rows = (int64_t)nodes * (q_heads / c.kv_heads), stride = ((int64_t)c.width * c.page + kTile - 1) / kTile * kTile;
    return m_rows <= kScoreRows && 4ull * c.rows * c.kv_heads * m_rows * stride <= kScoreBytes ? stride : 0;
}
uint64_t tree_weigh_bytes(const mfqb_cache& c, int q_heads, int nodes) {
    const uint64_t rows = (uint64_t)c.rows * c.kv_heads * nodes * (q_heads / c.kv_heads);
    return rows * 8 + 4 * rows * tree_score_stride(c, q_heads, nodes);
}

struct WeighShared {
    uint64_t k_full[kWeighRing], k_empty[kWeighRing], q_full, s_full[2], s_empty[2], all, half[4];
    int64_t scan[kWeighThreads / 32], first, last, off;
    int row0, failed;
    int bad;                         // the last head (its number in the CTA, from 1 on) with a row whose weights are no numbers, or that does not count
    uint32_t tmem;
    unsigned good[8];
    unsigned long long seen_by[kTreeNodes];   // by which nodes a node is
    float sum[4][kTile];         // of the rows' second half, of every fourth tile
    float4 shift[kWeighRows / 4];   // of every row: - maximum - log2(sum), so that weight = exp2(scale' score + shift)
};
constexpr size_t kWeighSmem = (size_t)kWeighRing * kTileBytes + (size_t)kWeighRows * kHeadDim * 2 + sizeof(WeighShared);
static_assert(kWeighSmem <= 227 * 1024, "shared memory of an SM");

// What tiles with nodes, which not every row sees, take in units of the others: they are shared out so (27 nodes of 13 sequences,
// with the attention: 42 us, 48 with even shares).
constexpr int kWeighNodes = 4;

// A CTA's tiles in order: sequence, kv head, tile of 128 positions.  A tile belongs to the CTA in whose units its first one lies.
struct WeighWalk {
    int r, kvh, t;
    int64_t left;   // units from the head's first one to the CTA's last
    bool fresh;     // the tile is the first of its head here
    TreeSeq seq;
    static __device__ __forceinline__ int unit_of(const TreeSeq& s, int t) { return t + (kWeighNodes - 1) * max(0, t - s.len / kTile); }
    static __device__ __forceinline__ int units_of(const TreeSeq& s) { return unit_of(s, s.tiles); }
    __device__ __forceinline__ void start(const TreeArgs& a, const WeighShared& sh) {
        left = sh.last - sh.first;
        if (left <= 0) return;
        r = sh.row0;
        seq = tree_seq(a, r);
        const int units = units_of(seq);
        kvh = (int)quotient(sh.off, units);
        const int u0 = (int)(sh.off - (int64_t)kvh * units), plain = seq.len / kTile;
        left += u0;
        t = (u0 <= plain ? u0 : plain + (u0 - plain + kWeighNodes - 1) / kWeighNodes) - 1;
        next(a);
        fresh = true;
    }
    __device__ __forceinline__ void next(const TreeArgs& a) {
        fresh = false;
        if (++t < seq.tiles) {
            if (unit_of(seq, t) >= left) left = 0;
            return;
        }
        left = max(left - units_of(seq), (int64_t)0);
        if (left == 0) return;
        t = 0;
        fresh = true;
        if (++kvh < a.kv_heads) return;
        kvh = 0;
        if (++r >= a.rows) {   // only where lengths change meanwhile
            left = 0;
            return;
        }
        seq = tree_seq(a, r);
    }
};

// A position that not every row sees, or (BAD) where weights of some rows are no numbers or some do not count (a shift of minus infinity, whatever the
// scores): a row counts where it sees the position and its score is above minus infinity.
template <bool BAD>
__device__ __noinline__ float weigh_some(const TreeArgs& a, const float4* s_shift, uint32_t col, int row0, int rows, unsigned long long seen) {
    const int m_rows = a.nodes * a.group;
    uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll 1
    for (int c = 0; c < rows; c += 16) {
        uint32_t s[16];
        __syncwarp();   // loads from tensor memory and their wait want the warp together; what lies between goes by the lane's position
        tmem_ld16_async(col + c, s);
        unsigned in = rows - c >= 16 ? 0xFFFFu : (1u << (rows - c)) - 1u;   // of these 16
        if (seen != ~0ull) {
            unsigned by = 0u;
            const int n0 = a.node_of(row0 + c), n1 = a.node_of(min(row0 + c + 15, m_rows - 1));
            for (int i = n0; i <= n1; ++i) {   // a node's rows, at most 16, follow each other
                const int from = i * a.group - (row0 + c);
                const unsigned run = (1u << a.group) - 1u;
                if ((seen >> i) & 1ull) by |= from >= 0 ? run << from : run >> -from;
            }
            in &= by;
        }
        __syncwarp();
        tmem_wait_ld16(s);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 m = s_shift[(c + e) / 4];
            const float shift[4] = {m.x, m.y, m.z, m.w};
            float p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float x = __uint_as_float(s[e + u]);
                p[u] = (in >> (e + u)) & 1u && (!BAD || (x != -INFINITY && shift[u] != -INFINITY)) ? exp2_approx(fmaf(x, a.scale_log2, shift[u])) : 0.f;
            }
            sum2[0] = add_f32x2(sum2[0], pair_f32(p[0], p[1]));
            sum2[1] = add_f32x2(sum2[1], pair_f32(p[2], p[3]));
        }
    }
    const float2 two = split_f32(add_f32x2(sum2[0], sum2[1]));
    return two.x + two.y;
}

// From the keys, by rows row0 .. row0 + rows of Q: S^T = K Q^T puts a position into each lane of tensor memory, so that the sum over the rows stays in
// a thread, and a tile of 128 positions is one product for up to 256 rows.  One warp asks for the pages' keys (a look into the table two tiles ahead: 3 us of
// 280), one issues tcgen05.mma, and of sixteen that sum a group of four has a half of the rows of every other tile; the second halves' sums
// wait in shared memory until the first group's next tile.
// weight = exp2(scale' s + shift), shift = - m - log2(l): one number per row, read from shared memory by all threads at once (two, m and 1 / l, made
// it 8 us more).  Its rounding grows with the scores: a shift of size 2^5 is off by 2^-19 at most and the weight by 0.7 times that of itself, one of 2^10 by 2^-14.  That is
// as much as a float32 score of this size is off by itself; weights from kept scores, which keep m and 1 / l apart, are nearer where scores happen to be exact.
// Bound by latency: the chain product - scores out of tensor memory (some 500 clocks a load) - exponentials - hand-over, with two tiles of scores in flight.  4
// sequences at 32768 positions, 64 nodes in groups of 4, 8 kv heads: 124 us where the exponentials' unit needs 62 and the keys 41.  Eight warps with
// loads of 32 rows ahead took 133 to 143, products of 128 rows each in four places 122 to 131 with slower short batches.
__global__ void __launch_bounds__(kWeighThreads, 1) tree_weigh_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap kmap, int row0, int rows) {
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
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.s_full[i], 1); mbar_init(&sh.s_empty[i], 8); }
        for (int i = 0; i < 4; ++i) mbar_init(&sh.half[i], 4);
        mbar_init(&sh.q_full, 4 * kWeighGroups);
        mbar_init(&sh.all, 4 * kWeighGroups);
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
            tiles_of[j] = kEach * tid + j < a.rows ? (int64_t)WeighWalk::units_of(tree_seq(a, kEach * tid + j)) * a.kv_heads : 0;
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
        auto look = [&](const WeighWalk& x) {   // this lane's page of a tile
            const int pos = x.t * kTile + lane * box;
            return x.left > 0 && lane < boxes && pos < x.seq.end ? __ldcg(a.table + (int64_t)x.r * a.width + pos / a.page) : -1;
        };
        WeighWalk ahead = w;   // two tiles ahead: a look into the table takes as long as a tile
        int pages[2];
        pages[0] = look(ahead);
        if (ahead.left > 0) ahead.next(a);
        pages[1] = look(ahead);
        for (; w.left > 0; w.next(a), ++j) {
            const int pos = w.t * kTile + lane * box;
            int page = pages[0];
            if (ahead.left > 0) ahead.next(a);
            pages[0] = pages[1];
            pages[1] = look(ahead);
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
        const uint32_t idesc = __shfl_sync(0xffffffffu, instr_desc_bf16(kTile, (rows + 31) / 32 * 32, false), 0);
        const uint32_t q_addr = smem_u32(q_tile), ring_addr = smem_u32(ring);
        uint32_t j = 0, items = 0;
        bool ok = true;
        for (; w.left > 0; w.next(a), ++j) {
            const uint32_t stage = j % kWeighRing, g = j & 1u;
            ok = (!w.fresh || warp_wait(&sh.q_full, items & 1u)) && warp_wait2(&sh.k_full[stage], (j / kWeighRing) & 1u, &sh.s_empty[g], ((j >> 1) & 1u) ^ 1u);
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
        // Two groups, g, for tiles in turns, of two halves, h, of the rows.
        const int g = (warp - 2) >> 3, h = ((warp - 2) >> 2) & 1, quarter = warp & 3, t = tid - 64, at = quarter * 32 + lane;
        const int first_row = h * ((rows + 63) / 64 * 32), some = h ? rows - first_row : min(rows, (rows + 63) / 64 * 32);   // this half; may be none of 32 rows or fewer
        const float4* my_shift = sh.shift + first_row / 4;
        const uint32_t col = tmem + ((uint32_t)(quarter * 32) << 16) + g * kWeighRows + first_row;
        const uint64_t scale2 = pair_f32(a.scale_log2, a.scale_log2);
        const unsigned long long every = a.nodes < 64 ? ~0ull << a.nodes : 0ull;   // nodes that there are not
        uint32_t j = 0, alls = 0;
        int items = 0;
        bool ok = true;
        auto all_sync = [&]() {
            warp_arrive(&sh.all);
            ok = ok && warp_wait(&sh.all, alls++ & 1u);
        };
        // A tile's sum waits for its second half until the group's next one.
        float* due_to = nullptr;
        float due_sum = 0.f;
        int due = -1;   // the tile
        auto put = [&]() {
            if (due < 0) return;
            ok = warp_wait(&sh.half[due & 3], (due >> 2) & 1);
            if (ok && due_to) *due_to = due_sum + sh.sum[due & 3][at];
        };
        for (; ok && w.left > 0; w.next(a), ++j) {
            if (w.fresh) {   // all tiles of the head before have been summed, and their products read the rows that change now
                all_sync();
                if (!ok) break;
                ++items;
                const int c = t & 15, padded = (rows + 31) / 32 * 32;
                constexpr int kStep = 8 * kWeighGroups, kLoads = 4;   // rows of a step: 16 threads each
#pragma unroll 1
                for (int r0 = t >> 4; r0 < padded; r0 += kStep * kLoads) {   // rows behind the last one repeat it
                    uint4 v[kLoads];
#pragma unroll
                    for (int u = 0; u < kLoads; ++u) {
                        const int rr = r0 + kStep * u;
                        if (rr < padded) v[u] = __ldcg(reinterpret_cast<const uint4*>(a.q + a.row_at(w.r, w.kvh, min(row0 + rr, m_rows - 1))) + c);
                    }
#pragma unroll
                    for (int u = 0; u < kLoads; ++u) {
                        const int rr = r0 + kStep * u;
                        if (rr < padded) *reinterpret_cast<uint4*>(q_tile + (c >> 3) * kQHalf + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[u];
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&sh.q_full);
                if (t < kWeighRows) {   // rows behind the last one count for nothing, nor do those that see nothing
                    const float2 ml = __ldcg(a.row_ml + ((int64_t)w.r * a.kv_heads + w.kvh) * m_rows + min(row0 + t, row0 + rows - 1));
                    const float shift = t < rows ? log2f(ml.y) - ml.x : -INFINITY;
                    reinterpret_cast<float*>(sh.shift)[t] = shift;
                    if (t < rows && !(fabsf(shift) < INFINITY)) sh.bad = items;   // NaN too
                }
                {   // a lane has two nodes' masks, a warp makes the bits of four nodes
                    const unsigned long long* masks = a.masks + (int64_t)w.r * a.nodes;
                    const unsigned long long lo = lane < a.nodes ? __ldcg(masks + lane) : 0ull, hi = lane + 32 < a.nodes ? __ldcg(masks + lane + 32) : 0ull;
#pragma unroll
                    for (int u = 0; u < kTreeNodes / (4 * kWeighGroups); ++u) {
                        const int node = (warp - 2) * (kTreeNodes / (4 * kWeighGroups)) + u;
                        const unsigned x = __ballot_sync(0xffffffffu, (lo >> node) & 1ull), y = __ballot_sync(0xffffffffu, (hi >> node) & 1ull);
                        if (lane == 0) sh.seen_by[node] = (unsigned long long)y << 32 | x;
                    }
                }
                all_sync();
                if (!ok) break;
            }
            if ((int)(j & 1u) != g) continue;
            const int pos = w.t * kTile + at, node = pos - w.seq.len;
            float* to = a.weights + ((int64_t)w.r * a.kv_heads + w.kvh) * a.width * a.page + pos;
            const bool adds = node < 0 || row0 > 0;   // to what is there
            const float before = h == 0 && adds && pos < w.seq.end ? *to : 0.f;
            ok = warp_wait(&sh.s_full[g], (j >> 1) & 1u);
            if (!ok) break;
            tc_fence_after_sync();
            const unsigned good = sh.good[j & 7];
            const bool page = (good >> (at >> 4)) & 1u;
            float sum = 0.f;   // columns behind the last row are products with it too
            // What comes of a position behind the end or without a page is not used.
            const unsigned long long seen = node < 0 || node >= a.nodes ? ~0ull : sh.seen_by[node] | every;
            if (__all_sync(0xffffffffu, seen == ~0ull) && sh.bad != items) {   // every row sees all 32 positions
                uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll 1
                for (int c = 0; c < some; c += 32) {
                    uint32_t s[32];
                    tmem_ld32(col + c, s);
                    tmem_wait_ld(s);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float4 m = my_shift[c / 4 + e];
                        const float2 x = split_f32(fma_f32x2(pair_f32(__uint_as_float(s[4 * e]), __uint_as_float(s[4 * e + 1])), scale2, pair_f32(m.x, m.y)));
                        const float2 y = split_f32(fma_f32x2(pair_f32(__uint_as_float(s[4 * e + 2]), __uint_as_float(s[4 * e + 3])), scale2, pair_f32(m.z, m.w)));
                        sum2[0] = add_f32x2(sum2[0], pair_f32(exp2_approx(x.x), exp2_approx(x.y)));
                        sum2[1] = add_f32x2(sum2[1], pair_f32(exp2_approx(y.x), exp2_approx(y.y)));
                    }
                }
                const float2 two = split_f32(add_f32x2(sum2[0], sum2[1]));
                sum = two.x + two.y;
            } else {
                sum = sh.bad == items ? weigh_some<true>(a, my_shift, col, row0 + first_row, some, seen) : weigh_some<false>(a, my_shift, col, row0 + first_row, some, seen);
            }
            if (!page) sum = 0.f;
            tc_fence_before_sync();
            if (h) {   // the sum of four tiles before was read before this product was issued
                sh.sum[j & 3][at] = sum;
                warp_arrive(&sh.half[j & 3]);
            } else {
                put();
                if (!ok) break;
            }
            warp_arrive(&sh.s_empty[g]);
            if (h == 0) {
                due_to = pos < w.seq.end && (page || !adds) ? to : nullptr;
                due_sum = before + sum;
                due = (int)j;
            }
        }
        if (ok && h == 0) put();
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

void launch_tree_weigh(const mfqb_cache& c, const TreeArgs& a, cudaStream_t s) {
    const int m_rows = a.nodes * a.group;
    const int64_t cap = (int64_t)c.width * c.page, items = (int64_t)c.rows * c.kv_heads;
    int device = 0;
    MFQB_CUDA(cudaGetDevice(&device));
    static std::once_flag once[64];
    std::call_once(once[device], [] { MFQB_CUDA(cudaFuncSetAttribute(tree_weigh_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kWeighSmem)); });
    const CUtensorMap kmap = page_map(a.k, c);
    const unsigned ctas = (unsigned)std::min<int64_t>(kTreeSms, items * ((cap + kTile - 1) / kTile));
    for (int row0 = 0; row0 < m_rows; row0 += kWeighRows)
        launch_chained(tree_weigh_kernel, dim3(ctas), dim3(kWeighThreads), kWeighSmem, s, a, kmap, row0, std::min(kWeighRows, m_rows - row0));
}

}  // namespace mfqb
