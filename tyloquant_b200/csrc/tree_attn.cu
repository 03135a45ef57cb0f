// Attention of a tree of drafted tokens over a paged key/value cache.
//
// Per sequence and kv head the queries of all nodes and of the heads that share the kv head are the rows of one matrix Q (row
// node * G + head): S = Q K^T, P = exp2(scale' S - m), O = P V over tiles of 128 positions, with a running maximum m and sum l per row.
// The work is cut into units (sequence, kv head, tile of 128 rows, tile of 128 positions), which are shared out evenly and in
// order over the CTAs, which fill the SMs, from the lengths as they are on the device: a batch of very different lengths loads
// the SMs alike, and a captured call follows the lengths of each replay.  A stretch of units of one (sequence, head, row tile) that
// covers all its positions is written as it is; otherwise the CTA leaves O, m and l, and tree_merge_kernel adds the parts in the order of
// the context (no atomics: a call repeats bit for bit).
//
// Roles in a CTA: one warp asks for pages (bulk tensor copies into a ring of 32 KB tiles, keys and values in the order of their use, with
// the 128-byte swizzle), one issues tcgen05.mma, four (or eight) do the softmax, a row a thread: S comes out of tensor memory, P goes back
// into it as the A operand of the second product, O stays there.  O is multiplied by a correction only when a row's maximum has
// grown by more than 2^8 (P then stays below 2^8, which bf16 holds as exactly as values below 1).
#include <cuda.h>
#include <cuda_bf16.h>

#include <mutex>

#include "paged.h"
#include "tc05.cuh"

namespace mfqb {

constexpr int kTreeSms = 148;
constexpr int kTile = 128;                           // rows of Q, positions of a tile
constexpr int kTileBytes = kTile * kHeadDim * 2, kHalfBytes = kTileBytes / 2;
constexpr int tree_ctas(int ns) { return ns == 2 ? kTreeSms : 2 * kTreeSms; }
constexpr int tree_ring(int ns) { return ns == 2 ? 5 : 2; }   // tiles
constexpr int tree_threads(int ns) { return 64 + 128 * ns; }
constexpr int kTreeWhole = 256;                       // positions
constexpr int kTreeStart = 2;                         // what starting and ending a stretch takes, in tiles

struct TreeArgs {
    const int* table;
    const int* lens;
    const __nv_bfloat16* q;
    const unsigned long long* masks;
    const __nv_bfloat16 *k, *v;   // of the layer
    __nv_bfloat16* out;
    float* part;                  // [CTA][first, last][rows of a tile][128], then their (maximum, sum)
    float2* part_ml;
    int64_t* before;              // [rows + 1]: units of one item of each sequence before a sequence; the units of a CTA
    int* error;
    int rows, width, pages, page, kv_heads, hq, group, nodes, row_tiles, tile_rows;   // row_tiles: of 128 rows a stream; tile_rows: rows of a part, at most that
    bool whole;                   // an item is one unit
    unsigned group_inv;           // ceil(65536 / group): row / group = row * group_inv >> 16 for rows below 1024, groups up to 16
    float scale_log2;
    __device__ __forceinline__ int node_of(int row_of_q) const { return (int)((unsigned)row_of_q * group_inv >> 16); }
    // element offset of a row of Q (or of the output) of sequence r and kv head kvh
    __device__ __forceinline__ int64_t row_at(int r, int kvh, int row_of_q) const {
        const int node = node_of(row_of_q);
        return (((int64_t)r * nodes + node) * hq + kvh * group + row_of_q - node * group) * kHeadDim;
    }
};

// a / b of numbers that are not negative; mostly they fit 32 bits, and a 64-bit division is some hundred instructions.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((unsigned)a / (unsigned)b) : a / b;
}

// Tiles of sequence r (at least one: a sequence has a node), its length and end.
struct TreeSeq {
    int len, end, tiles;
    int units;   // of an item: its tiles and its start, or 1 where items are not split (TreeArgs::whole)
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int r) {
    const int cap = a.width * a.page;   // at most 2^30
    TreeSeq s;
    s.len = min(max(__ldcg(a.lens + r), 0), cap);
    s.end = min(s.len + a.nodes, cap);
    s.tiles = (s.end + kTile - 1) / kTile;
    s.units = a.whole ? 1 : s.tiles + kTreeStart;
    return s;
}
struct TreeShared {
    uint64_t kv_full[5], kv_empty[5], q_full, s_full[2], p_full[2], o_done[2], drain, all, group[2];
    unsigned long long bad_nodes;   // nodes of the stretch whose values hold an infinity or NaN
    int64_t scan[10];
    int64_t first, last, item_off;  // the CTA's units; offset of its first one in its sequence's
    int row0;
    uint32_t tmem;
    unsigned good[8];               // per tile (index mod 8): bit g = the 16 positions of group g have a page
    int failed;
    float2 ml[2][kTile];            // the streams' (maximum in powers of two, sum)
};

constexpr size_t tree_smem(int ns) { return (size_t)(tree_ring(ns) + ns) * kTileBytes + sizeof(TreeShared); }   // ring, Q of every stream
static_assert(tree_smem(2) <= 227 * 1024 && 2 * (tree_smem(1) + 1024) <= 228 * 1024, "shared memory of an SM");

// A CTA's stretches in order: sequence, item (kv head, row tile), tiles [t0, t1) of seq.tiles.
struct TreeWalk {
    int r, item, t0, t1;
    int64_t left;   // units from the stretch on; units kTreeStart .. of an item are its tiles
    TreeSeq seq;
    __device__ __forceinline__ void start(const TreeArgs& a, const TreeShared& sh) {
        r = sh.row0;
        left = sh.last - sh.first;
        if (left > 0) {
            seq = tree_seq(a, r);
            item = (int)quotient(sh.item_off, seq.units);
            const int u0 = (int)(sh.item_off - (int64_t)item * seq.units);
            left += u0;   // as if the item's start were the CTA's too
            stretch(a, max(u0 - kTreeStart, 0));
        }
    }
    __device__ __forceinline__ void next(const TreeArgs& a) {
        left -= seq.units;
        if (left <= (a.whole ? 0 : kTreeStart)) {
            left = 0;
            return;
        }
        if (++item == a.kv_heads * a.row_tiles) {
            item = 0;
            seq = tree_seq(a, ++r);
        }
        stretch(a, 0);
    }

private:
    __device__ __forceinline__ void stretch(const TreeArgs& a, int first) {
        t0 = first;
        t1 = a.whole ? seq.tiles : (int)min((int64_t)seq.tiles, left - kTreeStart);
        if (t1 <= t0) left = 0;   // nothing but units of the start
    }
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}
// D (+)= A B^T, both operands in shared memory.
__device__ __forceinline__ void tc_mma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// bf16 x bf16 -> f32; B with its K index running over rows of 128 bytes (values: position by position) where mn is set.
constexpr uint32_t instr_desc_bf16(int m, int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Descriptor of a [positions][64 dims] half in 128-byte rows taken as B operand with the dims as its rows: eight positions 1024
// bytes apart, the next 64 dims one half further.
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(kHalfBytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
#define MFQB_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define MFQB_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
// 32 lanes x 32 columns, a lane's columns in its registers; the load's values may be used after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : MFQB_R8(r, 0), MFQB_R8(r, 8), MFQB_R8(r, 16), MFQB_R8(r, 24)
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : MFQB_R8(r, 0), MFQB_R8(r, 8)
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::MFQB_W8(r, 0), MFQB_W8(r, 8), MFQB_W8(r, 16), MFQB_W8(r, 24), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::MFQB_W8(r, 0), MFQB_W8(r, 8), "r"(taddr)
                 : "memory");
}
#define MFQB_P8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
// Waits for this thread's loads.  The 32 registers of a load pass through it, so that no use of them can be moved before the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    asm volatile("" : MFQB_P8(r, 0), MFQB_P8(r, 8));
    asm volatile("" : MFQB_P8(r, 16), MFQB_P8(r, 24));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    asm volatile("" : MFQB_P8(r, 0), MFQB_P8(r, 8));
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r, uint32_t* q) {
    tmem_wait_ld(r);
    asm volatile("" : MFQB_P8(q, 0), MFQB_P8(q, 8));
    asm volatile("" : MFQB_P8(q, 16), MFQB_P8(q, 24));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {   // one arrival for what all lanes have done
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
// Both of two barriers; the polls of barriers that are complete (the usual case of one of them) overlap.
__device__ __forceinline__ bool warp_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
    const bool da = mbar_test(a, pa), db = mbar_test(b, pb);
    if (__all_sync(0xffffffffu, da && db)) return true;
    return warp_wait(a, pa) && warp_wait(b, pb);
}

// exp2(scale s + mc) of 16 scores, rounded to bf16 into p; their sums are added to l, their maxima to top where TOP.
// The one rounding of the probabilities: the tensor core takes them in the values' type, and a second bf16 term would be the second product
// again and half of S's columns.  Against 64 bits the output is off by 0.0019 to 0.0023 of its size, where rounding it alone makes 0.0017.
template <bool TOP>
__device__ __forceinline__ void exp16(const uint32_t* s, uint64_t scale, uint64_t mc, uint64_t (&l)[2], float (&top)[2], uint32_t* p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = __uint_as_float(s[2 * e]), b = __uint_as_float(s[2 * e + 1]);
        if (TOP) top[e & 1] = fmaxf(fmaxf(top[e & 1], a), b);
        const float2 x = split_f32(fma_f32x2(pair_f32(a, b), scale, mc));
        const float u = exp2_approx(x.x), v = exp2_approx(x.y);
        l[e & 1] = add_f32x2(l[e & 1], pair_f32(u, v));
        p[e] = pack_bf16(u, v);
    }
}

// Values of a tile that is not whole, in shared memory: rows that no row of Q sees (behind the end up to the next 16, without a page)
// are cleared; an infinity or NaN of a node becomes 0 and the node is noted (add_bad_nodes).  The four warps of a stream; a row of 256
// bytes is two halves of 128.  Two streams may do the same tile at once: they write the same.
__device__ __noinline__ void clean_values(TreeShared& sh, unsigned char* tile, TreeSeq seq, int pos0, unsigned good, int quarter, int lane) {
    const int end = min(kTile, seq.end - pos0), first = max(0, seq.len - pos0);   // nodes are rows first .. end - 1
    unsigned char* piece = tile + ((lane >> 3) & 1) * kHalfBytes + (lane & 7) * 16;
    const int r0 = 2 * quarter + (lane >> 4);
    if (good != 0xFFu || (end & 15))
        for (int r = r0 + (good == 0xFFu ? end & ~15 : 0); r < ((end + 15) & ~15); r += 8)
            if (r >= end || !((good >> (r >> 4)) & 1u)) *reinterpret_cast<uint4*>(piece + r * 128) = make_uint4(0u, 0u, 0u, 0u);
    for (int r = first + r0; r < end; r += 8) {
        if (!((good >> (r >> 4)) & 1u)) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(piece + r * 128);
        uint32_t y[4] = {v.x, v.y, v.z, v.w};
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool lo = (y[e] & 0x7F80u) == 0x7F80u, hi = (y[e] & 0x7F800000u) == 0x7F800000u;
            bad |= lo | hi;
            y[e] &= (lo ? 0xFFFF0000u : 0xFFFFFFFFu) & (hi ? 0x0000FFFFu : 0xFFFFFFFFu);
        }
        if (bad) {
            *reinterpret_cast<uint4*>(piece + r * 128) = make_uint4(y[0], y[1], y[2], y[3]);
            atomicOr(&sh.bad_nodes, 1ull << (pos0 + r - seq.len));
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// Rare: values of visible nodes that hold an infinity or NaN were taken out of the product (0 in their place, so that rows which do not see
// the node keep clear of them); here they are added to the row's result, where the row sees them.
template <typename T>
__device__ __noinline__ void add_bad_nodes(const TreeArgs& a, unsigned long long bad, const TreeSeq& seq, int r, int kvh, int row, float mc, T* dst) {
    const __nv_bfloat16* q = a.q + a.row_at(r, kvh, row);
    bad &= a.masks[(int64_t)r * a.nodes + a.node_of(row)];
    for (; bad; bad &= bad - 1) {
        const int t = seq.len + (__ffsll((long long)bad) - 1);
        const int page = a.table[(int64_t)r * a.width + t / a.page];
        const int64_t at = (((int64_t)page * a.kv_heads + kvh) * a.page + (t & (a.page - 1))) * kHeadDim;
        float s = 0.f;
        for (int d = 0; d < kHeadDim; ++d) s += __bfloat162float(q[d]) * __bfloat162float(a.k[at + d]);
        const float p = exp2_approx(s * a.scale_log2 - mc);
        for (int d = 0; d < kHeadDim; ++d) {
            const float v = __bfloat162float(a.v[at + d]);
            if (!isfinite(v)) dst[d] = (T)((float)dst[d] + (p > 0.f ? v : NAN));
        }
    }
}

// NS = 1 (up to 128 rows): a CTA has one tile of rows, and two CTAs share an SM: while one's scores become probabilities the other's
// products run, and starts and ends of stretches overlap too (27 nodes of 13 sequences of up to 7000 tokens: 35 us with one CTA whose
// two halves took alternate tiles of a stretch).  NS = 2: the CTA has the SM and two streams of 128 rows each, which take every
// tile in turns, so that it is read once for 256 rows.  S of a step waits for the stream's last product, whose P lies in its place.
// One warp issues for both streams: with a warp each they fall into step, and the tensor core waits while both do softmax.
// REP: up to 32 (64) rows stand in Q four times (twice), and a copy's warps take a quarter (a half) of every tile's positions: their
// P is zero elsewhere.  A row's 128 exponentials in one thread are what a tile waits for otherwise.
template <int NS, int REP>
__global__ void __launch_bounds__(tree_threads(NS), NS == 2 ? 1 : 2) tree_attn_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap kmap,
                                                                                     const __grid_constant__ CUtensorMap vmap) {
    constexpr int kRing = tree_ring(NS);
    constexpr uint32_t kColumns = 256 * NS, kColS = 0, kColO = kTile * NS;   // tensor memory: S of the streams (P takes the place of its first half), their O
    extern __shared__ __align__(1024) unsigned char ring[];   // the swizzle's pattern repeats every 1024 bytes
    TreeShared& sh = *reinterpret_cast<TreeShared*>(ring + (size_t)(kRing + NS) * kTileBytes);
    unsigned char* q_tiles = ring + (size_t)kRing * kTileBytes;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (smem_u32(ring) & 1023u) {   // not the case with no static shared memory
        if (tid == 0) atomicExch(a.error, MFQB_ERR_CUDA);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) { mbar_init(&sh.kv_full[i], 1); mbar_init(&sh.kv_empty[i], 1); }
        for (int i = 0; i < NS; ++i) { mbar_init(&sh.group[i], 4); mbar_init(&sh.s_full[i], 1); mbar_init(&sh.p_full[i], 4); mbar_init(&sh.o_done[i], 1); }
        mbar_init(&sh.q_full, 4 * NS);
        mbar_init(&sh.all, 4 * NS);
        mbar_init(&sh.drain, 1);
        sh.bad_nodes = 0;
        sh.failed = 0;
        sh.first = sh.last = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(&sh.tmem, kColumns);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    chained_wait();
    {   // this CTA's units: thread t holds the sequences kEach * t ..
        constexpr int kEach = (kCacheRows + tree_threads(NS) - 1) / tree_threads(NS);
        int units_of[kEach];
        int64_t mine = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            units_of[j] = kEach * tid + j < a.rows ? tree_seq(a, kEach * tid + j).units : 0;
            mine += units_of[j];
        }
        int64_t upto = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) sh.scan[warp] = upto;
        __syncthreads();
        int64_t total = 0;
#pragma unroll
        for (int w = 0; w < tree_threads(NS) / 32; ++w) {
            if (w < warp) upto += sh.scan[w];
            total += sh.scan[w];
        }
        const int64_t items = (int64_t)a.kv_heads * a.row_tiles, units = total * items, quota = quotient(units + gridDim.x - 1, gridDim.x);
        const int64_t first = (int64_t)blockIdx.x * quota, last = min(units, first + quota);
        int64_t begin = (upto - mine) * items;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (blockIdx.x == 0 && kEach * tid + j < a.rows) a.before[kEach * tid + j] = quotient(begin, items);   // for tree_merge_kernel
            const int64_t end = begin + units_of[j] * items;
            if (first < last && begin <= first && first < end) {
                sh.row0 = kEach * tid + j;
                sh.item_off = first - begin;
                sh.first = first;
                sh.last = last;
            }
            begin = end;
        }
        if (blockIdx.x == 0 && tid == 0) a.before[a.rows] = quota;
        __syncthreads();
    }
    TreeWalk w;
    w.start(a, sh);
    if (warp == 0) {
        // -------- pages: lane b asks for box b of a tile (a page, or 128 positions of one), both halves --------
        const int box = min(a.page, kTile), boxes = kTile / box;
        uint32_t issued = 0, tile_no = 0;
        bool ok = true;
        auto ask = [&](const CUtensorMap* map, int kvh, int pos, int page) {
            const uint32_t stage = issued % kRing;
            ok = warp_wait(&sh.kv_empty[stage], ((issued / kRing) & 1u) ^ 1u);
            if (!ok) return;
            unsigned char* dst = ring + (size_t)stage * kTileBytes + lane * box * 128;
            const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) mbar_arrive_expect_tx(&sh.kv_full[stage], (uint32_t)__popc(have) * (uint32_t)box * 256u);
            __syncwarp();
            if (page >= 0) {
                const int y = pos & (a.page - 1);
                tma_load_4d(dst, map, 0, y, kvh, page, &sh.kv_full[stage]);
                tma_load_4d(dst + kHalfBytes, map, 64, y, kvh, page, &sh.kv_full[stage]);
            }
            __syncwarp();
            ++issued;
        };
        auto position = [&](int i) { return (w.t0 + i) * kTile + lane * box; };   // of this lane's box
        for (; ok && w.left > 0; w.next(a)) {
            const int kvh = w.item / a.row_tiles, n = w.t1 - w.t0;
            for (int i = 0; ok && i < n; ++i) {
                const int pos = position(i);
                int page = -1;
                if (lane < boxes && pos < w.seq.end) page = __ldcg(a.table + (int64_t)w.r * a.width + pos / a.page);
                if ((unsigned)page >= (unsigned)a.pages) page = -1;
                unsigned good = 0;   // groups of 16 positions with a page: box b covers groups b * box / 16 ..
                const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
                for (int g = 0; g < 8; ++g) good |= ((have >> (g * 16 / box)) & 1u) << g;
                if (lane == 0) sh.good[tile_no & 7] = good;
                ++tile_no;
                ask(&kmap, kvh, pos, page);
                if (ok) ask(&vmap, kvh, pos, page);
            }
        }
        if (!ok) sh.failed = 1;
        for (uint32_t i = 1; i <= min(issued, (uint32_t)kRing); ++i)   // no copy outlives the CTA, whatever became of the other roles
            if (!warp_wait(&sh.kv_full[(issued - i) % kRing], ((issued - i) / kRing) & 1u)) sh.failed = 1;
    } else if (warp == 1) {
        // -------- products: the warp stays together, an elected lane issues --------
        constexpr uint32_t idesc_s = instr_desc_bf16(kTile, kTile, false), idesc_o = instr_desc_bf16(kTile, kHeadDim, true);
        const uint32_t q_addr = smem_u32(q_tiles), ring_addr = smem_u32(ring);
        uint32_t base = 0, stretch = 0, steps = 0;   // ring position of the stretch, its number, tiles before it
        bool ok = true;
        // What the products' operands are made of is made warp-uniform by the shuffles: an instruction takes some 60 clocks then, its time on the
        // tensor core, and 120 otherwise.
        auto scores = [&](int u) {
            const int i = u / NS, st = u % NS;
            const uint32_t at = base + 2 * i, stage = at % kRing;
            ok = warp_wait(&sh.kv_full[stage], (at / kRing) & 1u) && (u < NS || warp_wait(&sh.o_done[st], (steps + i - 1) & 1u));
            if (!ok) return;
            tc_fence_after_sync();
            const uint32_t k_addr = __shfl_sync(0xffffffffu, ring_addr + stage * kTileBytes, 0), q = __shfl_sync(0xffffffffu, q_addr + st * kTileBytes, 0);
            const uint32_t d = __shfl_sync(0xffffffffu, tmem + kColS + st * kTile, 0);
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    tc_mma_f16_ss(d, smem_desc_sw128(q + (s >> 2) * kHalfBytes + (s & 3) * 32), smem_desc_sw128(k_addr + (s >> 2) * kHalfBytes + (s & 3) * 32), idesc_s, s > 0);
                tc_commit(&sh.s_full[st]);
                if (st == NS - 1) tc_commit(&sh.kv_empty[stage]);
            }
            __syncwarp();
        };
        auto values = [&](int u) {
            const int i = u / NS, st = u % NS;
            const uint32_t at = base + 2 * i + 1, stage = at % kRing;
            ok = warp_wait2(&sh.kv_full[stage], (at / kRing) & 1u, &sh.p_full[st], (steps + i) & 1u);
            if (!ok) return;
            tc_fence_after_sync();
            const uint32_t v_addr = __shfl_sync(0xffffffffu, ring_addr + stage * kTileBytes, 0), p = __shfl_sync(0xffffffffu, tmem + kColS + st * kTile, 0);
            const uint32_t d = __shfl_sync(0xffffffffu, tmem + kColO + st * kHeadDim, 0);
            const bool more = __shfl_sync(0xffffffffu, i > 0, 0);   // there is an O to add to
            const int groups = __shfl_sync(0xffffffffu, min(8, (w.seq.end - (w.t0 + i) * kTile + 15) >> 4), 0);   // of 16 positions; nothing is behind the end
            if (elect_one()) {
                if (groups == 8) {
#pragma unroll
                    for (int s = 0; s < 8; ++s) tc_mma_f16_ts(d, p + s * 8, smem_desc_sw128_mn(v_addr + s * 2048), idesc_o, s > 0 || more);
                } else {
#pragma unroll 1
                    for (int s = 0; s < groups; ++s) tc_mma_f16_ts(d, p + s * 8, smem_desc_sw128_mn(v_addr + s * 2048), idesc_o, s > 0 || more);
                }
                tc_commit(&sh.o_done[st]);
                if (st == NS - 1) tc_commit(&sh.kv_empty[stage]);
            }
            __syncwarp();
        };
        for (; ok && w.left > 0; w.next(a)) {
            const int n = w.t1 - w.t0;
            ok = warp_wait(&sh.q_full, stretch & 1u);
            for (int u = 0; ok && u < NS; ++u) scores(u);
            for (int u = 0; ok && u < NS * n; ++u) {
                values(u);
                if (ok && u + NS < NS * n) scores(u + NS);
            }
            base += 2 * n;
            steps += n;
            ++stretch;
        }
        if (elect_one()) tc_commit(&sh.drain);   // what was issued still reads the ring and the tensor memory
        __syncwarp();
        if (!warp_wait(&sh.drain, 0) || !ok) sh.failed = 1;
    } else {
        // -------- softmax: stream = warps 2-5 or 6-9, thread = lane of tensor memory: row lane_l % kSpan of the tile, copy lane_l / kSpan --------
        constexpr int kSpan = kTile / REP, kCols = kTile / REP;   // rows, a copy's positions of a tile
        const int st = (warp - 2) >> 2, quarter = warp & 3, lane_l = quarter * 32 + lane, row_l = lane_l % kSpan, copy = lane_l / kSpan;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), col_s = lanes + kColS + st * kTile, col_o = lanes + kColO + st * kHeadDim;
        unsigned char* q_tile = q_tiles + st * kTileBytes;
        uint32_t base = 0, alls = 0, groups = 0, steps = 0;   // steps: tiles before the stretch
        bool ok = true;
        int stretch = 0;
        auto all_sync = [&]() {   // all softmax warps, with a bound like every other wait
            warp_arrive(&sh.all);
            ok = ok && warp_wait(&sh.all, alls++ & 1u);
        };
        auto group_sync = [&]() {   // the stream's four
            warp_arrive(&sh.group[st]);
            ok = ok && warp_wait(&sh.group[st], groups++ & 1u);
        };
        const uint64_t scale2 = pair_f32(a.scale_log2, a.scale_log2);
        const int m_rows = a.nodes * a.group;   // rows of Q in all
        for (; ok && w.left > 0; w.next(a), ++stretch) {
            const int kvh = w.item / a.row_tiles, rt = w.item % a.row_tiles, n = w.t1 - w.t0;
            const int tile0 = (rt * NS + st) * kTile, row = tile0 + row_l;   // the stream's first row, this thread's
            const bool live = row < m_rows, busy = tile0 + (quarter * 32) % kSpan < m_rows;   // busy: some row of the warp is one
            // Q, 16 threads a row of 256 bytes, all loads at once; the products that read the last stretch's are done (its S has been
            // read).  Rows behind the last one repeat it.
            {
                constexpr int kStep = 8, kLoads = kTile / kStep;
                const int c = lane_l & 15, r0 = lane_l >> 4;
                uint4 v[kLoads / REP];
#pragma unroll
                for (int j = 0; j < kLoads / REP; ++j) {
                    v[j] = __ldcg(reinterpret_cast<const uint4*>(a.q + a.row_at(w.r, kvh, min(tile0 + r0 + kStep * j, m_rows - 1))) + c);
                }
#pragma unroll
                for (int j = 0; j < kLoads; ++j) {
                    const int rr = r0 + kStep * j;
                    *reinterpret_cast<uint4*>(q_tile + (c >> 3) * kHalfBytes + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[j % (kLoads / REP)];
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&sh.q_full);
            unsigned long long mask = live ? __ldcg(a.masks + (int64_t)w.r * a.nodes + a.node_of(row)) : 0ull;
            if (a.nodes < 64) mask &= (1ull << a.nodes) - 1ull;
            float m = -INFINITY;   // maximum of the scores so far (or less, see above)
            uint64_t l2[2] = {0ull, 0ull};   // the sum, in four parts
            bool seen = false;
            for (int i = 0; i < n; ++i) {
                ok = warp_wait(&sh.s_full[st], (steps + i) & 1u);
                if (!ok) break;
                tc_fence_after_sync();
                const unsigned good = sh.good[(steps + i) & 7];
                const int pos0 = (w.t0 + i) * kTile;
                const bool whole = pos0 + kTile <= w.seq.len && good == 0xFFu;   // every row sees all of the tile
                float known = -INFINITY;   // maximum of this thread's scores of a tile that is not whole
                if (!whole) {
                    const uint32_t at = base + 2 * i + 1, stage = at % kRing;
                    ok = warp_wait(&sh.kv_full[stage], (at / kRing) & 1u);
                    if (!ok) break;
                    clean_values(sh, ring + (size_t)stage * kTileBytes, w.seq, pos0, good, quarter, lane);
                    // what this row does not see of its copy's positions becomes minus infinity
#pragma unroll 1
                    for (int c = 0; c < kCols; c += 32) {
                        const int p0 = copy * kCols + c, ctx = w.seq.len - (pos0 + p0);   // positions from here on that are before the length
                        unsigned vis = ctx >= 32 ? 0xFFFFFFFFu : ctx <= 0 ? 0u : (1u << ctx) - 1u;
                        if (ctx <= 0 && ctx > -64) vis |= (unsigned)(mask >> -ctx);
                        else if (ctx > 0 && ctx < 32) vis |= (unsigned)(mask << ctx);
                        vis &= ((good >> (p0 >> 4)) & 1u ? 0x0000FFFFu : 0u) | ((good >> ((p0 >> 4) + 1)) & 1u ? 0xFFFF0000u : 0u);
                        seen |= vis != 0;
                        if (busy) {
                            uint32_t s[32];
                            tmem_ld32(col_s + p0, s);
                            tmem_wait_ld(s);
                            float t[2] = {known, known};
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if (!((vis >> e) & 1u)) s[e] = 0xFF800000u;
                                t[e & 1] = fmaxf(t[e & 1], __uint_as_float(s[e]));
                            }
                            known = fmaxf(t[0], t[1]);
                            if (__any_sync(0xffffffffu, vis != 0xFFFFFFFFu)) tmem_st32(col_s + p0, s);
                        }
                    }
                    tmem_wait_st();
                } else {
                    seen = true;
                }
                if (busy) {
                    auto rescale = [&](float high, bool raise) {   // l and O to a new maximum
                        const float corr = !raise ? 1.f : m == -INFINITY ? 0.f : exp2_approx((m - high) * a.scale_log2);
                        if (raise) m = high;
                        const uint64_t corr2 = pair_f32(corr, corr);
                        l2[0] = fma_f32x2(l2[0], corr2, 0ull);
                        l2[1] = fma_f32x2(l2[1], corr2, 0ull);
                        if (i > 0) {   // O holds the stream's steps before, all complete (this step's S was issued after them)
#pragma unroll 1
                            for (int c = 0; c < kHeadDim; c += 32) {
                                uint32_t o[32];
                                tmem_ld32(col_o + c, o);
                                tmem_wait_ld(o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st32(col_o + c, o);
                            }
                        }
                    };
                    auto too_high = [&](float high) { return live && high > -INFINITY && (m == -INFINITY || (high - m) * a.scale_log2 > 8.f); };
                    if constexpr (REP > 1) {
                        uint32_t s[kCols], p[kCols / 2];
#pragma unroll
                        for (int c = 0; c < kCols; c += 32) tmem_ld32(col_s + copy * kCols + c, s + c);
#pragma unroll
                        for (int c = 0; c < kCols; c += 32) tmem_wait_ld(s + c);
                        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int e = 0; e < kCols; e += 2) top[(e >> 1) & 3] = fmaxf(fmaxf(top[(e >> 1) & 3], __uint_as_float(s[e])), __uint_as_float(s[e + 1]));
                        const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                        const bool raise = too_high(high);
                        if (__any_sync(0xffffffffu, raise)) rescale(high, raise);
                        const float mc = m == -INFINITY ? 0.f : -m * a.scale_log2;
                        const uint64_t mc2 = pair_f32(mc, mc);
                        float unused[2] = {0.f, 0.f};
#pragma unroll
                        for (int c = 0; c < kCols; c += 16) exp16<false>(s + c, scale2, mc2, l2, unused, p + c / 2);
                        // P: this copy's positions, zero for the others'
                        uint32_t zero[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) zero[e] = 0u;
#pragma unroll
                        for (int k = 0; k < REP; ++k)
#pragma unroll
                            for (int c = 0; c < kCols / 2; c += 16) tmem_st16(col_s + k * (kCols / 2) + c, k == copy ? p + c : zero);
                    } else {
                        // The exponentials are formed with the maximum as it was, the tile's own is found beside them; only where it has grown
                        // too far they are formed again.  P waits in registers meanwhile, S in tensor memory.
                        uint32_t p[64];
                        if (!whole) {
                            const bool raise = too_high(known);
                            if (__any_sync(0xffffffffu, raise)) rescale(known, raise);
                        } else if (i == 0) {   // there is no maximum yet
                            float top = -INFINITY;
#pragma unroll 1
                            for (int c = 0; c < kTile; c += 32) {
                                uint32_t s[32];
                                tmem_ld32(col_s + c, s);
                                tmem_wait_ld(s);
                                float t[2] = {top, top};
#pragma unroll
                                for (int e = 0; e < 32; e += 2) t[(e >> 1) & 1] = fmaxf(fmaxf(t[(e >> 1) & 1], __uint_as_float(s[e])), __uint_as_float(s[e + 1]));
                                top = fmaxf(t[0], t[1]);
                            }
                            m = top;
                        }
                        for (;;) {
                            const float mc = m == -INFINITY ? 0.f : -m * a.scale_log2;
                            const uint64_t mc2 = pair_f32(mc, mc);
                            uint64_t sum[2] = {l2[0], l2[1]};
                            float top[2] = {-INFINITY, -INFINITY};
                            uint32_t s[2][16];
                            tmem_ld16_async(col_s, s[0]);
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                uint32_t* now = s[c & 1];
                                tmem_wait_ld16(now);
                                if (c < 7) tmem_ld16_async(col_s + 16 * (c + 1), s[(c + 1) & 1]);
                                exp16<true>(now, scale2, mc2, sum, top, p + 8 * c);
                            }
                            const float high = fmaxf(top[0], top[1]);
                            const bool raise = too_high(high);
                            if (!__any_sync(0xffffffffu, raise)) {
                                l2[0] = sum[0];
                                l2[1] = sum[1];
                                break;
                            }
                            rescale(high, raise);
                        }
                        tmem_st32(col_s, p);   // in the place of S, all of which has been read
                        tmem_st32(col_s + 32, p + 32);
                    }
                    tmem_wait_st();
                }
                tc_fence_before_sync();
                warp_arrive(&sh.p_full[st]);
            }
            if (!ok) break;
            const float2 la = split_f32(add_f32x2(l2[0], l2[1]));
            {
                // A part without a maximum counts for nothing beside others (its sum says what it is alone: NaN where every score is
                // minus infinity, 0 where nothing is seen); one with a NaN among its scores makes the row NaN in any company.
                float l = la.x + la.y;
                const float mc = m > -INFINITY ? m * a.scale_log2 : l != l ? 0.f : -INFINITY;
                if (mc == -INFINITY) l = seen ? NAN : 0.f;
                sh.ml[st][lane_l] = make_float2(mc, l);
            }
            base += 2 * n;
            steps += n;
            ok = warp_wait(&sh.o_done[st], (steps - 1) & 1u);
            all_sync();   // the copies' maxima and sums, every tile's bad nodes
            if (!ok) break;
            tc_fence_after_sync();
            const unsigned long long bad = sh.bad_nodes;
            const bool complete = n == w.seq.tiles;
            auto joint = [&](int rr) {   // maximum and sum over the copies of row rr
                float mc = -INFINITY, l = 0.f;
#pragma unroll
                for (int k = 0; k < REP; ++k) mc = fmaxf(mc, sh.ml[st][rr + k * kSpan].x);
#pragma unroll
                for (int k = 0; k < REP; ++k) {
                    const float2 x = sh.ml[st][rr + k * kSpan];
                    l += mc == -INFINITY ? x.y : x.x == -INFINITY ? 0.f : x.y * exp2_approx(x.x - mc);
                }
                return make_float2(mc, l);
            };
            const float2 sum = joint(row_l);
            // What this copy's values are multiplied by: its maximum against the joint one, the sum where the row is complete.
            const float x = sh.ml[st][lane_l].x, e = x == -INFINITY ? 0.f : exp2_approx(x - sum.x);
            const float f = !complete ? e : sum.y == 0.f ? 0.f : __fdividef(e, sum.y);
            const int64_t slot = ((int64_t)blockIdx.x * 2 + (stretch > 0)) * a.tile_rows + st * kTile;
            const int rows_here = min(kSpan, m_rows - tile0);   // may be 0 or less (NS = 2)
            auto take = [&](int c, uint32_t* o) {   // 32 columns of this thread's row; zero where it saw nothing (its O may be NaN then)
                tmem_ld32(col_o + c, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = f == 0.f ? 0u : __float_as_uint(__uint_as_float(o[k]) * f);
            };
            // Rows leave through the Q tile's place: a thread has a row of tensor memory, and a store instruction wants neighbouring columns (a row a
            // thread takes a line of the L1 cache per thread and instruction).
            if constexpr (REP == 1) {   // 8 KB a warp: its 32 rows, all columns in bf16 or half of them in float32
                unsigned char* stage = q_tile + quarter * 8192;
                auto place = [&](int rr, int c) { return reinterpret_cast<uint4*>(stage + rr * 256 + ((c ^ (rr & 7)) << 4)); };
                if (busy) {
#pragma unroll 1
                    for (int c = 0; c < kHeadDim; c += 32) {
                        uint32_t o[32];
                        take(c, o);
                        if (complete) {
#pragma unroll
                            for (int k = 0; k < 32; k += 8)
                                *place(lane, (c + k) >> 3) =
                                    make_uint4(pack_bf16(__uint_as_float(o[k]), __uint_as_float(o[k + 1])), pack_bf16(__uint_as_float(o[k + 2]), __uint_as_float(o[k + 3])),
                                               pack_bf16(__uint_as_float(o[k + 4]), __uint_as_float(o[k + 5])), pack_bf16(__uint_as_float(o[k + 6]), __uint_as_float(o[k + 7])));
                            if (c < 96) continue;
                        } else {
#pragma unroll
                            for (int k = 0; k < 32; k += 4) *place(lane, ((c & 32) + k) >> 2) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                            if (!(c & 32)) continue;
                        }
                        __syncwarp();
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            uint4 v[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] = *place(16 * half + 2 * k + (lane >> 4), lane & 15);   // two rows of 256 bytes at a time
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const int rr = quarter * 32 + 16 * half + 2 * k + (lane >> 4);
                                if (rr >= rows_here) continue;
                                if (complete) reinterpret_cast<uint4*>(a.out + a.row_at(w.r, kvh, tile0 + rr))[lane & 15] = v[k];
                                else reinterpret_cast<uint4*>(a.part + (slot + rr) * kHeadDim + (c & 64))[lane & 15] = v[k];
                            }
                        }
                        __syncwarp();
                    }
                }
            } else {   // 32 KB: the copies of a row are added; all columns at once, or half of them where there are more than 64 rows with the copies
                const int wide = rows_here * REP <= 64 ? 128 : 64, pieces = wide / 4, shift = wide == 128 ? 5 : 4;
                auto place = [&](int rr, int cp, int c) { return reinterpret_cast<float4*>(q_tile + ((cp * rows_here + rr) * pieces + (c ^ (rr & 7))) * 16); };
#pragma unroll 1
                for (int c0 = 0; c0 < kHeadDim; c0 += wide) {
                    if (c0) group_sync();   // the columns before have been read
                    if (!ok) break;
                    if (busy) {
#pragma unroll 1
                        for (int c = 0; c < wide; c += 64) {
                            uint32_t o[64];
                            tmem_ld32(col_o + c0 + c, o);
                            tmem_ld32(col_o + c0 + c + 32, o + 32);
                            tmem_wait_ld(o, o + 32);
                            if (live)
#pragma unroll
                                for (int k = 0; k < 64; k += 4)
                                    *place(row_l, copy, (c + k) >> 2) = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                                               : make_float4(__uint_as_float(o[k]) * f, __uint_as_float(o[k + 1]) * f,
                                                                                             __uint_as_float(o[k + 2]) * f, __uint_as_float(o[k + 3]) * f);
                            __syncwarp();
                        }
                    }
                    group_sync();
                    if (!ok) break;
                    for (int idx = lane_l; idx < rows_here << shift; idx += 128) {
                        const int rr = idx >> shift, c = idx & (pieces - 1);
                        float4 v = *place(rr, 0, c);
#pragma unroll
                        for (int k = 1; k < REP; ++k) {
                            const float4 u = *place(rr, k, c);
                            v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
                        }
                        if (complete) reinterpret_cast<uint2*>(a.out + a.row_at(w.r, kvh, tile0 + rr) + c0)[c] = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                        else reinterpret_cast<float4*>(a.part + (slot + rr) * kHeadDim + c0)[c] = v;
                    }
                }
                if (!ok) break;
                if (bad) group_sync();   // the rows' stores, before add_bad_nodes
                if (!ok) break;
            }
            if (live && copy == 0) {
                if (!complete) a.part_ml[slot + row_l] = sum;
                if (bad) {
                    if (complete) add_bad_nodes(a, bad, w.seq, w.r, kvh, row, sum.x, a.out + a.row_at(w.r, kvh, row));
                    else add_bad_nodes(a, bad, w.seq, w.r, kvh, row, sum.x, a.part + (slot + row_l) * kHeadDim);
                }
            }
            tc_fence_before_sync();
            all_sync();   // sums and bad nodes have been read
            if (tid == 64) sh.bad_nodes = 0;
        }
        if (!ok) sh.failed = 1;
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_free(tmem, kColumns);
        if (lane == 0 && sh.failed) atomicExch(a.error, MFQB_ERR_TIMEOUT);
    }
}

constexpr int kMergeParts = 16, kMergeWarps = 4;   // parts in flight for a row, rows of a CTA

// Rows whose positions were shared by several CTAs: a warp per output row adds the parts in the order of the context, with a running
// maximum.  Sixteen parts at a time are on their way, by asynchronous copies: with loads into registers eight were, and the ragged batch (rows of
// up to 28 parts) took 26.5 us in place of 25.
__global__ void __launch_bounds__(32 * kMergeWarps) tree_merge_kernel(const __grid_constant__ TreeArgs a, int streams, int rows) {
    chained_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warp = blockIdx.x * kMergeWarps + wid, m_rows = a.nodes * a.group, per_seq = a.kv_heads * m_rows;
    __shared__ float4 s_part[kMergeWarps][kMergeParts][32];
    __shared__ int64_t s_before[kMergeWarps], s_quota;   // what all rows ask for comes through one thread a CTA and sequence
    __shared__ TreeSeq s_seq[kMergeWarps];
    const int r0 = blockIdx.x * kMergeWarps / per_seq, r = min(warp, rows - 1) / per_seq;
    if (threadIdx.x < kMergeWarps && (int64_t)(r0 + threadIdx.x) * per_seq < min((int64_t)blockIdx.x * kMergeWarps + kMergeWarps, (int64_t)rows)) {
        s_before[threadIdx.x] = __ldcg(a.before + r0 + threadIdx.x);
        s_seq[threadIdx.x] = tree_seq(a, r0 + threadIdx.x);
    }
    if (threadIdx.x == 32) s_quota = __ldcg(a.before + a.rows);
    __syncthreads();
    if (warp >= rows) return;
    const int local = warp - r * per_seq, kvh = local / m_rows, row = local - kvh * m_rows;
    const int64_t before = s_before[r - r0], quota = s_quota;
    const TreeSeq seq = s_seq[r - r0];
    const int span = streams * kTile, rt = row / span, row_l = row - rt * span;
    const int64_t items = (int64_t)a.kv_heads * a.row_tiles;
    const int64_t s0 = before * items + (int64_t)(kvh * a.row_tiles + rt) * seq.units, c0 = quotient(s0 + kTreeStart, quota), c1 = quotient(s0 + seq.units - 1, quota);
    if (c0 == c1) return;
    // The item is its first CTA's second stretch unless it begins that CTA, and every later CTA's first.  At most 296 CTAs with two stretches of 256 rows.
    const int first = (int)c0, last = (int)c1, shift = s0 > c0 * quota ? 1 : 0;
    auto slot = [&](int c) { return (c * 2 + (c == first ? shift : 0)) * a.tile_rows + row_l; };
    float m = -INFINITY, l = 0.f, none = 0.f;   // none: of parts without a maximum, which count only among themselves
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = first; c <= last; c += kMergeParts) {
        const int n = min(kMergeParts, last - c + 1);
        for (int u = 0; u < n; ++u)   // a lane reads what it has copied itself
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&s_part[wid][u][lane])), "l"(a.part + (int64_t)slot(c + u) * kHeadDim + 4 * lane) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
        const float2 ml = lane < n ? __ldcg(&a.part_ml[slot(c + lane)]) : make_float2(-INFINITY, 0.f);
        float high = ml.x;
        for (int o = 16; o > 0; o >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        high = fmaxf(high, m);
        const float corr = m == -INFINITY ? 0.f : exp2_approx(m - high), f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - high);
        m = high;
        float sum = ml.x == -INFINITY ? 0.f : ml.y * f, empty = ml.x == -INFINITY ? ml.y : 0.f;
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            empty += __shfl_xor_sync(0xffffffffu, empty, o);
        }
        l = l * corr + sum;
        none += empty;
        acc.x *= corr; acc.y *= corr; acc.z *= corr; acc.w *= corr;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        for (int u = 0; u < n; ++u) {
            const float g = __shfl_sync(0xffffffffu, f, u);
            const float4 o = s_part[wid][u][lane];
            acc.x += o.x * g; acc.y += o.y * g; acc.z += o.z * g; acc.w += o.w * g;
        }
        __syncwarp();   // the parts have been read before the next come in their place
    }
    if (m == -INFINITY) l = none;
    const float inv = 1.f / l;
    if (l == 0.f) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    else acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(a.out + a.row_at(r, kvh, row) + 4 * lane) = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
}

// Keys or values of one layer as [page][head][position][128]: boxes of min(page, 128) positions x 64 dims with the 128-byte swizzle.
static CUtensorMap page_map(const void* base, const mfqb_cache& c) {
    typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static encode_fn encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            encode = reinterpret_cast<encode_fn>(p);
    });
    if (!encode) fail(MFQB_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    CUtensorMap map;
    const cuuint64_t dims[4] = {kHeadDim, (cuuint64_t)c.page, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {256, (cuuint64_t)c.page * 256, (cuuint64_t)c.kv_heads * c.page * 256};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(c.page, kTile), 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) fail(MFQB_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)rc);
    return map;
}

// Rows are paid for in steps, of which the last begin behind 128 and 256: 4 sequences at context 8192 over 8 kv heads take 47 us for 128 rows (32 nodes
// of groups of 4), 59 for 132, 64 for 256, 88 for 264, 98 for 512.
static int tree_streams(const mfqb_cache& c, int q_heads, int nodes) { return nodes * (q_heads / c.kv_heads) > kTile ? 2 : 1; }
static int64_t tree_parts(const mfqb_cache& c, int q_heads, int nodes) {   // rows of the parts
    const int ns = tree_streams(c, q_heads, nodes);
    return (int64_t)tree_ctas(ns) * 2 * std::min(ns * kTile, nodes * (q_heads / c.kv_heads));
}
static uint64_t tree_attention_work_bytes(const mfqb_cache& c, int q_heads, int nodes) {
    return (uint64_t)tree_parts(c, q_heads, nodes) * (kHeadDim * 4 + 8) + 8ull * (c.rows + 1);
}
static void check_heads(const mfqb_cache* c, int q_heads, const char* who) {
    if (q_heads < 1 || q_heads % c->kv_heads || q_heads / c->kv_heads > 16)
        fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to 16 query heads per kv head, got %d over %d", who, q_heads, c->kv_heads);
}

static void launch_tree_attention(const mfqb_cache& c, int layer, const void* q, int q_heads, int nodes, const uint64_t* masks, float scale, void* out, void* work,
                                  cudaStream_t s) {
    int device = 0;
    MFQB_CUDA(cudaGetDevice(&device));
    const int64_t per_layer = (int64_t)c.pages * c.kv_heads * c.page * kHeadDim;
    TreeArgs a{};
    a.table = c.table;
    a.lens = c.lens;
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.masks = reinterpret_cast<const unsigned long long*>(masks);
    a.k = static_cast<const __nv_bfloat16*>(c.k) + layer * per_layer;
    a.v = static_cast<const __nv_bfloat16*>(c.v) + layer * per_layer;
    a.out = static_cast<__nv_bfloat16*>(out);
    a.rows = c.rows;
    a.width = c.width;
    a.pages = c.pages;
    a.page = c.page;
    a.kv_heads = c.kv_heads;
    a.hq = q_heads;
    a.group = q_heads / c.kv_heads;
    a.nodes = nodes;
    a.group_inv = (65536u + a.group - 1) / a.group;
    const int ns = tree_streams(c, q_heads, nodes), m_rows = nodes * a.group;
    a.row_tiles = (m_rows + ns * kTile - 1) / (ns * kTile);
    a.tile_rows = std::min(ns * kTile, m_rows);
    a.part = static_cast<float*>(work);
    a.part_ml = reinterpret_cast<float2*>(a.part + tree_parts(c, q_heads, nodes) * kHeadDim);
    a.before = reinterpret_cast<int64_t*>(a.part_ml + tree_parts(c, q_heads, nodes));
    a.scale_log2 = scale * 1.4426950408889634f;
    a.error = device_status_word(device);
    const CUtensorMap kmap = page_map(a.k, c), vmap = page_map(a.v, c);
    auto* kernel = ns == 2 ? tree_attn_kernel<2, 1> : m_rows > 64 ? tree_attn_kernel<1, 1> : m_rows > 32 ? tree_attn_kernel<1, 2> : tree_attn_kernel<1, 4>;
    static std::once_flag once[64];
    std::call_once(once[device], [] {
        MFQB_CUDA(cudaFuncSetAttribute(tree_attn_kernel<2, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tree_smem(2)));
        for (auto* k : {tree_attn_kernel<1, 1>, tree_attn_kernel<1, 2>, tree_attn_kernel<1, 4>})
            MFQB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tree_smem(1)));
    });
    // Tables of up to kTreeWhole positions: an item is not split, and there is nothing to merge (one token at context 100: 8.1 us a pass, 9.3 with a table of
    // 8192 positions).
    a.whole = (int64_t)c.width * c.page <= kTreeWhole;
    const int64_t most = (int64_t)c.rows * c.kv_heads * a.row_tiles * (a.whole ? 1 : ((int64_t)c.width * c.page + kTile - 1) / kTile);   // tiles there can be
    const int ctas = (int)std::min<int64_t>(tree_ctas(ns), most);
    launch_chained(kernel, dim3(ctas), dim3(tree_threads(ns)), tree_smem(ns), s, a, kmap, vmap);
    if (a.whole) return;
    const int64_t rows = (int64_t)c.rows * c.kv_heads * m_rows;   // at most 1024 x 1024 x 1024
    launch_chained(tree_merge_kernel, dim3((unsigned)((rows + kMergeWarps - 1) / kMergeWarps)), dim3(32 * kMergeWarps), 0, s, a, ns, (int)rows);
}

}  // namespace mfqb

using namespace mfqb;

extern "C" {
#pragma GCC visibility push(default)

int mfqb_tree_attention_work(const mfqb_cache* c, int q_heads, int nodes, uint64_t* bytes) {
    return guarded([&] {
        check_cache(c, "mfqb_tree_attention_work");
        check_nodes(c, nodes, "mfqb_tree_attention_work");
        check_heads(c, q_heads, "mfqb_tree_attention_work");
        if (!bytes) fail(MFQB_ERR_ARG, "mfqb_tree_attention_work: null argument");
        ready_device();
        *bytes = tree_attention_work_bytes(*c, q_heads, nodes);
    });
}

int mfqb_tree_attention(const mfqb_cache* c, int layer, const void* q, int q_heads, int nodes, const uint64_t* masks, float scale, void* out,
                        void* work, uint64_t work_bytes, mfqb_stream_t stream) {
    return guarded([&] {
        check_cache(c, "mfqb_tree_attention");
        check_nodes(c, nodes, "mfqb_tree_attention");
        check_heads(c, q_heads, "mfqb_tree_attention");
        if (!q || !masks || !out || !work) fail(MFQB_ERR_ARG, "mfqb_tree_attention: null argument");
        if (((uintptr_t)q & 15) || ((uintptr_t)out & 15)) fail(MFQB_ERR_ARG, "mfqb_tree_attention: q and out must be 16-byte aligned");
        if ((uintptr_t)masks & 7) fail(MFQB_ERR_ARG, "mfqb_tree_attention: masks must be 8-byte aligned");
        if (layer < 0 || layer >= c->layers) fail(MFQB_ERR_ARG, "mfqb_tree_attention: layer %d of %d", layer, c->layers);
        if (!(scale > 0.f) || scale > 1e30f) fail(MFQB_ERR_ARG, "mfqb_tree_attention: scale must be positive and finite");
        if (((uintptr_t)work & 15) || work_bytes < tree_attention_work_bytes(*c, q_heads, nodes))
            fail(MFQB_ERR_ARG, "mfqb_tree_attention: work must be 16-byte aligned and hold %llu bytes, got %llu",
                 (unsigned long long)tree_attention_work_bytes(*c, q_heads, nodes), (unsigned long long)work_bytes);
        // add_bad_nodes reads the queries of rows that have been written
        const uint64_t bytes = 256ull * c->rows * nodes * q_heads;
        check_apart(out, bytes, q, bytes, "mfqb_tree_attention", "q and out");
        launch_tree_attention(*c, layer, q, q_heads, nodes, masks, scale, out, work, stream);
    });
}

#pragma GCC visibility pop
}  // extern "C"
