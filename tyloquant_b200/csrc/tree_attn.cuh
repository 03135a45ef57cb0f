// What the attention over pages and the sums of its weights share.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include <mutex>

#include "paged.h"
#include "tc05.cuh"

namespace mfqb {

constexpr int kTreeSms = 148;
constexpr int kTile = 128;                           // rows of Q, positions of a tile
constexpr int kTileBytes = kTile * kHeadDim * 2, kHalfBytes = kTileBytes / 2;
constexpr int kScoreRows = 64;                       // up to so many rows the attention may keep its scores
constexpr int kTreeStart = 2;                        // what starting and ending a stretch takes, in tiles

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
    float2* row_ml;               // [rows][kv_heads][rows of Q]: maximum (in powers of two) and 1 / sum of every row, where weights are added up
    float* scores;                // [rows][kv_heads][rows of Q][score_stride]: raw scores, minus infinity where a row does not see, or null
    int64_t score_stride;
    float* weights;               // of the layer: [rows][kv_heads][width * page], or null
    bool used;                    // nodes whose mask is 0 stand for none: their rows' (maximum, 1 / sum) is (0, 0)
    unsigned group_inv;           // ceil(65536 / group): row / group = row * group_inv >> 16 for rows below 1024, groups up to 16
    float scale_log2;
    __device__ __forceinline__ int node_of(int row_of_q) const { return (int)((unsigned)row_of_q * group_inv >> 16); }
    // Do a node's rows count among the weights?
    __device__ __forceinline__ bool counts(unsigned long long mask) const { return !used || (nodes < 64 ? mask & ((1ull << nodes) - 1ull) : mask) != 0; }
    __device__ __forceinline__ bool row_counts(int r, int row_of_q) const { return !used || counts(__ldcg(masks + (int64_t)r * nodes + node_of(row_of_q))); }
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

// Keys or values of one layer as [page][head][position][128]: boxes of min(page, 128) positions x 64 dims with the 128-byte swizzle.
inline CUtensorMap page_map(const void* base, const mfqb_cache& c) {
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


// What a position of sequence r gets, from the scores that the attention has kept: exp2(scale' score - x) y of every row's (x, y), in their order, nothing
// for a score of minus infinity, nor of a row with y = 0, whatever its scores are.  Positions pos .. pos + N - 1 lie in one page.
template <int N>
__device__ __forceinline__ void add_weights(const TreeArgs& a, const TreeSeq& seq, int r, int kvh, const float2* scale, int m_rows, int pos) {
    const int64_t item = (int64_t)r * a.kv_heads + kvh;
    const float* scores = a.scores + item * m_rows * a.score_stride + pos;
    float* to = a.weights + item * a.width * a.page + pos;
    const int page = __ldcg(a.table + (int64_t)r * a.width + pos / a.page);
    const bool good = (unsigned)page < (unsigned)a.pages;
    float before[N], sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        before[e] = pos + e < seq.len ? to[e] : 0.f;
        sum[e] = 0.f;
    }
#pragma unroll 4
    for (int row = 0; row < m_rows; ++row) {
        const float2 ml = scale[row];
        float v[N];
        if constexpr (N == 4) {
            const float4 s = __ldcg(reinterpret_cast<const float4*>(scores + row * a.score_stride));
            v[0] = s.x; v[1] = s.y; v[2] = s.z; v[3] = s.w;
        } else {
            v[0] = __ldcg(scores + row * a.score_stride);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[e] == -INFINITY || ml.y == 0.f ? 0.f : exp2_approx(fmaf(v[e], a.scale_log2, -ml.x)) * ml.y;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (pos + e >= seq.end) break;
        if (pos + e >= seq.len) to[e] = good ? sum[e] : 0.f;   // a node's
        else if (good) to[e] = before[e] + sum[e];
    }
}

// The sums of the attention's weights where it has not kept its scores (tree_weigh.cu), from row_ml and the keys.
uint64_t tree_weigh_bytes(const mfqb_cache& c, int q_heads, int nodes);
int64_t tree_score_stride(const mfqb_cache& c, int q_heads, int nodes);   // 0 where scores are not kept
void launch_tree_weigh(const mfqb_cache& c, const TreeArgs& a, cudaStream_t s);

}  // namespace mfqb
