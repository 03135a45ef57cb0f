// Attention of a tree of drafted tokens over a paged key/value cache.
#include <cuda_bf16.h>

#include "paged.h"

namespace mfqb {

// CTA (query head, node, sequence), four warps that take every fourth position each.
__global__ void __launch_bounds__(128) tree_attn_kernel(mfqb_cache c, int layer, const __nv_bfloat16* __restrict__ q, int hq, int nodes,
                                                        const unsigned long long* __restrict__ masks, float scale, __nv_bfloat16* __restrict__ out) {
    chained_wait();
    __shared__ float s_acc[4][kHeadDim], s_m[4], s_l[4];
    const int h = blockIdx.x, node = blockIdx.y, r = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = h / (hq / c.kv_heads);
    const int64_t cap = (int64_t)c.width * c.page;
    const int64_t len = min(max((int64_t)c.lens[r], (int64_t)0), cap), end = min(len + nodes, cap);
    const int64_t item = ((int64_t)r * nodes + node) * hq + h;
    const unsigned long long mask = masks[(int64_t)r * nodes + node];
    auto load4 = [](const __nv_bfloat16* p) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
    };
    float4 qv = load4(q + item * kHeadDim + 4 * lane);
    const float f = scale * 1.4426950408889634f;
    qv.x *= f; qv.y *= f; qv.z *= f; qv.w *= f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    bool seen = false;
    for (int64_t t = warp; t < end; t += 4) {
        if (t >= len && !((mask >> (t - len)) & 1ull)) continue;
        const int page = c.table[(int64_t)r * c.width + t / c.page];
        if ((unsigned)page >= (unsigned)c.pages) continue;
        const int64_t off = ((((int64_t)layer * c.pages + page) * c.kv_heads + kvh) * c.page + (t & (c.page - 1))) * kHeadDim + 4 * lane;
        const float4 kv = load4(static_cast<const __nv_bfloat16*>(c.k) + off), vv = load4(static_cast<const __nv_bfloat16*>(c.v) + off);
        float s = qv.x * kv.x + qv.y * kv.y + qv.z * kv.z + qv.w * kv.w;
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        seen = true;
        const float mn = fmaxf(m, s);
        const float corr = m == -INFINITY ? 0.f : exp2f(m - mn);
        const float p = __bfloat162float(__float2bfloat16_rn(mn == -INFINITY ? 0.f : exp2f(s - mn)));
        l = l * corr + p;
        acc.x = acc.x * corr + p * vv.x; acc.y = acc.y * corr + p * vv.y; acc.z = acc.z * corr + p * vv.z; acc.w = acc.w * corr + p * vv.w;
        m = mn;
    }
    if (m == -INFINITY && seen) l = NAN;   // every score minus infinity
    *reinterpret_cast<float4*>(&s_acc[warp][4 * lane]) = acc;
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    __syncthreads();
    float mm = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), ll = 0.f, a = 0.f;
    for (int w = 0; w < 4; ++w) {
        const float cw = s_m[w] == mm ? 1.f : exp2f(s_m[w] - mm);
        if (s_m[w] == -INFINITY && mm > -INFINITY) continue;
        ll += s_l[w] * cw;
        a += s_acc[w][threadIdx.x] * cw;
    }
    out[item * kHeadDim + threadIdx.x] = __float2bfloat16_rn(ll == 0.f ? 0.f : a / ll);
}

static uint64_t tree_attention_work_bytes(const mfqb_cache&, int, int) { return 16; }
static void check_heads(const mfqb_cache* c, int q_heads, const char* who) {
    if (q_heads < 1 || q_heads % c->kv_heads || q_heads / c->kv_heads > 16)
        fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to 16 query heads per kv head, got %d over %d", who, q_heads, c->kv_heads);
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
        if (layer < 0 || layer >= c->layers) fail(MFQB_ERR_ARG, "mfqb_tree_attention: layer %d of %d", layer, c->layers);
        if (((uintptr_t)work & 15) || work_bytes < tree_attention_work_bytes(*c, q_heads, nodes))
            fail(MFQB_ERR_ARG, "mfqb_tree_attention: work must be 16-byte aligned and hold %llu bytes, got %llu",
                 (unsigned long long)tree_attention_work_bytes(*c, q_heads, nodes), (unsigned long long)work_bytes);
        launch_chained(tree_attn_kernel, dim3(q_heads, nodes, c->rows), dim3(128), 0, stream, *c, layer, static_cast<const __nv_bfloat16*>(q), q_heads, nodes,
                       reinterpret_cast<const unsigned long long*>(masks), scale, static_cast<__nv_bfloat16*>(out));
    });
}

#pragma GCC visibility pop
}  // extern "C"
