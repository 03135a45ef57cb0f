// Checks and launch helpers shared by the kernels on a paged key/value cache (mfqb_cache).
#pragma once
#include <algorithm>

#include "cuda_util.h"

namespace mfqb {

int* device_status_word(int device);
// What the attention needs of a device beside its arguments, the status word of its bounded waits, is allocated here and not at the first call,
// which may be in a stream capture.  Without a device there is nothing to ready.
inline void ready_device() {
    int device = 0;
    if (cudaGetDevice(&device) == cudaSuccess) device_status_word(device);
    else cudaGetLastError();
}

constexpr int kHeadDim = 128;
constexpr int kTreeNodes = 64;    // nodes of a drafted tree: one bit of a mask each
constexpr int kCacheRows = 1024;  // sequences of a cache: one thread each in the kernels that give out pages

// Throws unless the view describes a cache that the kernels take.  Their index arithmetic relies on these bounds: positions fit 31
// bits, page numbers and table entries too; offsets into the pools are formed in 64 bits.
inline void check_cache(const mfqb_cache* c, const char* who) {
    if (!c) fail(MFQB_ERR_ARG, "%s: null cache", who);
    if (!c->k || !c->v || !c->table || !c->lens || !c->refs) fail(MFQB_ERR_ARG, "%s: the cache has a null pointer", who);
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) fail(MFQB_ERR_ARG, "%s: key and value pools must be 16-byte aligned", who);
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1))) fail(MFQB_ERR_UNSUPPORTED, "%s: a page must hold 16 to 1024 tokens, a power of two, got %d", who, c->page);
    if (c->layers < 1 || c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024) fail(MFQB_ERR_ARG, "%s: layers, pages and heads must be positive (heads at most 1024)", who);
    if (c->rows < 1 || c->rows > kCacheRows) fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d sequences, got %d", who, kCacheRows, c->rows);
    if (c->width < 1 || (int64_t)c->width * c->page > (1ll << 30) || (int64_t)c->width * c->rows > (1ll << 30))
        fail(MFQB_ERR_UNSUPPORTED, "%s: at most 2^30 positions per sequence and table entries, got %d pages of %d", who, c->width, c->page);
}
inline void check_nodes(const mfqb_cache* c, int nodes, const char* who) {
    if (nodes < 1 || nodes > kTreeNodes) fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d nodes per sequence, got %d", who, kTreeNodes, nodes);
    if ((int64_t)nodes > (int64_t)c->width * c->page) fail(MFQB_ERR_ARG, "%s: %d nodes do not fit a table of %d pages of %d", who, nodes, c->width, c->page);
}

inline void check_apart(const void* out, uint64_t out_bytes, const void* in, uint64_t in_bytes, const char* who, const char* what) {
    const uintptr_t o = (uintptr_t)out, i = (uintptr_t)in;
    if (o < i + in_bytes && i < o + out_bytes) fail(MFQB_ERR_ARG, "%s: %s overlap", who, what);
}

// Launched with the programmatic-dependent-launch attribute: the kernel becomes resident while its predecessor runs and waits
// (after_predecessor) until that one has completed.
template <typename... KArgs, typename... Args>
void launch_chained(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MFQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
}

#if defined(__CUDACC__)
// The kernels here start while the one before them runs, so what that one writes is not constant for their lifetime: they read it after this
// wait, from the L2 cache (__ldcg) or by loads that the compiler may not take for constant (no const __restrict__).
__device__ __forceinline__ void chained_wait() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two float32 values in one register pair, for the instructions that take both at once.
__device__ __forceinline__ uint64_t pair_f32(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 split_f32(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
#endif

}  // namespace mfqb
