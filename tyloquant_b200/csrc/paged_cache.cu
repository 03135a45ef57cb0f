// A key/value cache in pages: reserving, sharing, copying and freeing pages, rotary embedding and write of a step's queries, keys
// and values, and keeping the accepted branch of a tree of drafted tokens.
#include <cuda_bf16.h>

#include "paged.h"

namespace mfqb {

// Inclusive sum over the 1024 threads of a CTA; every thread calls it.
__device__ __forceinline__ int scan1024(int v, int* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();   // the sums of an earlier call have been read
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    int before = warp_sums[lane];
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    return v + (warp ? __shfl_sync(0xffffffffu, before, warp - 1) : 0);
}

// The `need` lowest page numbers that are free (refs, plus delta where given, 0 or less) into list; returns how many there are, at
// most need.  All 1024 threads take part; four pages a thread and round, so that a round is one trip to memory.
__device__ __forceinline__ int find_free(const int* refs, const int* delta, int pages, int need, int* list, int* warp_sums) {
    int found = 0;
    for (int base = 0; base < pages && found < need; base += 4096) {
        int mine = 0;
        bool f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = base + (int)threadIdx.x * 4 + j;
            f[j] = p < pages && refs[p] + (delta ? delta[p] : 0) <= 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += f[j];
        const int upto = scan1024(mine, warp_sums);
        int at = found + upto - mine;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (f[j]) {
                if (at < need) list[at] = base + (int)threadIdx.x * 4 + j;
                ++at;
            }
        __shared__ int total;
        if (threadIdx.x == 1023) total = upto;
        __syncthreads();
        found += total;
        __syncthreads();
    }
    return min(found, need);
}

// One CTA, a thread per sequence.  Bound by its chain of trips to memory (lengths, table, counts, table), not by their number.
__global__ void __launch_bounds__(1024) extend_kernel(mfqb_cache c, const int* tokens, int* status) {
    chained_wait();
    __shared__ int warp_sums[32], list[1024];
    __shared__ unsigned long long lack_table;
    const int r = threadIdx.x;
    if (r == 0) lack_table = 0;
    __syncthreads();
    int first = 0, last = 0, need = 0;   // table entries [first, last) have to hold pages
    int* row = c.table + (int64_t)min(r, c.rows - 1) * c.width;
    const int more = r < c.rows ? __ldcg(tokens + r) : 0;
    if (more > 0) {
        const int64_t len = min(max((int64_t)c.lens[r], (int64_t)0), (int64_t)c.width * c.page);
        const int64_t want = (len + more + c.page - 1) / c.page;
        first = (int)(len / c.page);
        last = (int)min(want, (int64_t)c.width);
        if (want > c.width) atomicAdd(&lack_table, (unsigned long long)(want - c.width));
        for (int i = first; i < last; ++i) need += (unsigned)row[i] >= (unsigned)c.pages;
    }
    const int upto = scan1024(need, warp_sums);
    __shared__ int total;
    if (r == 1023) total = upto;
    __syncthreads();
    // Up to 1024 pages come from one search; more are counted first, so that nothing has changed when the pool turns out too small.
    int have = 0;
    if (total > 1024) {
        for (int base = 0; base < c.pages && have < total; base += 1024) {
            const int p = base + r;
            have += __syncthreads_count(p < c.pages && c.refs[p] <= 0);
        }
    } else if (total) {
        have = find_free(c.refs, nullptr, c.pages, total, list, warp_sums);
    }
    if (have < total || lack_table) {
        if (r == 0) *status = (int)min(lack_table + max(0, total - have), 0x7FFFFFFFull);
        return;
    }
    if (r == 0) *status = 0;
    int next = first, left = need, at = upto - need;   // this thread's next entry, and the rank of the page it waits for
    for (int done = 0; done < total; done += 1024) {
        const int n = total > 1024 ? find_free(c.refs, nullptr, c.pages, min(1024, total - done), list, warp_sums) : total;
        __syncthreads();
        while (left > 0 && at < done + n) {
            while ((unsigned)row[next] < (unsigned)c.pages) ++next;
            const int p = list[at - done];
            row[next] = p;
            c.refs[p] = 1;
            ++at;
            --left;
        }
        __syncthreads();
    }
}

// What fork_plan_kernel leaves for fork_copy_kernel: how many copies, then one entry each.
struct ForkCopy {
    int src, dst, tokens, pad;
};
struct ForkWork {
    int* count;        // [4]
    ForkCopy* copies;  // [rows]
    int* delta;        // [pages]: change of the counts
    int* table;        // [rows][width]
};
static ForkWork fork_work(const mfqb_cache& c, void* work) {
    ForkWork w;
    w.count = static_cast<int*>(work);
    w.copies = reinterpret_cast<ForkCopy*>(w.count + 4);
    w.delta = reinterpret_cast<int*>(w.copies + c.rows);
    w.table = w.delta + (c.pages + 3) / 4 * 4;
    return w;
}
static uint64_t fork_work_bytes(const mfqb_cache& c) {
    return 16 + 16ull * c.rows + 4ull * ((c.pages + 3) / 4 * 4) + 4ull * c.rows * c.width;
}

constexpr int kForkSmall = 8 * 1024;   // pages and table entries together that find room in shared memory

// One CTA: the new table and the change of the counts are made beside the old ones and put in place at the end, when it is known
// that the pages suffice.  Counts change by integer atomics, whose order does not matter.  Bound by its chain of dependent trips, not by their
// size: where both fit they are in shared memory.  With the copies of 32 pages in two layers, 64 sequences at context 4090 on pages of 64: 11.7 us over
// a pool of 1200 pages, 13.3 over 5000, 17.0 over 20000.
__global__ void __launch_bounds__(1024) fork_plan_kernel(mfqb_cache c, const int* parents, int* status, ForkWork w, bool small) {
    chained_wait();
    __shared__ int warp_sums[32], list[1024], s_len[kCacheRows], s_last[kCacheRows], total;
    extern __shared__ int s_small[];
    const int r = threadIdx.x, bits = __ffs(c.page) - 1;
    if (small) {
        w.delta = s_small;
        w.table = s_small + c.pages;
    }
    int parent = -1, len = 0;
    bool bad = false;
    if (r < c.rows) {
        parent = __ldcg(parents + r);
        bad = parent < -1 || parent >= c.rows;
        if (!bad && parent >= 0) len = (int)min(max((int64_t)c.lens[parent], (int64_t)0), (int64_t)c.width * c.page);
    }
    s_len[r] = len;
    for (int p = r; p < c.pages; p += 1024) w.delta[p] = 0;
    if (__syncthreads_or(bad)) {
        if (r == 0) {
            *status = -1;
            w.count[0] = 0;
        }
        return;
    }
    auto valid = [&](int p) { return (unsigned)p < (unsigned)c.pages; };
    const int entries = c.rows * c.width;
    for (int e = r; e < entries; e += 1024) {
        const int row = e / c.width, i = e - row * c.width;
        const int old = c.table[e];
        int now = -1;
        if (((int64_t)i << bits) < s_len[row]) now = c.table[(int64_t)__ldcg(parents + row) * c.width + i];
        if (!valid(now)) now = -1;
        w.table[e] = now;
        const bool part = now >= 0 && i == (s_len[row] >> bits) && (s_len[row] & (c.page - 1));   // counted below, once it is known whose it is
        if (valid(old)) atomicSub(w.delta + old, 1);
        if (now >= 0 && !part) atomicAdd(w.delta + now, 1);
    }
    __syncthreads();
    const int at = len >> bits, fill = len & (c.page - 1);
    const int last = r < c.rows && fill ? w.table[(int64_t)r * c.width + at] : -1;
    s_last[r] = last;
    __syncthreads();
    bool twin = false;
    if (last >= 0)
        for (int j = 0; j < r; ++j) twin |= s_last[j] == last;
    if (last >= 0 && !twin) atomicAdd(w.delta + last, 1);
    const int upto = scan1024(twin, warp_sums);
    if (r == 1023) total = upto;
    __syncthreads();
    const int need = total, have = need ? find_free(c.refs, w.delta, c.pages, need, list, warp_sums) : 0;
    __syncthreads();
    if (have < need) {
        if (r == 0) {
            *status = need - have;
            w.count[0] = 0;
        }
        return;
    }
    if (twin) {
        const int p = list[upto - 1];
        w.table[(int64_t)r * c.width + at] = p;
        w.copies[upto - 1] = ForkCopy{last, p, fill, 0};
        w.delta[p] = (int)(1u - (unsigned)c.refs[p]);   // one holder, whatever a free page's count was
    }
    if (r == 0) {
        *status = 0;
        w.count[0] = need;
    }
    if (r < c.rows) c.lens[r] = len;
    __syncthreads();
    for (int e = r; e < entries; e += 1024) c.table[e] = w.table[e];
    for (int p = r; p < c.pages; p += 1024)
        if (const int d = w.delta[p]) c.refs[p] = (int)((unsigned)c.refs[p] + (unsigned)d);
}

// Copies of the filled part of a page: (copy, layer, head, keys or values) is one contiguous stretch of tokens * 256 bytes.  Bound by memory: 32
// pages in six layers, 51 MB read and written, 10 us with the launch.
__global__ void __launch_bounds__(256) fork_copy_kernel(mfqb_cache c, ForkWork w) {
    chained_wait();
    const int heads = c.kv_heads;
    const int64_t per = (int64_t)c.layers * heads * 2, units = per * w.count[0];
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const ForkCopy f = w.copies[u / per];
        const int64_t rest = u % per, lh = rest >> 1, layer = lh / heads, head = lh % heads;
        char* pool = static_cast<char*>(rest & 1 ? c.v : c.k);
        const int64_t stride = (int64_t)c.page * 256;
        const uint4* src = reinterpret_cast<const uint4*>(pool + ((layer * c.pages + f.src) * heads + head) * stride);
        uint4* dst = reinterpret_cast<uint4*>(pool + ((layer * c.pages + f.dst) * heads + head) * stride);
        const int n = f.tokens * 16;
        int i = threadIdx.x;
        for (; i + 3 * 256 < n; i += 4 * 256) {
            const uint4 a = src[i], b = src[i + 256], d = src[i + 512], e = src[i + 768];
            dst[i] = a; dst[i + 256] = b; dst[i + 512] = d; dst[i + 768] = e;
        }
        for (; i < n; i += 256) dst[i] = src[i];
    }
}

// A warp per sequence, two nodes a lane.  mask = own bit | mask of the parent: pointers are doubled, six rounds for 64 nodes.  A
// chain that does not end at a root of its own leaves no bit 0: the node is unused.
__global__ void __launch_bounds__(32) tree_masks_kernel(const int* parents, int nodes, unsigned long long* masks, int* depths) {
    chained_wait();
    __shared__ unsigned long long s_mask[kTreeNodes];
    __shared__ int s_up[kTreeNodes];
    const int* row = parents + (int64_t)blockIdx.x * nodes;
    const int lane = threadIdx.x;
    const bool rooted = __ldcg(row) == -1;
#pragma unroll
    for (int j = lane; j < kTreeNodes; j += 32) {
        const int p = j > 0 && j < nodes ? __ldcg(row + j) : -1;
        s_up[j] = p >= 0 && p < j ? p : -1;
        s_mask[j] = 1ull << j;
    }
    __syncwarp();
    for (int round = 0; round < 6; ++round) {
        unsigned long long m[2];
        int up[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = lane + 32 * h, p = s_up[j];
            m[h] = s_mask[j] | (p >= 0 ? s_mask[p] : 0ull);
            up[h] = p >= 0 ? s_up[p] : -1;
        }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s_mask[lane + 32 * h] = m[h];
            s_up[lane + 32 * h] = up[h];
        }
        __syncwarp();
    }
    for (int j = lane; j < nodes; j += 32) {
        const unsigned long long m = rooted && (s_mask[j] & 1ull) ? s_mask[j] : 0ull;
        masks[(int64_t)blockIdx.x * nodes + j] = m;
        depths[(int64_t)blockIdx.x * nodes + j] = m ? __popcll(m) - 1 : 0;
    }
}

// CTA (heads of one sixteenth, node, sequence): 16 threads per head, four pairs (j, j + 64) a thread.  The angle is formed and reduced
// to [-pi, pi] in 64 bits (a float32 product is off by 2e-3 radians at position 32768), its sine and cosine are taken once per
// CTA.  Queries are rounded to bf16 once, the type in which the attention's first product takes them.  Bound by memory: six bytes per value (64
// nodes of 16 sequences, 32 + 2 x 8 heads: 7.1 us, 5.3 TB/s).
__global__ void __launch_bounds__(256) cache_write_kernel(mfqb_cache c, int layer, const float* qkv, int hq, int nodes, const int* depths, const double* freqs,
                                                          __nv_bfloat16* q_out) {
    chained_wait();
    __shared__ float s_cos[64], s_sin[64];
    const int node = blockIdx.y, r = blockIdx.z, t = threadIdx.x, heads = hq + 2 * c.kv_heads;
    const int64_t cap = (int64_t)c.width * c.page;
    const int64_t len = min(max((int64_t)c.lens[r], (int64_t)0), cap);
    const int64_t item = (int64_t)r * nodes + node;
    if (t < 64) {
        const double a = (double)(len + __ldcg(depths + item)) * __ldcg(freqs + t);
        const double n = rint(a * 0.15915494309189533577);
        float sn, cs;
        sincosf((float)fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586477, a)), &sn, &cs);
        s_cos[t] = cs;
        s_sin[t] = sn;
    }
    __syncthreads();
    const int64_t slot = len + node;
    int page = -1;
    if (slot < cap) page = c.table[(int64_t)r * c.width + slot / c.page];
    const bool room = (unsigned)page < (unsigned)c.pages;
    const int j = 4 * (t & 15);   // this thread's pairs
    const float4 cs = *reinterpret_cast<const float4*>(s_cos + j), sn = *reinterpret_cast<const float4*>(s_sin + j);
    for (int h = blockIdx.x * 16 + (t >> 4); h < heads; h += gridDim.x * 16) {
        const float* src = qkv + (item * heads + h) * kHeadDim + j;
        float4 lo = __ldcg(reinterpret_cast<const float4*>(src)), hi = __ldcg(reinterpret_cast<const float4*>(src + 64));
        if (h < hq + c.kv_heads) {
            const float4 a = lo, b = hi;
            lo = make_float4(a.x * cs.x - b.x * sn.x, a.y * cs.y - b.y * sn.y, a.z * cs.z - b.z * sn.z, a.w * cs.w - b.w * sn.w);
            hi = make_float4(b.x * cs.x + a.x * sn.x, b.y * cs.y + a.y * sn.y, b.z * cs.z + a.z * sn.z, b.w * cs.w + a.w * sn.w);
        }
        __nv_bfloat16* dst;
        if (h < hq) {
            dst = q_out + (item * hq + h) * kHeadDim;
        } else {
            if (!room) continue;
            const int kv = h < hq + c.kv_heads ? h - hq : h - hq - c.kv_heads;
            dst = static_cast<__nv_bfloat16*>(h < hq + c.kv_heads ? c.k : c.v) +
                  ((((int64_t)layer * c.pages + page) * c.kv_heads + kv) * c.page + (slot & (c.page - 1))) * kHeadDim;
        }
        const __nv_bfloat162 l0 = __floats2bfloat162_rn(lo.x, lo.y), l1 = __floats2bfloat162_rn(lo.z, lo.w);
        const __nv_bfloat162 h0 = __floats2bfloat162_rn(hi.x, hi.y), h1 = __floats2bfloat162_rn(hi.z, hi.w);
        *reinterpret_cast<uint2*>(dst + j) = make_uint2(*reinterpret_cast<const uint32_t*>(&l0), *reinterpret_cast<const uint32_t*>(&l1));
        *reinterpret_cast<uint2*>(dst + j + 64) = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
    }
}

// Four of a head's values at dims d .., as float32.
__device__ __forceinline__ float4 rope_load4(const float* p) { return __ldcg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 rope_load4(const __nv_bfloat16* p) {
    const uint2 v = __ldcg(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
}
__device__ __forceinline__ float rope_load(const float* p) { return __ldcg(p); }
__device__ __forceinline__ float rope_load(const __nv_bfloat16* p) { return __bfloat162float(__ldcg(p)); }
__device__ __forceinline__ uint2 rope_pack(float a, float b, float c, float d) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(a, b), hi = __floats2bfloat162_rn(c, d);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// How a thread's four pairs of a head lie: pairs (2j, 2j + 1); pairs (j, j + P) with P a multiple of four; with any P.
enum RopeForm { kRopeNeighbours, kRopeHalves4, kRopeHalves };

// cache_write_kernel's work for P <= 64 pairs, in other layouts and with a factor on what is turned.  (That one stays for whole heads in halves: 6.5 us where this takes 6.9,
// for 64 nodes of 16 sequences with 48 heads in float32, and its sums round as they did; neighbouring pairs 7.0, any other number of pairs 10.3.)  Bound by memory.  Dims from 2P on pass, as pairs of neighbours: a head
// has 64 pairs in all, of which thread t of 16 takes 4t .. 4t + 3 (kRopeHalves: t, t + 16, ..).
template <typename T, RopeForm FORM>
__global__ void __launch_bounds__(256) cache_rope_kernel(mfqb_cache c, int layer, const T* qkv, int hq, int nodes, const int* depths, const double* freqs, int pairs, float factor,
                                                         __nv_bfloat16* q_out) {
    chained_wait();
    __shared__ float s_cos[64], s_sin[64];
    const int node = blockIdx.y, r = blockIdx.z, t = threadIdx.x, heads = hq + 2 * c.kv_heads;
    const int64_t cap = (int64_t)c.width * c.page;
    const int64_t len = min(max((int64_t)c.lens[r], (int64_t)0), cap);
    const int64_t item = (int64_t)r * nodes + node;
    if (t < pairs) {
        const double a = (double)(len + __ldcg(depths + item)) * __ldcg(freqs + t);
        const double n = rint(a * 0.15915494309189533577);
        float sn, cs;
        sincosf((float)fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586477, a)), &sn, &cs);
        s_cos[t] = cs * factor;
        s_sin[t] = sn * factor;
    }
    __syncthreads();
    const int64_t slot = len + node;
    int page = -1;
    if (slot < cap) page = c.table[(int64_t)r * c.width + slot / c.page];
    const bool room = (unsigned)page < (unsigned)c.pages;
    const int p0 = t & 15;
    float cs[4], sn[4];
    bool turn[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int j = FORM == kRopeHalves ? p0 + 16 * e : 4 * p0 + e;
        turn[e] = j < pairs;
        cs[e] = turn[e] ? s_cos[j] : 0.f;
        sn[e] = turn[e] ? s_sin[j] : 0.f;
    }
    for (int h = blockIdx.x * 16 + (t >> 4); h < heads; h += gridDim.x * 16) {
        const T* src = qkv + (item * heads + h) * kHeadDim;
        __nv_bfloat16* dst;
        if (h < hq) {
            dst = q_out + (item * hq + h) * kHeadDim;
        } else {
            if (!room) continue;
            const int kv = h < hq + c.kv_heads ? h - hq : h - hq - c.kv_heads;
            dst = static_cast<__nv_bfloat16*>(h < hq + c.kv_heads ? c.k : c.v) +
                  ((((int64_t)layer * c.pages + page) * c.kv_heads + kv) * c.page + (slot & (c.page - 1))) * kHeadDim;
        }
        const bool near = FORM == kRopeNeighbours || !turn[0];   // this thread's pairs are eight dims in a row (not asked in kRopeHalves)
        float x[4], y[4];
        if (FORM == kRopeHalves) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = p0 + 16 * e;
                x[e] = rope_load(src + (turn[e] ? j : 2 * j));
                y[e] = rope_load(src + (turn[e] ? j + pairs : 2 * j + 1));
            }
        } else {
            const float4 u = rope_load4(src + (near ? 8 * p0 : 4 * p0)), v = rope_load4(src + (near ? 8 * p0 + 4 : 4 * p0 + pairs));
            x[0] = u.x; x[1] = near ? u.z : u.y; x[2] = near ? v.x : u.z; x[3] = near ? v.z : u.w;
            y[0] = near ? u.y : v.x; y[1] = near ? u.w : v.y; y[2] = near ? v.y : v.z; y[3] = v.w;
        }
        if (h < hq + c.kv_heads) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (turn[e]) {
                    const float a = x[e], b = y[e];
                    x[e] = a * cs[e] - b * sn[e];
                    y[e] = b * cs[e] + a * sn[e];
                }
        }
        if (FORM == kRopeHalves) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = p0 + 16 * e;
                dst[turn[e] ? j : 2 * j] = __float2bfloat16_rn(x[e]);
                dst[turn[e] ? j + pairs : 2 * j + 1] = __float2bfloat16_rn(y[e]);
            }
        } else if (near) {
            const uint2 u = rope_pack(x[0], y[0], x[1], y[1]), v = rope_pack(x[2], y[2], x[3], y[3]);
            *reinterpret_cast<uint4*>(dst + 8 * p0) = make_uint4(u.x, u.y, v.x, v.y);
        } else {
            *reinterpret_cast<uint2*>(dst + 4 * p0) = rope_pack(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint2*>(dst + 4 * p0 + pairs) = rope_pack(y[0], y[1], y[2], y[3]);
        }
    }
}

template <typename T>
static void launch_cache_rope(const mfqb_cache& c, int layer, const void* qkv, int q_heads, int nodes, const int32_t* depths, const double* freqs, int pairs, int layout,
                              float factor, void* q_out, cudaStream_t s) {
    const int parts = c.rows * nodes >= 148 ? 1 : (q_heads + 2 * c.kv_heads + 15) / 16;
    auto* kernel = layout == MFQB_ROPE_INTERLEAVED ? cache_rope_kernel<T, kRopeNeighbours> : pairs % 4 == 0 ? cache_rope_kernel<T, kRopeHalves4> : cache_rope_kernel<T, kRopeHalves>;
    launch_chained(kernel, dim3(parts, nodes, c.rows), dim3(256), 0, s, c, layer, static_cast<const T*>(qkv), q_heads, nodes, depths, freqs, pairs, factor,
                   static_cast<__nv_bfloat16*>(q_out));
}

// CTA (some layers' heads, sequence): its first warp walks the tree, two nodes a lane, the first CTA of a sequence leaves the results, and all move
// the branch's rows, 64 at a time, which are its nodes in as many heads as that makes.  Every row is read into registers before the first one is
// written, since a slot that one node leaves is another one's place.  A chain from the lengths to the rows: one tree of 8 nodes 4.2 us, 16 of 48
// with branches of 13 in 128 heads 8.6 (a launch for the walk and one for the rows: 5.0 and 9.0; with a CTA for each head of each layer 11).  Lengths
// that change in place are a second launch, 0.7 and 1.1 us more.
// WEIGH: the branch's sums in weights (mfqb_tree_attention_weigh) move along.  A form of its own: as a pointer that may be null it took calls without weights from 9.0 to
// 10.3 us (16 trees of 48 nodes).
template <bool WEIGH>
__global__ void __launch_bounds__(256) accept_kernel(mfqb_cache c, const int* ids, const int* parents, const int* targets, int nodes, int* count, int* token,
                                                     int* path, int* lens_out, float* weights) {
    chained_wait();
    __shared__ int s_path[kTreeNodes], s_n, s_token;
    __shared__ int64_t s_from[kTreeNodes], s_to[kTreeNodes];   // rows of the branch in 16-byte pieces, for head 0 of layer 0; -1: stays
    const int r = blockIdx.y, t = threadIdx.x, lane = t & 31, heads = c.layers * c.kv_heads;
    const int64_t base = (int64_t)r * nodes, cap = (int64_t)c.width * c.page, len = min(max((int64_t)c.lens[r], (int64_t)0), cap);
    if (t < 32) {
        int id[2], up[2], to[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = lane + 32 * h;
            const bool in = j < nodes;
            id[h] = in ? __ldcg(ids + base + j) : 0;
            up[h] = in ? __ldcg(parents + base + j) : -2;
            to[h] = in ? __ldcg(targets + base + j) : 0;
        }
        int cur = 0, n = 0, want = -1;
        if (__shfl_sync(0xffffffffu, up[0], 0) == -1) {
            for (;;) {
                if (lane == 0) s_path[n] = cur;
                ++n;
                want = __shfl_sync(0xffffffffu, cur < 32 ? to[0] : to[1], cur & 31);
                const unsigned lo = __ballot_sync(0xffffffffu, lane > cur && up[0] == cur && id[0] == want);
                const unsigned hi = __ballot_sync(0xffffffffu, lane + 32 > cur && up[1] == cur && id[1] == want);
                if (!(lo | hi)) break;
                cur = lo ? __ffs(lo) - 1 : __ffs(hi) + 31;
            }
        }
        if (lane == 0) {
            s_n = n;
            s_token = want;
        }
    }
    __syncthreads();
    const int n = s_n;
    if (blockIdx.x == 0) {
        if (t < nodes) path[base + t] = t < n ? s_path[t] : -1;
        if (t == 0) {
            count[r] = n;
            token[r] = s_token;
            if (lens_out) lens_out[r] = (int)len + n;
        }
    }
    if (n < 2) return;
    const int each = kTreeNodes / n;   // heads at a time
    if (t < n) {
        auto slot = [&](int64_t p) -> int64_t {   // -1 where there is no page
            const int page = p < cap ? c.table[(int64_t)r * c.width + p / c.page] : -1;
            return (unsigned)page < (unsigned)c.pages ? ((int64_t)page * c.kv_heads * c.page + (p & (c.page - 1))) * 16 : -1;
        };
        const int from = s_path[t];
        s_to[t] = slot(len + t);
        s_from[t] = from == t || s_to[t] < 0 ? -1 : slot(len + from);
    }
    __syncthreads();
    for (int64_t h0 = (int64_t)blockIdx.x * each; h0 < heads; h0 += (int64_t)gridDim.x * each) {
        uint4 kv[4][2];
        int64_t to[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // 16 threads a row, 16 rows a round
            const int x = 16 * i + (t >> 4), h = x / n, node = x - h * n, head = (int)h0 + h;
            to[i] = -1;
            if (h >= each || head >= heads || s_from[node] < 0) continue;
            const int layer = head / c.kv_heads;
            const int64_t at = ((int64_t)layer * c.pages * c.kv_heads + (head - layer * c.kv_heads)) * c.page * 16 + (t & 15);
            to[i] = s_to[node] + at;
            kv[i][0] = static_cast<const uint4*>(c.k)[s_from[node] + at];
            kv[i][1] = static_cast<const uint4*>(c.v)[s_from[node] + at];
        }
        float* sums = nullptr;   // of the head that this thread moves a sum of; positions have one whether they have a page or not
        float sum = 0.f;
        if constexpr (WEIGH) {
            if (t < each * n && h0 + t / n < heads) {
                const int64_t head = h0 + t / n, layer = head / c.kv_heads;
                const int node = t % n;
                float* base = weights + ((layer * c.rows + r) * c.kv_heads + (head - layer * c.kv_heads)) * cap + len;
                if (s_path[node] != node && len + s_path[node] < cap) {   // a node of a branch is never before its place
                    sum = __ldcg(base + s_path[node]);
                    sums = base + node;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (to[i] >= 0) {
                static_cast<uint4*>(c.k)[to[i]] = kv[i][0];
                static_cast<uint4*>(c.v)[to[i]] = kv[i][1];
            }
        if constexpr (WEIGH)
            if (sums) *sums = sum;
    }
}

// The new lengths, where they take the place of the old ones, which all of accept_kernel's CTAs read.
__global__ void __launch_bounds__(1024) accept_lens_kernel(mfqb_cache c, const int* count, int* lens_out) {
    chained_wait();
    const int r = threadIdx.x;
    int len = 0;
    if (r < c.rows) len = (int)min(max((int64_t)c.lens[r], (int64_t)0), (int64_t)c.width * c.page) + __ldcg(count + r);
    __syncthreads();
    if (r < c.rows) lens_out[r] = len;
}

static void accept(const mfqb_cache* c, const int32_t* ids, const int32_t* parents, const int32_t* targets, int nodes, int32_t* count, int32_t* token,
                   int32_t* path, int32_t* lens_out, float* weights, cudaStream_t s, const char* who) {
    check_cache(c, who);
    check_nodes(c, nodes, who);
    if (!ids || !parents || !targets || !count || !token || !path || !lens_out) fail(MFQB_ERR_ARG, "%s: null argument", who);
    if ((int64_t)c->layers * c->kv_heads > (1ll << 30)) fail(MFQB_ERR_UNSUPPORTED, "%s: too many layers x heads", who);
    // enough CTAs for the SMs, at least one head each (how many nodes a branch has is known on the device alone)
    const int per_row = std::min(c->layers * c->kv_heads, std::max(1, 148 * 5 / c->rows));
    const bool in_place = lens_out < c->lens + c->rows && c->lens < lens_out + c->rows;
    launch_chained(weights ? accept_kernel<true> : accept_kernel<false>, dim3((unsigned)per_row, c->rows), dim3(256), 0, s, *c, ids, parents, targets, nodes, count, token, path,
                   in_place ? nullptr : lens_out, weights);
    if (in_place) launch_chained(accept_lens_kernel, dim3(1), dim3(1024), 0, s, *c, static_cast<const int*>(count), lens_out);
}

}  // namespace mfqb

using namespace mfqb;

extern "C" {
#pragma GCC visibility push(default)

int mfqb_cache_extend(const mfqb_cache* c, const int32_t* tokens, int32_t* status, mfqb_stream_t stream) {
    return guarded([&] {
        check_cache(c, "mfqb_cache_extend");
        if (!tokens || !status) fail(MFQB_ERR_ARG, "mfqb_cache_extend: null argument");
        launch_chained(extend_kernel, dim3(1), dim3(1024), 0, stream, *c, tokens, status);
    });
}

int mfqb_cache_fork_work(const mfqb_cache* c, uint64_t* bytes) {
    return guarded([&] {
        check_cache(c, "mfqb_cache_fork_work");
        if (!bytes) fail(MFQB_ERR_ARG, "mfqb_cache_fork_work: null argument");
        ready_device();
        *bytes = fork_work_bytes(*c);
    });
}

int mfqb_cache_fork(const mfqb_cache* c, const int32_t* parents, int32_t* status, void* work, uint64_t work_bytes, mfqb_stream_t stream) {
    return guarded([&] {
        check_cache(c, "mfqb_cache_fork");
        if (!parents || !status || !work) fail(MFQB_ERR_ARG, "mfqb_cache_fork: null argument");
        if (((uintptr_t)work & 15) || work_bytes < fork_work_bytes(*c))
            fail(MFQB_ERR_ARG, "mfqb_cache_fork: work must be 16-byte aligned and hold %llu bytes, got %llu", (unsigned long long)fork_work_bytes(*c), (unsigned long long)work_bytes);
        const ForkWork w = fork_work(*c, work);
        const int64_t ints = (int64_t)c->pages + (int64_t)c->rows * c->width;
        const bool small = ints <= kForkSmall;   // with the kernel's other arrays below the 48 KB that need no attribute
        launch_chained(fork_plan_kernel, dim3(1), dim3(1024), small ? (size_t)ints * 4 : 0, stream, *c, parents, status, w, small);
        const int64_t most = (int64_t)c->rows * c->layers * c->kv_heads * 2;   // stretches, if every sequence got a copy
        launch_chained(fork_copy_kernel, dim3((unsigned)std::min<int64_t>(most, 148 * 8)), dim3(256), 0, stream, *c, w);
    });
}

int mfqb_tree_masks(const int32_t* parents, int rows, int nodes, uint64_t* masks, int32_t* depths, mfqb_stream_t stream) {
    return guarded([&] {
        if (!parents || !masks || !depths) fail(MFQB_ERR_ARG, "mfqb_tree_masks: null argument");
        if (rows < 1 || rows > kCacheRows) fail(MFQB_ERR_UNSUPPORTED, "mfqb_tree_masks: 1 to %d sequences, got %d", kCacheRows, rows);
        if ((uintptr_t)masks & 7) fail(MFQB_ERR_ARG, "mfqb_tree_masks: masks must be 8-byte aligned");
        if (nodes < 1 || nodes > kTreeNodes) fail(MFQB_ERR_UNSUPPORTED, "mfqb_tree_masks: 1 to %d nodes per sequence, got %d", kTreeNodes, nodes);
        launch_chained(tree_masks_kernel, dim3(rows), dim3(32), 0, stream, parents, nodes, reinterpret_cast<unsigned long long*>(masks), depths);
    });
}

int mfqb_cache_write(const mfqb_cache* c, int layer, const float* qkv, int q_heads, int nodes, const int32_t* depths, const double* freqs,
                     void* q_out, mfqb_stream_t stream) {
    return guarded([&] {
        check_cache(c, "mfqb_cache_write");
        check_nodes(c, nodes, "mfqb_cache_write");
        if (!qkv || !depths || !freqs || !q_out) fail(MFQB_ERR_ARG, "mfqb_cache_write: null argument");
        if (((uintptr_t)qkv & 15) || ((uintptr_t)q_out & 15)) fail(MFQB_ERR_ARG, "mfqb_cache_write: qkv and q_out must be 16-byte aligned");
        if ((uintptr_t)freqs & 7) fail(MFQB_ERR_ARG, "mfqb_cache_write: freqs must be 8-byte aligned");
        if (layer < 0 || layer >= c->layers) fail(MFQB_ERR_ARG, "mfqb_cache_write: layer %d of %d", layer, c->layers);
        if (q_heads < 1 || q_heads > 16384) fail(MFQB_ERR_ARG, "mfqb_cache_write: bad number of query heads %d", q_heads);
        const uint64_t tokens = (uint64_t)c->rows * nodes;   // a head's queries are written elsewhere than they are read, while other CTAs read
        check_apart(q_out, 256 * tokens * q_heads, qkv, 512 * tokens * (q_heads + 2 * c->kv_heads), "mfqb_cache_write", "qkv and q_out");
        // one CTA per token once there are CTAs for every SM, else its heads spread over more of them
        const int parts = c->rows * nodes >= 148 ? 1 : (q_heads + 2 * c->kv_heads + 15) / 16;
        launch_chained(cache_write_kernel, dim3(parts, nodes, c->rows), dim3(256), 0, stream, *c, layer, qkv, q_heads, nodes, depths, freqs,
                       static_cast<__nv_bfloat16*>(q_out));
    });
}

int mfqb_cache_write_rope(const mfqb_cache* c, int layer, const void* qkv, int qkv_dtype, int q_heads, int nodes, const int32_t* depths, const double* freqs, int pairs,
                          int layout, float factor, void* q_out, mfqb_stream_t stream) {
    return guarded([&] {
        const char* who = "mfqb_cache_write_rope";
        check_cache(c, who);
        check_nodes(c, nodes, who);
        if (!qkv || !depths || !freqs || !q_out) fail(MFQB_ERR_ARG, "%s: null argument", who);
        if (qkv_dtype != MFQB_F32 && qkv_dtype != MFQB_BF16) fail(MFQB_ERR_ARG, "%s: bad type of qkv %d", who, qkv_dtype);
        if (((uintptr_t)qkv & 15) || ((uintptr_t)q_out & 15)) fail(MFQB_ERR_ARG, "%s: qkv and q_out must be 16-byte aligned", who);
        if ((uintptr_t)freqs & 7) fail(MFQB_ERR_ARG, "%s: freqs must be 8-byte aligned", who);
        if (layer < 0 || layer >= c->layers) fail(MFQB_ERR_ARG, "%s: layer %d of %d", who, layer, c->layers);
        if (q_heads < 1 || q_heads > 16384) fail(MFQB_ERR_ARG, "%s: bad number of query heads %d", who, q_heads);
        if (pairs < 1 || pairs > kHeadDim / 2) fail(MFQB_ERR_UNSUPPORTED, "%s: 1 to %d pairs of dims, got %d", who, kHeadDim / 2, pairs);
        if (layout != MFQB_ROPE_HALVES && layout != MFQB_ROPE_INTERLEAVED) fail(MFQB_ERR_ARG, "%s: bad layout %d", who, layout);
        if (!(factor > 0.f) || factor > 1e30f) fail(MFQB_ERR_ARG, "%s: factor must be positive and finite", who);
        const uint64_t tokens = (uint64_t)c->rows * nodes, size = qkv_dtype == MFQB_F32 ? 4 : 2;
        check_apart(q_out, 256 * tokens * q_heads, qkv, size * kHeadDim * tokens * (q_heads + 2 * c->kv_heads), who, "qkv and q_out");
        if (qkv_dtype == MFQB_F32) launch_cache_rope<float>(*c, layer, qkv, q_heads, nodes, depths, freqs, pairs, layout, factor, q_out, stream);
        else launch_cache_rope<__nv_bfloat16>(*c, layer, qkv, q_heads, nodes, depths, freqs, pairs, layout, factor, q_out, stream);
    });
}

int mfqb_tree_accept(const mfqb_cache* c, const int32_t* ids, const int32_t* parents, const int32_t* targets, int nodes, int32_t* count,
                     int32_t* token, int32_t* path, int32_t* lens_out, mfqb_stream_t stream) {
    return guarded([&] { accept(c, ids, parents, targets, nodes, count, token, path, lens_out, nullptr, stream, "mfqb_tree_accept"); });
}

int mfqb_tree_accept_weigh(const mfqb_cache* c, const int32_t* ids, const int32_t* parents, const int32_t* targets, int nodes, int32_t* count,
                           int32_t* token, int32_t* path, int32_t* lens_out, float* weights, mfqb_stream_t stream) {
    return guarded([&] {
        const char* who = "mfqb_tree_accept_weigh";
        if (!weights || ((uintptr_t)weights & 3)) fail(MFQB_ERR_ARG, "%s: weights must be float32 values on 4-byte boundaries", who);
        accept(c, ids, parents, targets, nodes, count, token, path, lens_out, weights, stream, who);
    });
}

#pragma GCC visibility pop
}  // extern "C"
