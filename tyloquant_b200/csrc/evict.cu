// Eviction from a paged cache: every head of every layer keeps the positions with the largest weights and the latest ones; their keys and
// values close up, and the pages behind them go back.
#include <mutex>
#include <type_traits>

#include "select.cuh"

namespace mfqb {

constexpr int kEvictThreads = 256, kEvictWarps = kEvictThreads / 32;
constexpr int kEvictStep = 8 * kEvictThreads;          // slots that are looked at together, and room for as many as are found
constexpr int kEvictCached = 48 * 1024;                // positions whose keys fit shared memory

struct EvictRow {
    int len, keep;   // keep -1: the sequence stays as it is
    int swapped;     // some of its first pages have been exchanged for others
    int pad;
};
struct EvictWork {
    EvictRow* row;   // [rows]
    int* old;        // [rows][width]: the table as it was
    int* rank;       // [rows][width]: which of the new pages an entry gets, -1 none
    int* free;       // [pages]
};
static EvictWork evict_work(const mfqb_cache& c, void* work) {
    const int64_t entries = (int64_t)c.rows * c.width;
    EvictWork w;
    w.row = static_cast<EvictRow*>(work);
    w.old = reinterpret_cast<int*>(w.row + c.rows);
    w.rank = w.old + entries;
    w.free = w.rank + entries;
    return w;
}
static uint64_t evict_work_bytes(const mfqb_cache& c) { return 16ull * c.rows + 8ull * c.rows * c.width + 4ull * c.pages; }

// One CTA.  Which entries change is settled from the counts as they were: a page that two sequences have is exchanged in both, so that no
// page is written that another one still reads from, and the new pages are among those that were free before.
__global__ void __launch_bounds__(1024) evict_plan_kernel(mfqb_cache c, const int* keep, int* dropped, int* status, EvictWork w) {
    chained_wait();
    __shared__ int sums[33], s_keep[kCacheRows], s_swapped[kCacheRows];
    const int r = threadIdx.x;
    const int64_t cap = (int64_t)c.width * c.page;
    int len = 0, to = -1;
    if (r < c.rows) {
        len = (int)min(max((int64_t)c.lens[r], (int64_t)0), cap);
        to = __ldcg(keep + r);
        if (to >= len) to = -1;
        to = max(to, -1);
    }
    s_keep[r] = to;
    s_swapped[r] = 0;
    __syncthreads();
    auto valid = [&](int p) { return (unsigned)p < (unsigned)c.pages; };
    const int entries = c.rows * c.width;
    int need = 0;
    for (int base = 0; base < entries; base += 1024) {
        const int e = base + r;
        int swap = 0, row = 0;
        if (e < entries) {
            row = e / c.width;
            const int p = c.table[e];
            w.old[e] = p;
            swap = (int64_t)(e - row * c.width) * c.page < s_keep[row] && valid(p) && c.refs[p] > 1;
        }
        const int upto = block_scan<1024>(swap, sums);
        if (e < entries) w.rank[e] = swap ? need + upto - 1 : -1;
        if (swap) s_swapped[row] = 1;
        __syncthreads();
        need += sums[32];
    }
    int have = 0;
    if (need > 0) {   // the lowest free pages, in order
        for (int base = 0; base < c.pages && have < need; base += 1024) {
            const int p = base + r;
            const int is = p < c.pages && c.refs[p] <= 0;
            const int upto = block_scan<1024>(is, sums);
            if (is && have + upto <= need) w.free[have + upto - 1] = p;
            __syncthreads();
            have += sums[32];
        }
        have = min(have, need);
    }
    const bool go = have == need;
    if (r == 0) *status = need - have;
    if (r < c.rows) {
        if (!go) to = -1;
        w.row[r] = EvictRow{len, to, s_swapped[r], 0};
        dropped[r] = to < 0 ? 0 : len - to;
        if (to >= 0) c.lens[r] = to;
    }
    __syncthreads();
    if (!go) return;
    for (int e = r; e < entries; e += 1024) {
        const int row = e / c.width, k = s_keep[row];
        if (k < 0) continue;
        const int p = w.old[e], at = w.rank[e];
        if ((int64_t)(e - row * c.width) * c.page >= k) {
            c.table[e] = -1;
            if (valid(p)) atomicSub(c.refs + p, 1);
        } else if (at >= 0) {
            const int fresh = w.free[at];
            c.table[e] = fresh;
            c.refs[fresh] = 1;   // whatever a free page's count was
            atomicSub(c.refs + p, 1);
        }
    }
}

template <typename Slot>
struct EvictShared {
    union {   // the search for the cut, then what is to be moved
        CutShared cut;
        struct {
            Slot holes[kEvictStep], movers[kEvictStep];
        };
    };
    int sums[kEvictWarps + 1];
};

// Bound by memory where much moves (4096 positions cut to 2048 in 32 layers x 8 heads: 68 us for 253 MB read and written, of which the search takes 10), by
// instructions and trips where little does (16 sequences of 2112 cut to 2048, 6 layers: 34 us for 97 MB, of which the search is half).
// Four CTAs of 256 threads on an SM: three, with more registers, took 97 us in the first case.
// Keys take four bytes of shared memory for each position that the table can hold, whatever the lengths: the second case takes 27 us (kernel alone, behind the plan) in a table of
// 2112 positions, 29 in one of 8192, 35 of 16384, 69 of 32768, and 48 of 65536, where keys come from the weights themselves.  The latest rows go through one CTA, 64 at a time,
// where they are more than those that go: 16 sequences of 2049 cut to 2048, 6 layers: 15 us for none, 19 for 64, 90 for 512, 310 for 2048.
//
// A cluster per head of a layer of a sequence.  Each of its CTAs finds the cut and the same lists of free slots and of rows to move, and moves its
// share; the latest rows follow when all others have moved.  Rows are read before a slot that holds one is written: the others go to
// slots below the new length's older part, where none of them lies, and the latest ones in ascending order.
template <bool CACHED>
__global__ void __launch_bounds__(kEvictThreads, 4) evict_kernel(mfqb_cache c, float* weights, int recent_most, EvictWork w) {
    extern __shared__ uint4 s_keys[];   // four slots each; 0, which no value has, behind the last one
    using Slot = typename std::conditional<CACHED, unsigned short, int>::type;
    static_assert(!CACHED || kEvictCached <= 65536, "a slot in 16 bits");
    __shared__ EvictShared<Slot> sh;
    chained_wait();
    unsigned part, parts;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
    const int layer = blockIdx.z, r = blockIdx.y, head = blockIdx.x / parts, tid = threadIdx.x;
    const int64_t unit = ((int64_t)layer * c.rows + r) * c.kv_heads + head;
    const EvictRow row = w.row[r];
    if (row.keep < 0) return;   // the whole cluster
    const int n = row.len, k = row.keep, recent = min(recent_most, k), older = n - recent, b = k - recent;   // of `older` slots b stay, the first b of the new ones
    const int bits = __ffs(c.page) - 1, low = c.page - 1;
    const int *old_table = w.old + (int64_t)r * c.width, *table = c.table + (int64_t)r * c.width;
    float* wt = weights + unit * c.width * c.page;
    constexpr int kTeams = kEvictThreads / 16;   // a row is 16 threads'
    const int lane = tid & 15, team = tid >> 4, stride = c.kv_heads * c.page;
    uint4* const kp = static_cast<uint4*>(c.k) + ((int64_t)layer * c.pages * c.kv_heads + head) * c.page * 16 + lane;   // this thread's part of row 0 of page 0
    uint4* const vp = static_cast<uint4*>(c.v) + ((int64_t)layer * c.pages * c.kv_heads + head) * c.page * 16 + lane;
    auto at = [&](const int* t, int slot) -> int64_t {   // of a slot, -1 without a page
        const int p = t[slot >> bits];
        return (unsigned)p < (unsigned)c.pages ? ((int64_t)p * stride + (slot & low)) * 16 : -1;
    };
    auto read = [&](int i) {   // keys of slots 4i ..
        const float4 x = __ldcg(reinterpret_cast<const float4*>(wt) + i);
        return make_uint4(ordered_f32(x.x), 4 * i + 1 < older ? ordered_f32(x.y) : 0u, 4 * i + 2 < older ? ordered_f32(x.z) : 0u, 4 * i + 3 < older ? ordered_f32(x.w) : 0u);
    };
    auto keys = [&](int i) { return CACHED ? s_keys[i] : read(i); };
    auto sync_all = [&]() {
        __syncwarp();   // the aligned form wants the warp together: lanes have read different numbers of keys
        if (parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else __syncthreads();
    };
    if (b > 0) {
        const int fours = (older + 3) / 4;
        unsigned low = 0xFFFFFFFFu, high = 0u, above = 0xFFFFFFFFu;
#pragma unroll 2
        for (int i = tid; i < fours; i += kEvictThreads) {
            const uint4 k = read(i);
            if (CACHED) s_keys[i] = k;
            low = min(min(low, k.x - 1u), min(k.y - 1u, min(k.z - 1u, k.w - 1u)));   // less 1, so that none is the largest
            high = max(max(high, k.x), max(k.y, max(k.z, k.w)));
            above = min(min(above, k.x - kCutZero - 1u), min(k.y - kCutZero - 1u, min(k.z - kCutZero - 1u, k.w - kCutZero - 1u)));   // what is not above zero wraps
        }
        if (low != 0xFFFFFFFFu) ++low;
        above = above < kCutZero - 1u ? above + kCutZero + 1u : 0xFFFFFFFFu;
        if (CACHED) sync_all();   // no CTA moves weights that another one has not read
        const Cut cut = select_cut<kEvictThreads>(b, low, high, above, older, sh.cut, [&](auto f) {
#pragma unroll 2
            for (int i = tid; i < fours; i += kEvictThreads) {
                const uint4 k = keys(i);
                f(k.x, 4 * i); f(k.y, 4 * i + 1); f(k.z, 4 * i + 2); f(k.w, 4 * i + 3);
            }
        });
        // Walks slots [slot, end) until it has found some that `take` wants (stays: is the slot kept?), in ascending order; a step whose finds have no room
        // beside the ones before it is walked again.
        struct Walk {
            int slot, end, n, used;
        };
        auto fill = [&](Walk& x, Slot* list, auto take) {
            x.n = x.used = 0;
            while (x.slot < x.end) {
                const int i0 = (x.slot & ~7) + 8 * tid;
                unsigned found = 0;
                if (i0 < x.end) {
                    const uint4 k = keys(i0 >> 2), l = i0 + 4 < x.end ? keys((i0 >> 2) + 1) : make_uint4(0u, 0u, 0u, 0u);
                    const unsigned o[8] = {k.x, k.y, k.z, k.w, l.x, l.y, l.z, l.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (i0 + e >= x.slot && i0 + e < x.end && take(cut.in(o[e], i0 + e), i0 + e)) found |= 1u << e;
                }
                const int want = __popc(found), upto = block_scan<kEvictThreads>(want, sh.sums);
                __syncthreads();
                const int more = sh.sums[kEvictWarps];
                if (x.n + more > kEvictStep) break;
                int to = x.n + upto - want;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((found >> e) & 1u) list[to++] = (Slot)(i0 + e);
                x.n += more;
                x.slot = min(x.end, (x.slot & ~7) + kEvictStep);
            }
            __syncthreads();
        };
        // Moves `count` rows, 16 threads each; the CTAs of the cluster take them in turns.
        auto move = [&](const Slot* from, const Slot* to, int count) {
            for (int i0 = (int)part * kTeams + team; i0 < count; i0 += (int)parts * kTeams * 4) {
                uint4 a[4], v[4];
                unsigned there = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int i = i0 + u * (int)parts * kTeams;
                    if (i >= count) continue;
                    const int64_t src = at(old_table, from[i]);
                    if (src >= 0) {
                        there |= 1u << u;
                        a[u] = kp[src];
                        v[u] = vp[src];
                    }
                    if (lane == 0 && from[i] != to[i]) wt[to[i]] = wt[from[i]];
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (!((there >> u) & 1u)) continue;
                    const int64_t dst = at(table, to[i0 + u * (int)parts * kTeams]);
                    if (dst >= 0) {
                        kp[dst] = a[u];
                        vp[dst] = v[u];
                    }
                }
            }
        };
        if (row.swapped) {   // what stays in its slot on a page that has been exchanged
            Walk x = {0, b, 0, 0};
            for (;;) {
                fill(x, sh.holes, [&](bool stays, int slot) { return stays && old_table[slot >> bits] != table[slot >> bits]; });
                if (x.n == 0) break;
                move(sh.holes, sh.holes, x.n);
                __syncthreads();
            }
        }
        Walk hole = {0, b, 0, 0}, mover = {b, older, 0, 0};
        for (;;) {
            if (hole.used == hole.n) fill(hole, sh.holes, [](bool stays, int) { return !stays; });
            if (hole.n == 0) break;
            if (mover.used == mover.n) fill(mover, sh.movers, [](bool stays, int) { return stays; });
            const int count = min(hole.n - hole.used, mover.n - mover.used);   // as many rows move as there are free slots
            if (count <= 0) break;
            move(sh.movers + mover.used, sh.holes + hole.used, count);
            hole.used += count;
            mover.used += count;
            __syncthreads();
        }
    }
    sync_all();
    // The latest rows: a CTA reads a batch before it writes any of it, and later ones lie behind all that has been written.  Where they are fewer than
    // those that go, no place is another one's source, and the CTAs share them.
    const bool apart = n - k >= recent;
    if (apart || part == 0) {
        constexpr int kBatch = 4 * kTeams;
        for (int i0 = apart ? (int)part * kBatch : 0; i0 < recent; i0 += apart ? (int)parts * kBatch : kBatch) {
            uint4 a[4], v[4];
            float f[4];
            unsigned there = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kTeams + team;
                if (i >= recent) continue;
                const int64_t src = at(old_table, older + i);
                if (src >= 0) {
                    there |= 1u << u;
                    a[u] = kp[src];
                    v[u] = vp[src];
                }
                f[u] = wt[older + i];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kTeams + team;
                if (i >= recent) continue;
                if ((there >> u) & 1u) {
                    const int64_t dst = at(table, b + i);
                    if (dst >= 0) {
                        kp[dst] = a[u];
                        vp[dst] = v[u];
                    }
                }
                if (lane == 0) wt[b + i] = f[u];
            }
        }
    }
}

static void launch_evict(const mfqb_cache& c, float* weights, const int* keep, int recent, int* dropped, int* status, EvictWork w, cudaStream_t s) {
    int device = 0;
    MFQB_CUDA(cudaGetDevice(&device));
    static std::once_flag once[64];
    std::call_once(once[device], [] { MFQB_CUDA(cudaFuncSetAttribute(evict_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictCached * 4)); });
    launch_chained(evict_plan_kernel, dim3(1), dim3(1024), 0, s, c, keep, dropped, status, w);
    const int64_t cap = (int64_t)c.width * c.page, units = (int64_t)c.layers * c.rows * c.kv_heads;
    const bool cached = cap <= kEvictCached;
    // CTAs of a head: until there are two for every SM (four: 83 in place of 73 us in the first case above, each repeats the search).  Keys that are read from the
    // weights themselves may not be read by one CTA while another one moves weights.
    int parts = 1;
    while (cached && parts < 8 && units * parts < 2 * 148) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(c.kv_heads * parts), c.rows, c.layers);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = cached ? (size_t)cap * 4 : 0;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    MFQB_CUDA(cudaLaunchKernelEx(&cfg, cached ? evict_kernel<true> : evict_kernel<false>, c, weights, recent, w));
}

}  // namespace mfqb

using namespace mfqb;

extern "C" {
#pragma GCC visibility push(default)

int mfqb_cache_evict_work(const mfqb_cache* c, uint64_t* bytes) {
    return guarded([&] {
        check_cache(c, "mfqb_cache_evict_work");
        if (!bytes) fail(MFQB_ERR_ARG, "mfqb_cache_evict_work: null argument");
        ready_device();
        *bytes = evict_work_bytes(*c);
    });
}

int mfqb_cache_evict(const mfqb_cache* c, float* weights, const int32_t* keep, int recent, int32_t* dropped, int32_t* status, void* work, uint64_t work_bytes,
                     mfqb_stream_t stream) {
    return guarded([&] {
        check_cache(c, "mfqb_cache_evict");
        if (!weights || !keep || !dropped || !status || !work) fail(MFQB_ERR_ARG, "mfqb_cache_evict: null argument");
        if ((uintptr_t)weights & 15) fail(MFQB_ERR_ARG, "mfqb_cache_evict: weights must be 16-byte aligned");
        if (recent < 0) fail(MFQB_ERR_ARG, "mfqb_cache_evict: the number of latest positions must not be negative, got %d", recent);
        if (c->layers > 65535) fail(MFQB_ERR_UNSUPPORTED, "mfqb_cache_evict: at most 65535 layers, got %d", c->layers);
        if (((uintptr_t)work & 15) || work_bytes < evict_work_bytes(*c))
            fail(MFQB_ERR_ARG, "mfqb_cache_evict: work must be 16-byte aligned and hold %llu bytes, got %llu", (unsigned long long)evict_work_bytes(*c),
                 (unsigned long long)work_bytes);
        launch_evict(*c, weights, keep, recent, dropped, status, evict_work(*c, work), stream);
    });
}

#pragma GCC visibility pop
}  // extern "C"
