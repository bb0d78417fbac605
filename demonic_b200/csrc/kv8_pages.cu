// kv8_pages.cu -- pages of the 8-bit KV cache: reserving (with copy-on-write), forking, releasing, compacting, copying.
//
// The bookkeeping (who holds which page, which are free) lives on the device and is changed there, so that a decode
// loop with all its page traffic can be one captured graph.  It is a few thousand integers with steps that depend on one
// another: one CTA (reserve) or one cluster of 8 CTAs whose steps are separated by cluster barriers, never the whole
// device.  What moves bytes is one copy kernel over a list of (source, destination) that the bookkeeping leaves in the
// scratch area: 250 pages of 8 layers, 262 MB both ways, in 43 us = 6.1 TB/s (0.93 of a plain copy's rate).  The bookkeeping is
// bound by latency, barriers the longest stall by far: fork 7 us (56 slots), reserve 9 (64 slots), compact 11 (1000 pages).
#include <cooperative_groups.h>

#include <algorithm>

#include "gemv.cuh"
#include "kv8_host.h"

namespace cg = cooperative_groups;

namespace dmc {
namespace {

constexpr int kThreads = 1024, kCluster = 8;
constexpr int kHeader = 16;            // ints before the lists in the scratch area; [0]: copies in the list, [1]: its first source
constexpr int kReserveBatch = 4096;

struct PageArgs {
    int *table, *lens, *refs, *free_list, *free_count, *flags;
    int *scratch;  // header | src [pages] | dst [pages] | map [pages]
    long long table_stride;
    int slots, pages, page_tokens, cap;
    const int *ids, *ids2;  // slot ids / counts; fork: src, dst
    int *moved;
    int count, tokens;
};
__device__ __forceinline__ int *list_src(const PageArgs &a) { return a.scratch + kHeader; }
__device__ __forceinline__ int *list_dst(const PageArgs &a) { return a.scratch + kHeader + a.pages; }
__device__ __forceinline__ int *page_map(const PageArgs &a) { return a.scratch + kHeader + 2 * a.pages; }
__device__ __forceinline__ int held_pages(const PageArgs &a, int len) {
    return min(max(len, 0), a.cap) / a.page_tokens + (min(max(len, 0), a.cap) % a.page_tokens != 0);
}

// Exclusive sum over the CTA's 1024 threads; *total gets the sum.  Ends with a barrier.
__device__ __forceinline__ int block_scan(int v, int *total) {
    __shared__ int ws[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) ws[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int w = ws[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += up;
        }
        ws[lane] = w;
    }
    __syncthreads();
    const int before = warp ? ws[warp - 1] : 0;
    *total = ws[31];
    __syncthreads();
    return before + inc - v;
}

// ---- reserve ---------------------------------------------------------------------------------------------------
// Rows in order: a row asks for a copy of its last page (if new tokens go into it and others hold it too), then for new
// pages.  Request i takes free_list[count - 1 - i].  Nothing is changed before all requests are known to fit.
struct ReserveSmem {
    int slot[kReserveBatch], last[kReserveBatch], have[kReserveBatch], len[kReserveBatch], start[kReserveBatch];
    unsigned seen[kKv8MaxSlots / 32];
};

__global__ void __launch_bounds__(kThreads) kv8_reserve_kernel(PageArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    ReserveSmem &sm = *reinterpret_cast<ReserveSmem *>(raw);
    __shared__ int bad, copies;
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, fc = *a.free_count;
    for (int i = tid; i < kKv8MaxSlots / 32; i += kThreads) sm.seen[i] = 0;
    if (tid == 0) bad = copies = 0;
    __syncthreads();
    constexpr int R = kReserveBatch / kThreads;
    int want[R], held_by[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int b = r * kThreads + tid;
        want[r] = held_by[r] = 0;
        if (b >= a.count) continue;
        int s = a.ids ? a.ids[b] : b, last = -1, have = 0, len = 0;
        if (s < -1 || s >= a.slots) {
            atomicOr(&bad, DMC_KV8_BAD_SLOT);
            s = -1;
        }
        if (s >= 0) {
            if (atomicOr(&sm.seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) atomicOr(&bad, DMC_KV8_BAD_SLOT);
            const int old = max(a.lens[s], 0), n = max(a.ids2 ? a.ids2[b] : a.tokens, 0);
            if (old > a.cap || n > a.cap - old) {
                atomicOr(&bad, DMC_KV8_TOO_LONG);
            } else {
                len = old + n;
                have = held_pages(a, old);
                want[r] = held_pages(a, len) - have;
                if (n > 0 && old % a.page_tokens) {
                    const int p = a.table[(size_t)s * a.table_stride + have - 1];
                    if ((unsigned)p >= (unsigned)a.pages) atomicOr(&bad, DMC_KV8_BAD_PAGE);
                    else if ((held_by[r] = a.refs[p]) > 1) last = p;
                }
            }
        }
        sm.slot[b] = s;
        sm.last[b] = last;
        sm.have[b] = have;
        sm.len[b] = len;
    }
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r * kThreads >= a.count) break;
        const int b = r * kThreads + tid;
        int copy = 0;
        if (b < a.count && sm.last[b] >= 0) {
            int same = 0, later = 0;
            for (int i = 0; i < a.count; ++i) {
                const int eq = sm.last[i] == sm.last[b];
                same += eq;
                later |= eq & (i > b);
            }
            copy = same < held_by[r] || later;  // the last of a page's holders keeps it
        }
        int total;
        const int at = block_scan(b < a.count ? want[r] + copy : 0, &total);
        if (b < a.count) sm.start[b] = base + at;
        base += total;
        want[r] = copy;  // (all that is still needed of it)
    }
    if (tid == 0 && !bad && (base > fc || fc > a.pages)) bad = DMC_KV8_NO_PAGES;
    __syncthreads();
    if (bad) {
        if (tid == 0) {
            atomicOr(a.flags, bad);
            a.scratch[0] = a.scratch[1] = 0;
        }
        return;
    }
    // (the requests are read before the last pages are struck from the rows that copy them)
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int b = r * kThreads + tid;
        if (b < a.count) {
            if (!want[r]) sm.last[b] = -1;
            if (sm.slot[b] >= 0) a.lens[sm.slot[b]] = sm.len[b];
        }
    }
    __syncthreads();
    for (int i = tid; i < base; i += kThreads) {
        int lo = 0, hi = a.count - 1;  // the last row with start <= i
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sm.start[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        const int page = a.free_list[fc - 1 - i], j = i - sm.start[lo], copy = sm.last[lo] >= 0;
        if ((unsigned)page >= (unsigned)a.pages) {  // a damaged stack
            atomicOr(a.flags, DMC_KV8_BAD_PAGE);
            continue;
        }
        int *row = a.table + (size_t)sm.slot[lo] * a.table_stride + sm.have[lo];
        if (copy && j == 0) {
            const int n = atomicAdd(&copies, 1);
            list_src(a)[n] = sm.last[lo];
            list_dst(a)[n] = page;
            atomicSub(&a.refs[sm.last[lo]], 1);
            row[-1] = page;
        } else {
            row[j - copy] = page;
        }
        a.refs[page] = 1;
    }
    __syncthreads();
    if (tid == 0) {
        *a.free_count = fc - base;
        a.scratch[0] = copies;
        a.scratch[1] = 0;
    }
}

// ---- fork, release, compact: one cluster --------------------------------------------------------------------------

// first[s]: the first place in ids that names slot s (each CTA has its own copy).
__device__ __forceinline__ void first_namings(const PageArgs &a, const int *ids, int *first) {
    for (int i = threadIdx.x; i < a.slots; i += kThreads) first[i] = INT32_MAX;
    __syncthreads();
    for (int i = threadIdx.x; i < a.count; i += kThreads) {
        const int s = ids[i];
        if (s >= 0 && s < a.slots) atomicMin(&first[s], i);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) kv8_fork_kernel(PageArgs a) {
    extern __shared__ __align__(16) int first[];
    cg::cluster_group cl = cg::this_cluster();
    griddep_launch_dependents();
    griddep_wait();
    first_namings(a, a.ids2, first);
    const int gid = blockIdx.x * kThreads + threadIdx.x;
    auto valid = [&](int i, int *src, int *dst) {
        *src = a.ids[i];
        *dst = a.ids2[i];
        return *src >= 0 && *src < a.slots && *dst >= 0 && *dst < a.slots && first[*dst] == i && a.lens[*dst] <= 0;
    };
    int src = 0, dst = 0, len = 0;
    bool mine = false;
    if (gid < a.count) {
        mine = valid(gid, &src, &dst);
        if (mine) len = a.lens[src];
        if (mine && len > a.cap) {
            atomicOr(a.flags, DMC_KV8_TOO_LONG);
            mine = false;
        } else if (!mine && (dst != -1 || src < -1 || src >= a.slots)) {
            atomicOr(a.flags, DMC_KV8_BAD_SLOT);
        }
    }
    const long long entries = (long long)a.count * a.table_stride;
    for (long long e = gid; e < entries; e += kCluster * kThreads) {
        int s, d;
        const int col = (int)(e % a.table_stride);
        if (!valid((int)(e / a.table_stride), &s, &d)) continue;
        const int n = a.lens[s];
        if (n > a.cap || col >= held_pages(a, n)) continue;
        const int p = a.table[(size_t)s * a.table_stride + col];
        a.table[(size_t)d * a.table_stride + col] = p;
        if ((unsigned)p < (unsigned)a.pages) atomicAdd(&a.refs[p], 1);
        else atomicOr(a.flags, DMC_KV8_BAD_PAGE);
    }
    cl.sync();  // every length has been read
    if (mine) a.lens[dst] = len;
}

__global__ void __launch_bounds__(kThreads) kv8_release_kernel(PageArgs a) {
    extern __shared__ __align__(16) int first[];
    __shared__ int counts[kCluster];
    cg::cluster_group cl = cg::this_cluster();
    griddep_launch_dependents();
    griddep_wait();
    first_namings(a, a.ids, first);
    int *claim = page_map(a);
    const long long entries = (long long)a.count * a.table_stride;  // (below 2^31)
    const int rank = blockIdx.x;
    const long long e0 = entries * rank / kCluster, e1 = entries * (rank + 1) / kCluster;
    auto page_at = [&](long long e) -> int {  // page that entry e gives back, or -1
        const int i = (int)(e / a.table_stride), s = a.ids[i];
        if (s < 0 || s >= a.slots || first[s] != i) return -1;
        const int n = a.lens[s];
        if (n > a.cap || (int)(e % a.table_stride) >= held_pages(a, n)) return -1;
        const int p = a.table[(size_t)s * a.table_stride + e % a.table_stride];
        if ((unsigned)p < (unsigned)a.pages) return p;
        atomicOr(a.flags, DMC_KV8_BAD_PAGE);
        return -1;
    };
    for (int i = rank * kThreads + threadIdx.x; i < a.count; i += kCluster * kThreads) {
        const int s = a.ids[i];
        if (s < -1 || s >= a.slots || (s >= 0 && first[s] != i)) atomicOr(a.flags, DMC_KV8_BAD_SLOT);
        else if (s >= 0 && a.lens[s] > a.cap) atomicOr(a.flags, DMC_KV8_TOO_LONG);
    }
    for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
        const int p = page_at(e);
        if (p < 0) continue;
        atomicSub(&a.refs[p], 1);
        claim[p] = INT32_MAX;
    }
    cl.sync();
    for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
        const int p = page_at(e);
        if (p >= 0 && __ldcg(&a.refs[p]) <= 0) atomicMin(&claim[p], (int)e);
    }
    cl.sync();
    // the first naming of a page that lost its last holder pushes it
    int mine = 0;
    for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
        const int p = page_at(e);
        mine += p >= 0 && __ldcg(&claim[p]) == (int)e && __ldcg(&a.refs[p]) == 0;
    }
    int total, fc = *a.free_count;
    block_scan(mine, &total);
    if (threadIdx.x < kCluster) cl.map_shared_rank(counts, threadIdx.x)[rank] = total;
    cl.sync();
    int at = fc, all = 0;
    for (int c = 0; c < kCluster; ++c) {
        if (c < rank) at += counts[c];
        all += counts[c];
    }
    for (long long x = e0; x < e1; x += kThreads) {
        const long long e = x + threadIdx.x;
        const int p = e < e1 ? page_at(e) : -1;
        const bool owner = p >= 0 && __ldcg(&claim[p]) == (int)e;
        const int refs = owner ? __ldcg(&a.refs[p]) : 1;
        const int place = at + block_scan(owner && refs == 0, &total);
        if (owner && refs == 0 && place >= 0 && place < a.pages) a.free_list[place] = p;
        if (owner && refs < 0) {  // it had no holder before: it is on the stack already
            a.refs[p] = 0;
            atomicOr(a.flags, DMC_KV8_BAD_PAGE);
        }
        at += total;
    }
    cl.sync();  // every length has been read
    for (int i = rank * kThreads + threadIdx.x; i < a.count; i += kCluster * kThreads) {
        const int s = a.ids[i];
        if (s >= 0 && s < a.slots && a.lens[s] <= a.cap) a.lens[s] = 0;
    }
    if (rank == 0 && threadIdx.x == 0) *a.free_count = min(fc + all, a.pages);
}

// One running count of the pages in use, `before`, gives both ends of every move: an unused page p below `live` is the
// (p - before)-th hole, a used one from `live` on the (before - before(live))-th mover.
__global__ void __launch_bounds__(kThreads) kv8_compact_kernel(PageArgs a) {
    __shared__ int live_by[kCluster], before_live;
    cg::cluster_group cl = cg::this_cluster();
    griddep_launch_dependents();
    griddep_wait();
    const int rank = blockIdx.x, gid = rank * kThreads + threadIdx.x;
    const int p0 = (int)((long long)a.pages * rank / kCluster), p1 = (int)((long long)a.pages * (rank + 1) / kCluster);
    int mine = 0, total;
    for (int p = p0 + threadIdx.x; p < p1; p += kThreads) mine += a.refs[p] > 0;
    block_scan(mine, &total);
    if (threadIdx.x == 0) before_live = a.pages;  // (all in use: nobody finds page `live`)
    cl.sync();
    if (threadIdx.x < kCluster) cl.map_shared_rank(live_by, threadIdx.x)[rank] = total;
    cl.sync();
    int live = 0, at = 0;
    for (int c = 0; c < kCluster; ++c) {
        if (c < rank) at += live_by[c];
        live += live_by[c];
    }
    for (int x = p0; x < p1; x += kThreads) {
        const int p = x + threadIdx.x;
        const bool used = p < p1 && a.refs[p] > 0;
        const int before = at + block_scan(used, &total);
        at += total;
        if (p >= p1) continue;
        page_map(a)[p] = p;
        if (p == live)
            for (int c = 0; c < kCluster; ++c) *cl.map_shared_rank(&before_live, c) = before;
        if (p < live && !used) list_dst(a)[p - before] = p;
        if (p >= live && used) list_src(a)[before] = p;
    }
    cl.sync();
    const int first = before_live, moves = live == a.pages ? 0 : live - first;
    for (int i = gid; i < moves; i += kCluster * kThreads) {
        const int from = __ldcg(&list_src(a)[first + i]), to = __ldcg(&list_dst(a)[i]);
        page_map(a)[from] = to;
        a.refs[to] = a.refs[from];
        a.refs[from] = 0;
    }
    cl.sync();
    const long long entries = (long long)a.slots * a.table_stride;
    for (long long e = gid; e < entries; e += kCluster * kThreads) {
        const int s = (int)(e / a.table_stride), col = (int)(e % a.table_stride), n = a.lens[s];
        if (n > a.cap && col == 0) atomicOr(a.flags, DMC_KV8_TOO_LONG);  // (renamed as far as it goes: its pages move too)
        if (col >= held_pages(a, n)) continue;
        const int p = a.table[e];
        if ((unsigned)p < (unsigned)a.pages) a.table[e] = __ldcg(&page_map(a)[p]);
        else atomicOr(a.flags, DMC_KV8_BAD_PAGE);
    }
    for (int p = gid; p < a.pages; p += kCluster * kThreads) {
        if (p < a.pages - live) a.free_list[p] = a.pages - 1 - p;
        if (a.moved) a.moved[p] = __ldcg(&page_map(a)[p]);
    }
    if (gid == 0) {
        *a.free_count = a.pages - live;
        a.scratch[0] = moves;
        a.scratch[1] = first;
    }
}

// ---- copy ------------------------------------------------------------------------------------------------------
// A page is kv_heads * page_tokens * head_dim contiguous bytes per layer and kind (K, V).  A CTA takes 16 KiB at a time,
// four 16-byte loads in flight per thread.
constexpr int kCopyThreads = 256;

struct CopyArgs {
    uint4 *k, *v;
    float *ks, *vs;
    const int *src, *dst, *count_at;  // count_at: the list's length and its first source, or null
    int *flags;
    int count, pages, layers, hk;
    int vecs;    // 16-byte pieces of a page
    int chunks;  // CTA turns of a page
};

__global__ void __launch_bounds__(kCopyThreads) kv8_copy_kernel(CopyArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    const int *src = a.src + (a.count_at ? a.count_at[1] : 0);
    const long long n = (long long)(a.count_at ? *a.count_at : a.count) * a.layers * 2 * a.chunks;
    for (long long i = blockIdx.x; i < n; i += gridDim.x) {
        const int chunk = (int)(i % a.chunks), kind = (int)(i / a.chunks % 2);
        const int layer = (int)(i / (2 * a.chunks) % a.layers), c = (int)(i / ((long long)2 * a.chunks * a.layers));
        const int from = src[c], to = a.dst[c];
        if ((unsigned)from >= (unsigned)a.pages || (unsigned)to >= (unsigned)a.pages) {
            if (threadIdx.x == 0) atomicOr(a.flags, DMC_KV8_BAD_PAGE);
            continue;
        }
        const size_t base = (size_t)layer * a.pages;
        const uint4 *x = (kind ? a.v : a.k) + (base + from) * a.vecs;
        uint4 *y = (kind ? a.v : a.k) + (base + to) * a.vecs;
        uint4 r[4];
        const int at = chunk * kCopyThreads * 4 + threadIdx.x;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (at + u * kCopyThreads < a.vecs) r[u] = __ldcs(x + at + u * kCopyThreads);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (at + u * kCopyThreads < a.vecs) y[at + u * kCopyThreads] = r[u];
        if (chunk == 0) {
            const float *xs = (kind ? a.vs : a.ks) + (base + from) * a.hk;
            float *ys = (kind ? a.vs : a.ks) + (base + to) * a.hk;
            for (int h = threadIdx.x; h < a.hk; h += kCopyThreads) ys[h] = xs[h];
        }
    }
}

int launch_copy(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, const int *src, const int *dst, const int *count_at, int count,
                cudaStream_t s) {
    CopyArgs a;
    a.k = (uint4 *)c.k;
    a.v = (uint4 *)c.v;
    a.ks = c.k_scale;
    a.vs = c.v_scale;
    a.src = src;
    a.dst = dst;
    a.count_at = count_at;
    a.flags = q.flags;
    a.count = count_at ? 0 : count;
    a.pages = (int)c.pages;
    a.layers = c.layers;
    a.hk = c.kv_heads;
    a.vecs = c.kv_heads * c.page_tokens * c.head_dim / 16;
    a.chunks = (a.vecs + kCopyThreads * 4 - 1) / (kCopyThreads * 4);
    // (`count` is the most that a list on the device can hold)
    const int64_t units = (int64_t)std::max(count, 1) * c.layers * 2 * a.chunks;
    void *params[] = {&a};
    return launch_on((const void *)kv8_copy_kernel, dim3((unsigned)std::min<int64_t>(units, ctx().sm_count * 8)), dim3(kCopyThreads),
                     0, s, params);
}

PageArgs args_of(const dmc_kv8_cache &c, const dmc_kv8_seqs &q) {
    PageArgs a = {};
    a.table = q.table;
    a.lens = q.lens;
    a.refs = q.refs;
    a.free_list = q.free_list;
    a.free_count = q.free_count;
    a.flags = q.flags;
    a.scratch = (int *)q.scratch;
    a.table_stride = q.table_stride;
    a.slots = q.slots;
    a.pages = (int)c.pages;
    a.page_tokens = c.page_tokens;
    a.cap = (int)(q.table_stride * c.page_tokens);
    return a;
}

#define PAGE_POINTERS(q)                                                                                              \
    {(q)->refs, 4, "seqs.refs"}, {(q)->free_list, 4, "seqs.free_list"}, {(q)->free_count, 4, "seqs.free_count"}, {(q)->scratch, 16, "seqs.scratch"}

int check_ids(const dmc_kv8_seqs *q, int count, const char *who) {
    if (count < 0) return fail(DMC_CUDA_ERR_BAD_ARG, "%s: negative count", who);
    if (count > kKv8MaxSlots || (int64_t)count * q->table_stride > INT32_MAX)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "%s: more than %d slots, or than 2^31-1 table entries, in one call", who, kKv8MaxSlots);
    return DMC_CUDA_OK;
}

template <typename K>
int launch_cluster(K *fn, PageArgs a, size_t smem, cudaStream_t s) {
    void *params[] = {&a};
    return launch_on((const void *)fn, dim3(kCluster), dim3(kThreads), smem, s, params, kCluster);
}

// The start of every call: the library's state and the descriptors.
#define KV8_ENTER(who)                                   \
    std::lock_guard<std::mutex> lock(ctx_mutex());       \
    if (dmc::status()) return dmc::status();             \
    OnDevice on;                                         \
    int rc;                                              \
    if ((rc = check_kv8(cache, seqs, who))) return rc

}  // namespace

int launch_kv8_reserve(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, const int *slot_ids, const int *counts, int batch, int tokens,
                       cudaStream_t s) {
    PageArgs a = args_of(c, q);
    a.ids = slot_ids;
    a.ids2 = counts;
    a.count = batch;
    a.tokens = tokens;
    DMC_CUDA_TRY(cudaFuncSetAttribute((const void *)kv8_reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)sizeof(ReserveSmem)));
    void *params[] = {&a};
    int rc = launch_on((const void *)kv8_reserve_kernel, dim3(1), dim3(kThreads), sizeof(ReserveSmem), s, params);
    if (rc) return rc;
    return launch_copy(c, q, a.scratch + kHeader, a.scratch + kHeader + a.pages, a.scratch, batch, s);
}

int launch_kv8_fork(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, const int *src, const int *dst, int count, cudaStream_t s) {
    PageArgs a = args_of(c, q);
    a.ids = src;
    a.ids2 = dst;
    a.count = count;
    return launch_cluster(kv8_fork_kernel, a, (size_t)q.slots * 4, s);
}

int launch_kv8_release(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, const int *slot_ids, int count, cudaStream_t s) {
    PageArgs a = args_of(c, q);
    a.ids = slot_ids;
    a.count = count;
    return launch_cluster(kv8_release_kernel, a, (size_t)q.slots * 4, s);
}

int launch_kv8_compact(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, int *moved, cudaStream_t s) {
    PageArgs a = args_of(c, q);
    a.moved = moved;
    int rc = launch_cluster(kv8_compact_kernel, a, 0, s);
    if (rc) return rc;
    return launch_copy(c, q, a.scratch + kHeader, a.scratch + kHeader + a.pages, a.scratch, (int)c.pages, s);
}

}  // namespace dmc

using namespace dmc;

extern "C" int64_t dmc_kv8_scratch_bytes(int64_t pages, int slots) {
    (void)slots;
    return pages < 0 ? 0 : ((int64_t)kHeader + 3 * pages) * 4;
}

extern "C" int dmc_kv8_reserve(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, const int *slot_ids, const int *counts,
                               int batch, int tokens, void *stream) {
    KV8_ENTER("kv8_reserve");
    if (batch < 0 || tokens < 0) return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_reserve: negative batch or tokens");
    if ((rc = check_ids(seqs, batch, "kv8_reserve"))) return rc;  // (so the requests' number fits an int)
    if (batch > kReserveBatch) return fail(DMC_CUDA_ERR_UNSUPPORTED, "kv8_reserve: batch %d beyond %d", batch, kReserveBatch);
    if (!slot_ids && batch > seqs->slots)
        return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_reserve: batch %d of %d slots without slot_ids", batch, seqs->slots);
    if (batch == 0) return DMC_CUDA_OK;
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), PAGE_POINTERS(seqs), {slot_ids, 4, "slot_ids", true}, {counts, 4, "counts", true}})))
        return rc;
    return launch_kv8_reserve(*cache, *seqs, slot_ids, counts, batch, tokens, (cudaStream_t)stream);
}

extern "C" int dmc_kv8_fork(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, const int *src, const int *dst, int count,
                            void *stream) {
    KV8_ENTER("kv8_fork");
    if ((rc = check_ids(seqs, count, "kv8_fork"))) return rc;
    if (count == 0) return DMC_CUDA_OK;
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), PAGE_POINTERS(seqs), {src, 4, "src"}, {dst, 4, "dst"}}))) return rc;
    return launch_kv8_fork(*cache, *seqs, src, dst, count, (cudaStream_t)stream);
}

extern "C" int dmc_kv8_release(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, const int *slot_ids, int count, void *stream) {
    KV8_ENTER("kv8_release");
    if ((rc = check_ids(seqs, count, "kv8_release"))) return rc;
    if (count == 0) return DMC_CUDA_OK;
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), PAGE_POINTERS(seqs), {slot_ids, 4, "slot_ids"}}))) return rc;
    return launch_kv8_release(*cache, *seqs, slot_ids, count, (cudaStream_t)stream);
}

extern "C" int dmc_kv8_compact(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, int *moved, void *stream) {
    KV8_ENTER("kv8_compact");
    if ((int64_t)seqs->slots * seqs->table_stride > INT32_MAX)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "kv8_compact: a table of more than 2^31-1 entries");
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), PAGE_POINTERS(seqs), {moved, 4, "moved", true}}))) return rc;
    return launch_kv8_compact(*cache, *seqs, moved, (cudaStream_t)stream);
}

extern "C" int dmc_kv8_copy_pages(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, const int *src, const int *dst, int count,
                                  void *stream) {
    KV8_ENTER("kv8_copy_pages");
    if (count < 0 || count > cache->pages) return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_copy_pages: count %d of %lld pages", count, (long long)cache->pages);
    if (count == 0) return DMC_CUDA_OK;
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), {src, 4, "src"}, {dst, 4, "dst"}}))) return rc;
    return launch_copy(*cache, *seqs, src, dst, nullptr, count, (cudaStream_t)stream);
}
