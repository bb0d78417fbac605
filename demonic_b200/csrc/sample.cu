// sample.cu -- one token per row of logits: temperature, top-k, top-p, min-p and a given uniform number.
//
// A row belongs to one thread-block cluster, which brings it into the shared memory of its CTAs once (f32 slices); every
// further step works there and exchanges a few words through distributed shared memory, so the logits are read
// from HBM once and there is no workspace.  Masses are 64-bit integers: w = exp((x - max) / T) in double, times 2^44,
// rounded.  Integer sums have no order, so histograms may be built with atomics and every CTA comes to the same result.
//
// The k-th largest logit, or the one at which the mass reaches top_p, is found by histogram: 1024 bins over the distance
// from the maximum (an order-preserving map, whatever its rounding) and the bin that holds the answer.  While no more
// than 512 logits lie in the bins up to it, one CTA takes those, sorts them and finishes alone; else the bin's members are
// ranked one against another, or split again while they are many -- by the bits of the values, since different logits may lie
// at one rounded distance -- and the whole cluster goes on with the cut.
//
// Measured on B200 (us a call): one row of 32000 f32 5.4 for the maximum alone, 7 without a filter, 12 with top-k, 25 with top-p;
// 64 rows of 128000 f32 15 (33 MB, 2.1 TB/s) / 31 / 44 / 83, 55 mixed; 256 rows of 50257 bf16 16 / 35 / 37 / 112.  No unit is full: in
// the last case without a filter issue slots are 58 % busy, ALU 34 %, FP64 25 %, HBM 8 %, 26 warps per SM; with mixed filters 47 %,
// 30 %, 7 %, 7 %, and barriers the longest stall.  A cluster loads its row, then works on it: while it does the one it does not do
// the other, and 256 rows are 1.8 times what runs at once.  One row is latency: barriers of its cluster, and steps of one CTA.
// At 64 registers the builds spill 8 (512 threads) and 32 bytes (256).
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "gemv.cuh"
#include "runtime.h"

namespace cg = cooperative_groups;

namespace dmc {
namespace {

// CTAs of 256 threads while a slice is at most 28 KiB, else of 512: 1024 threads per SM either way (64 registers each, while
// shared memory holds so many slices), but four CTAs in different phases hide one another's barriers (256 rows of 50257 bf16
// logits, 25 KiB: 57 us with two CTAs of 512 threads, 35 with four of 256).  From 28 to 43 KiB four CTAs fit as well, and which is
// better goes by the rows: 64 of 128256 bf16 (31 KiB) 31 us with 512 threads and 23 with 256 without a filter, 54 and 58 mixed; 256
// of them 106 and 72, 184 and 127 mixed; but 16 of them 38 and 52 with top-p, since the longest row then counts; 64 of 80000 f32
// (39 KiB) 25 and 20, 47 and 51 mixed.  Clusters of 16 were slower than 8 with larger slices (64 rows of 128000: 20 us against 15
// up to the maximum).
constexpr int kMaxCluster = 8;
constexpr int kBinBits = 10, kBins = 1 << kBinBits, kList = 512;
constexpr int kMaxSlice = kSampleMaxVocab / kMaxCluster;  // logits of a row per CTA: 128 KiB of f32 at most
constexpr double kOne = (double)(1ull << 44);    // mass of weight 1
constexpr float kFar = 32.0f;                    // e^-32 * 2^44 rounds to 0
constexpr int kTable = 16;                       // 2^(j / 16)
typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    const float *temperature, *top_p, *min_p, *u;
    const int *top_k;
    int *tokens;
    float *prob;
    long long row_stride;
    int vocab, slice;
    int batch;  // rows, if those that take longest are to be taken first; else 0
};

struct Found {       // where a query's answer lies: a bin, and what comes before it
    unsigned members, count_before;
    int bin;
    u64 before, inside;
};

struct Histogram {
    unsigned count[kBins], lo[kBins], hi[kBins];  // this CTA's members: how many, and their mass in two words
};
struct Lists {                      // once the histograms have been read
    u64 list[kList];                // keys of this CTA's members
    u64 all[kList], mass[kList];    // in the first CTA: the cluster's keys, and their masses
};
struct SampleSmem {
    union {
        Histogram h;
        Lists l;
    };
    double table[kTable];           // 2^44 * 2^(j / 16)
    float top[kMaxCluster];         // largest value of each CTA
    int first[kMaxCluster];         // where the row's largest value is first found
    u64 seg_mass[kMaxCluster];
    unsigned seg_count[kMaxCluster];
    Found found;
    unsigned least_key[kMaxCluster], most_key[kMaxCluster];  // extent of each CTA's members of a bin
    u64 part[kMaxCluster];
    u64 ws[16];
    unsigned wc[16];
    int n_list;                     // members of the bin, or of the leading bins, in this CTA
    u64 cut_key, cut_mass;
    float red_f[16];
    unsigned red_u[16], red_v[16];
    int red_i[16];
    int row;
};

// Greater value first, then lower index: a smaller key.  Values are equal where their keys' high words are.
__device__ __forceinline__ unsigned value_key(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);  // (-0 orders as 0)
    return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ u64 key_of(float x, int i) { return ((u64)value_key(x) << 32) | (unsigned)i; }
__device__ __forceinline__ float value_of(u64 key) {
    const unsigned ord = ~(unsigned)(key >> 32);
    return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7FFFFFFFu) : ~ord);
}

struct Row {
    float top, far;       // largest logit (finite); distance from which on there is no mass: 32 T
    double c, b;          // 16 log2(e) / T and -top times that
    const double *table;
    __device__ __forceinline__ float dist(float x) const { return top - x; }
    __device__ __forceinline__ bool near(float d) const { return d <= far; }
    // 2^44 w for a near x.  16 (x - top) log2(e) / T = 16 n + j + r with |r| <= 1 / 2; 2^(r / 16) by a polynomial of degree 4
    // through the Chebyshev points of that interval (2^-38 off at most), 2^(j / 16) from the table, n into the exponent.
    // b is off by half a unit of its last place, 2^-34 while |top| log2(e) / T is below 2^16 (the kernel sees to that): a
    // factor of 2^(2^-34 / 16), less than 1 + 2^-38, which all weights of the row share.
    __device__ __forceinline__ double scaled(float x) const {
        const double y = fma((double)x, c, b);
        const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low word
        const double k = y + magic;
        const double r = y - (k - magic);
        const int q = __double2loint(k);
        double p = fma(9.618314296478376e-3 / 65536, r, 5.550573631387555e-2 / 4096);
        p = fma(p, r, 0.24022650691572542 / 256);
        p = fma(p, r, 0.6931471801625689 / 16);
        p = fma(p, r, 1.0) * table[q & (kTable - 1)];
        return __hiloint2double(__double2hiint(p) + (q & -kTable) * (1 << 16), __double2loint(p));
    }
    // (without a branch, so that several can be under way)
    __device__ __forceinline__ u64 mass(float x) const {
        const double m = scaled(x) + 4503599627370496.0;  // + 2^52: rounded to an integer, in the low 52 bits
        return near(dist(x)) ? (u64)__double_as_longlong(m) & 0xFFFFFFFFFFFFFull : 0ull;
    }
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum of v over the threads before this one; *total the CTA's.  Ends with a barrier.
template <int TH, typename T>
__device__ __forceinline__ T block_before(T v, T *ws, T *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) ws[warp] = inc;
    __syncthreads();
    T at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < (TH / 32); ++w) {
        if (w < warp) at += ws[w];
        all += ws[w];
    }
    *total = all;
    __syncthreads();
    return at + inc - v;
}

// The row slice in shared memory, as it came, and what a CTA knows of its cluster.
template <bool BF16>
struct Slice {
    using T = typename std::conditional<BF16, uint16_t, float>::type;
    T *x;
    int n, first;  // elements, index of the first
    int rank, ranks;
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (BF16) return __uint_as_float((uint32_t)x[i] << 16);
        else return x[i];
    }
};

// Everything from a value on: greater values, and the value itself up to an index.
struct Cut {
    float value;
    int index;
    __device__ __forceinline__ bool keeps(float x, int i) const { return x > value || (x == value && i <= index); }
};
__device__ __forceinline__ Cut cut_of(u64 key) { return Cut{value_of(key), (int)(unsigned)key}; }

constexpr int kUnroll = 4;  // elements that a thread has under way

// f(value, position) for the elements begin, begin + step, ... below end, kUnroll at a time.
template <bool BF16, typename F>
__device__ __forceinline__ void each(const Slice<BF16> &x, int begin, int end, int step, F f) {
    int i = begin;
    for (; i + (kUnroll - 1) * step < end; i += kUnroll * step) {
        float v[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) v[j] = x[i + j * step];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) f(v[j], i + j * step);
    }
    for (; i < end; i += step) f(x[i], i);
}

// n <= kList keys of sm.l.all, ascending, all different; sm.l.mass is overwritten.  Runs of 32 by a bitonic network in a warp's
// registers, then every key finds its place among the other runs by bisection: two barriers (45 of a network over all of
// 512 keys took 10 us).
template <int TH>
__device__ __noinline__ void sort_keys(SampleSmem &sm, int n) {
    const int lane = threadIdx.x & 31, runs = (n + 31) / 32;
    for (int run = threadIdx.x >> 5; run < runs; run += TH / 32) {
        const int i = run * 32 + lane;
        u64 key = i < n ? sm.l.all[i] : ~0ull;
#pragma unroll
        for (int k = 2; k <= 32; k *= 2)
#pragma unroll
            for (int j = k / 2; j > 0; j /= 2) {
                const u64 other = __shfl_xor_sync(0xffffffffu, key, j);
                const bool up = (lane & k) == 0 || k == 32, low = (lane & j) == 0;
                key = (key < other) == (up == low) ? key : other;
            }
        sm.l.mass[i] = key;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < runs * 32; i += TH) {
        const u64 key = sm.l.mass[i];
        int place = i & 31;
        for (int run = 0; run < runs; ++run) {
            if (run == i >> 5) continue;
            const u64 *r = sm.l.mass + run * 32;
            int below = 0;
#pragma unroll
            for (int step = 16; step > 0; step /= 2)
                if (r[below + step - 1] < key) below += step;
            place += below + (r[below] < key);
        }
        if (key != ~0ull) sm.l.all[place] = key;
    }
    __syncthreads();
}

// Every CTA's count to every CTA (a barrier of the cluster): the sum of those before this one, and of all.
template <bool BF16>
__device__ __forceinline__ int share_count(SampleSmem &sm, cg::cluster_group &cl, const Slice<BF16> &s, int mine, int *total) {
    if (threadIdx.x < s.ranks) cl.map_shared_rank(sm.seg_count, threadIdx.x)[s.rank] = (unsigned)mine;
    cl.sync();
    int before = 0, all = 0;
    for (int r = 0; r < s.ranks; ++r) {
        if (r < s.rank) before += (int)sm.seg_count[r];
        all += (int)sm.seg_count[r];
    }
    *total = all;
    return before;
}

// What is asked of a row: its shortest leading part, in order (value down, index up), that has at least `need` members, or
// (need == 0) at least `part` of the mass of what is kept so far, which leading_part leaves in `of`.
struct Query {
    unsigned need;
    double part;
    u64 of;
    bool sparse;  // first count the threads' own maxima alone: the need-th largest of them is not above the row's
};

// The answer in *cut (within what *cut keeps already), or false if the bins up to the one that holds it have at most kList
// members, which *lead_bin then names (bins from distance 0, *lead_step per unit).  Every thread of the cluster gets the same.
// With q.sparse the bin named may have more members, or be kBins: nothing found.
template <int TH, bool BF16>
__device__ __forceinline__ bool leading_part(SampleSmem &sm, const Slice<BF16> s, const Row row, float own, Query &query, Cut *cut,
                                          int *lead_bin, float *lead_step) {
    cg::cluster_group cl = cg::this_cluster();
    const Query q = query;
    const Cut limit = *cut;
    const int tid = threadIdx.x;
    const bool by_mass = q.need == 0;
    // Level 0 has its bins by distance; what is in the one it finds is binned by the value's key from then on, 10 bits of the
    // members' extent at a time.  The map to bins is monotone at every level, so the members are the logits of an interval.
    u64 before = 0, inside = 0;
    unsigned count_before = 0, members = 0;
    double target = 0.0;
    const float step0 = (float)kBins / row.far;
    auto bin_of = [&](float d) { return min(kBins - 1, (int)(d * step0)); };
    int bin0 = -1;                             // level 0's bin
    unsigned from = 0, width = 0xFFFFFFFFu;    // keys from .. from + width, of which the bins have 2^shift each
    int shift = 0, level = 0;
    auto member = [&](float x, int i) {
        const float d = row.dist(x);
        return row.near(d) && limit.keeps(x, s.first + i) && (bin0 < 0 || bin_of(d) == bin0) && value_key(x) - from <= width;
    };
#pragma unroll 1
    for (;; ++level) {
        for (int i = tid; i < kBins; i += TH) sm.h.count[i] = sm.h.lo[i] = sm.h.hi[i] = 0;
        __syncthreads();
        if (q.sparse) {
            if (row.near(row.dist(own))) atomicAdd(&sm.h.count[bin_of(row.dist(own))], 1u);
        } else {
            each(s, tid, s.n, TH, [&](float x, int i) {
                const u64 m = by_mass ? row.mass(x) : 0;
                if (!member(x, i)) return;
                const int b = level == 0 ? bin_of(row.dist(x)) : (int)((value_key(x) - from) >> shift);
                if (by_mass) {
                    const unsigned lo = (unsigned)m, was = atomicAdd(&sm.h.lo[b], lo);
                    const unsigned hi = (unsigned)(m >> 32) + (was + lo < was ? 1u : 0u);
                    if (hi) atomicAdd(&sm.h.hi[b], hi);
                }
                atomicAdd(&sm.h.count[b], 1u);
            });
        }
        cl.sync();
        // each CTA adds up its share of the bins over the cluster (seg <= 1024 bins over 256 threads and more)
        const int seg = kBins / s.ranks, per = (seg + TH - 1) / TH, mine = s.rank * seg + tid * per;
        unsigned c = 0, cs[4] = {0, 0, 0, 0};
        u64 m = 0, ms[4] = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            if (r >= s.ranks) break;
            const Histogram *h = cl.map_shared_rank(&sm.h, r);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < per && mine + j < (s.rank + 1) * seg) {
                    cs[j] += h->count[mine + j];
                    if (by_mass) ms[j] += (u64)h->hi[mine + j] << 32 | h->lo[mine + j];
                }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c += cs[j], m += ms[j];
        unsigned c_all;
        u64 m_all = 0, m_at = 0;
        const unsigned c_at = block_before<TH>(c, sm.wc, &c_all);
        if (by_mass) m_at = block_before<TH>(m, sm.ws, &m_all);
        if (tid < s.ranks) {
            cl.map_shared_rank(sm.seg_mass, tid)[s.rank] = m_all;
            cl.map_shared_rank(sm.seg_count, tid)[s.rank] = c_all;
        }
        cl.sync();
        // the bin at which the running count or mass reaches what is asked
        u64 mb = before, m_row = before;
        unsigned cb = count_before, c_row = count_before;
        for (int r = 0; r < s.ranks; ++r) {
            if (r < s.rank) mb += sm.seg_mass[r], cb += sm.seg_count[r];
            m_row += sm.seg_mass[r], c_row += sm.seg_count[r];
        }
        mb += m_at, cb += c_at;
        if (level == 0 && by_mass) {
            query.of = m_row;
            target = fmax(q.part * (double)m_row, 1.0);
        }
        // (asked for more than there is: the last member is the answer)
        const unsigned want = min(q.need, c_row);
        const double goal = fmin(target, (double)m_row);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool here = cs[j] && (by_mass ? (double)mb < goal && (double)(mb + ms[j]) >= goal : cb < want && cb + cs[j] >= want);
            if (here)
                for (int r = 0; r < s.ranks; ++r) *cl.map_shared_rank(&sm.found, r) = Found{cs[j], cb, mine + j, mb, ms[j]};
            mb += ms[j], cb += cs[j];
        }
        cl.sync();
        const Found f = sm.found;
        if (level == 0) {
            bin0 = f.bin;
        } else {
            from += (unsigned)f.bin << shift;
            width = min(width - ((unsigned)f.bin << shift), (1u << shift) - 1);  // (the last bin ends with its level)
        }
        before = f.before, count_before = f.count_before, members = f.members, inside = f.inside;
        if (level == 0 && (q.sparse || count_before + members <= kList)) {
            *lead_bin = q.sparse && c_row < q.need ? kBins : f.bin;  // (fewer maxima than asked for say nothing)
            *lead_step = step0;
            return false;
        }
        if (members <= kList) break;
        // many members: their own extent for the next level.  It is less than 2^32 of keys at level 1 and than 2^10 times less
        // at each further one, so level 5 would be one of equal values.
        unsigned least = 0xFFFFFFFFu, most = 0;
        each(s, tid, s.n, TH, [&](float x, int i) {
            if (member(x, i)) least = min(least, value_key(x)), most = max(most, value_key(x));
        });
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if ((tid & 31) == 0) sm.red_u[tid >> 5] = least, sm.red_v[tid >> 5] = most;
        __syncthreads();
        for (int w = 0; w < TH / 32; ++w) least = min(least, sm.red_u[w]), most = max(most, sm.red_v[w]);
        if (tid < s.ranks) {
            cl.map_shared_rank(sm.least_key, tid)[s.rank] = least;
            cl.map_shared_rank(sm.most_key, tid)[s.rank] = most;
        }
        cl.sync();
        for (int r = 0; r < s.ranks; ++r) least = min(least, sm.least_key[r]), most = max(most, sm.most_key[r]);
        if (least == most) break;  // all equal
        from = least;
        width = most - least;
        shift = max(0, 32 - __clz((int)width) - kBinBits);
    }
    if (members <= kList) {  // the first CTA takes them, sorts them and tells the others
        if (tid == 0) sm.n_list = 0;
        __syncthreads();
        each(s, tid, s.n, TH, [&](float x, int i) {
            if (member(x, i)) sm.l.list[atomicAdd(&sm.n_list, 1)] = key_of(x, s.first + i);
        });
        __syncthreads();
        int n;
        u64 *const to = cl.map_shared_rank(sm.l.all, 0) + share_count(sm, cl, s, sm.n_list, &n);
        for (int i = tid; i < sm.n_list; i += TH) to[i] = sm.l.list[i];
        cl.sync();
        if (s.rank == 0) {
            sort_keys<TH>(sm, n);
            const unsigned want = min(q.need, count_before + members);
            const double goal = fmin(target, (double)(before + inside));
            constexpr int EACH = kList / TH;
            u64 own_mass[EACH], sum = 0, all;
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const int i = EACH * tid + j;
                own_mass[j] = by_mass && i < n ? row.mass(value_of(sm.l.all[i])) : 0;
                sum += own_mass[j];
            }
            u64 run = before + block_before<TH>(sum, sm.ws, &all);
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const int i = EACH * tid + j;
                const bool here = by_mass ? (double)run < goal && (double)(run + own_mass[j]) >= goal : count_before + i + 1 == want;
                if (i < n && here)
                    for (int r = 0; r < s.ranks; ++r) *cl.map_shared_rank(&sm.cut_key, r) = sm.l.all[i];
                run += own_mass[j];
            }
        }
        cl.sync();
        *cut = cut_of(sm.cut_key);
    } else {
        // so many equal values: they are taken by index
        float x = 0.0f;
        unsigned c = 0;
        const int per = (s.n + TH - 1) / TH, i0 = min(s.n, tid * per), i1 = min(s.n, i0 + per);
        for (int i = i0; i < i1; ++i) {
            if (member(s[i], i)) {
                x = s[i];
                ++c;
            }
        }
        unsigned here;
        const unsigned at = block_before<TH>(c, sm.wc, &here);
        if (tid < s.ranks) cl.map_shared_rank(sm.seg_count, tid)[s.rank] = here;
        cl.sync();
        unsigned below = 0;
        for (int r = 0; r < s.rank; ++r) below += sm.seg_count[r];
        if (c) {
            unsigned k = 1;  // how many of them are kept
            if (by_mass) {
                const u64 own = row.mass(x);  // (the same for all of them)
                const double goal = fmin(target, (double)(before + inside));
                unsigned a = 1, b = members;  // the smallest k with before + k * own >= goal
                while (a < b) {
                    const unsigned mid = (a + b) / 2;
                    if ((double)(before + mid * own) >= goal) b = mid;
                    else a = mid + 1;
                }
                k = a;
            } else {
                k = min(q.need - count_before, members);
            }
            if (below + at < k && below + at + c >= k) {
                unsigned j = below + at;
                for (int i = i0; i < i1; ++i)
                    if (member(s[i], i) && ++j == k)
                        for (int r = 0; r < s.ranks; ++r) *cl.map_shared_rank(&sm.cut_key, r) = key_of(s[i], s.first + i);
            }
        }
        cl.sync();
        *cut = cut_of(sm.cut_key);
    }
    return true;
}

__device__ __forceinline__ bool filters_by_k(int k, int vocab) { return k > 0 && k < vocab; }
// k is small enough for the k-th largest of `threads` threads' maxima to lie near the k-th largest logit.
__device__ __forceinline__ bool few(int k, int threads) { return k <= min(kList / 2, threads / 4); }

// The row that the `turn`-th cluster takes: rows that need a histogram of all their logits first (they take two to three times as
// long), the others behind them, each kind in order.
constexpr int kRowsEach = 4;  // rows that a thread looks at
template <int TH>
__device__ __forceinline__ int row_of_turn(const int *top_k, const float *top_p, int batch, int vocab, SampleSmem &sm, int turn, int ranks) {
    unsigned slow[kRowsEach], mine = 0, all;
#pragma unroll
    for (int j = 0; j < kRowsEach; ++j) {
        const int r = threadIdx.x * kRowsEach + j;
        slow[j] = 0;
        if (r < batch) {
            const int k = top_k ? top_k[r] : 0;
            const float p = top_p ? top_p[r] : 1.0f;
            slow[j] = filters_by_k(k, vocab) ? !few(k, ranks * TH) : p < 1.0f;
        }
        mine += slow[j];
    }
    int before = (int)block_before<TH>(mine, sm.wc, &all);
#pragma unroll
    for (int j = 0; j < kRowsEach; ++j) {
        const int r = threadIdx.x * kRowsEach + j;
        if (r < batch && turn == (slow[j] ? before : (int)all + r - before)) sm.row = r;
        before += (int)slow[j];
    }
    __syncthreads();
    return sm.row;
}

template <int TH, bool BF16>
__global__ void __launch_bounds__(TH, 1024 / TH) sample_kernel(SampleArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    SampleSmem &sm = *reinterpret_cast<SampleSmem *>(raw);
    cg::cluster_group cl = cg::this_cluster();
    griddep_launch_dependents();
    cl.barrier_arrive();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    using T = typename Slice<BF16>::T;
    Slice<BF16> s;
    s.rank = (int)cl.block_rank();
    s.ranks = (int)cl.num_blocks();
    long long r = blockIdx.x / s.ranks;
    if (a.batch) r = row_of_turn<TH>(a.top_k, a.top_p, a.batch, a.vocab, sm, (int)r, s.ranks);
    s.first = min(a.vocab, s.rank * a.slice);
    s.n = min(a.vocab, s.first + a.slice) - s.first;
    const float t = a.temperature ? a.temperature[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    const int k = a.top_k ? a.top_k[r] : 0;
    const double u = (double)a.u[r];
    if (tid < kTable) sm.table[tid] = exp2((double)tid / kTable) * kOne;

    // ---- the slice into shared memory, and its largest value.  Pieces of 16 bytes from the first boundary on.
    const T *g = (const T *)a.logits + r * a.row_stride + s.first;
    constexpr int VEC = 16 / sizeof(T);
    const int head = min(s.n, (int)((16 - (uintptr_t)g % 16) % 16 / sizeof(T)));
    s.x = reinterpret_cast<T *>(raw + (sizeof(SampleSmem) + 15) / 16 * 16) + (VEC - head) % VEC;  // (x + head has a boundary, too)
    float top = -INFINITY;
    bool nan = false;
    auto take = [&](float v) {
        nan |= !(v == v);
        top = fmaxf(top, v);  // (passes over NaN)
    };
    const int nv = (s.n - head) / VEC;
    if (tid < head) s.x[tid] = g[tid], take(s[tid]);
    for (int i = head + nv * VEC + tid; i < s.n; i += TH) s.x[i] = g[i], take(s[i]);
    const uint4 *gv = (const uint4 *)(g + head);
    uint4 *xv = (uint4 *)(s.x + head);
    auto put = [&](int v, uint4 w) {
        xv[v] = w;
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (BF16) take(__uint_as_float(q[k] << 16)), take(__uint_as_float(q[k] & 0xFFFF0000u));
            else take(__uint_as_float(q[k]));
        }
    };
    int v = tid;
    for (; v + 3 * TH < nv; v += 4 * TH) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = ld_stream16(gv + v + j * TH);
#pragma unroll
        for (int j = 0; j < 4; ++j) put(v + j * TH, w[j]);
    }
    for (; v < nv; v += TH) put(v, ld_stream16(gv + v));
    auto rewrite = [&](auto f) {
        for (int i = tid; i < s.n; i += TH) {
            const float y = f(s[i]);
            if constexpr (BF16) s.x[i] = (uint16_t)(__float_as_uint(y) >> 16);  // (0, -inf or a difference, exact in 8 bits)
            else s.x[i] = y;
        }
        __syncthreads();
    };
    if (__syncthreads_or(nan)) rewrite([](float y) { return y == y ? y : -INFINITY; });
    float own = top;  // the largest of this thread's elements
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sm.red_f[warp] = top;
    __syncthreads();
    cl.barrier_wait();  // (every CTA of the cluster runs: its shared memory may be written)
    if (tid < s.ranks) {
        for (int w = 0; w < (TH / 32); ++w) top = fmaxf(top, sm.red_f[w]);
        cl.map_shared_rank(sm.top, tid)[s.rank] = top;
    }
    cl.sync();
    top = sm.top[0];
    for (int k = 1; k < s.ranks; ++k) top = fmaxf(top, sm.top[k]);
    if (top == -INFINITY || !(t > 0.0f) || mp > 1.0f) {  // nothing to draw from, or only the first maximum
        int at = INT32_MAX;
        each(s, tid, s.n, TH, [&](float y, int i) {
            if (y == top) at = min(at, s.first + i);
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
        if (lane == 0) sm.red_i[warp] = at;
        __syncthreads();
        for (int w = 0; w < (TH / 32); ++w) at = min(at, sm.red_i[w]);
        if (tid == 0) cl.map_shared_rank(sm.first, 0)[s.rank] = at;
        cl.sync();
        if (s.rank == 0 && tid == 0) {
            for (int k = 0; k < s.ranks; ++k) at = min(at, sm.first[k]);
            a.tokens[r] = top == -INFINITY ? -1 : at;
            if (a.prob) a.prob[r] = top == -INFINITY ? 0.0f : 1.0f;
        }
        return;  // (nobody writes another CTA's shared memory after the last cluster barrier)
    }
    if (top == INFINITY) {  // all mass is on the infinite ones
        rewrite([](float y) { return y == INFINITY ? 0.0f : -INFINITY; });
        top = 0.0f;
        own = own == INFINITY ? 0.0f : -INFINITY;
    }
    // A temperature that is tiny beside the largest logit: whatever has mass lies within 32 T of it, less than half of it, so
    // that the difference is exact.
    if (fabsf(top) > 45000.0f * t) {
        const float shift = top;
        rewrite([=](float y) { return y - shift; });
        top = 0.0f;
        own -= shift;
    }

    // ---- the filters
    Row row;
    row.top = top;
    row.far = fminf(kFar * t, 3.402823466e38f);
    row.c = 16.0 * 1.4426950408889634 / (double)t;
    row.b = -((double)top * row.c);
    row.table = sm.table;
    const u64 least = mp > 0.0f ? (u64)ceil((double)mp * (double)row.mass(top)) : 0;  // mass of w = min_p
    Cut cut{-INFINITY, INT32_MAX};
    const bool by_k = filters_by_k(k, a.vocab), by_p = p < 1.0f;
    // the mass that u points at, of all that is kept (u of 1 and more, or NaN: the largest double below the whole)
    auto aim_at = [&](u64 total) {
        const double most = __longlong_as_double(__double_as_longlong((double)total) - 1);
        return u < 1.0 ? fmax(0.0, fmin(u * (double)total, most)) : most;
    };
    auto answer = [&](int token, float value, u64 total) {
        a.tokens[r] = token;
        if (a.prob) a.prob[r] = (float)(row.scaled(value) / (double)total);
    };

#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        // 0: the k-th largest by way of the threads' maxima, while k is small among them; 1: the same by all; 2: top_p
        if (pass == 0 ? !by_k || !few(k, s.ranks * TH) : pass == 1 ? !by_k : !by_p) continue;
        Query q{pass < 2 ? (unsigned)k : 0u, (double)p, 0, pass == 0};
        int lead_bin;
        float lead_step;
        if (leading_part<TH>(sm, s, row, own, q, &cut, &lead_bin, &lead_step)) continue;
        // few logits lead: the first CTA takes them all and finishes
        if (tid == 0) sm.n_list = 0;
        __syncthreads();
        u64 *const list = sm.l.list;
        if (lead_bin < kBins)
            each(s, tid, s.n, TH, [&](float v, int i) {
                const float d = row.dist(v);
                if (!row.near(d) || min(kBins - 1, (int)(d * lead_step)) > lead_bin || !cut.keeps(v, s.first + i)) return;
                const int to = atomicAdd(&sm.n_list, 1);
                if (to < kList) list[to] = key_of(v, s.first + i);
            });
        else if (tid == 0) sm.n_list = kList + 1;
        __syncthreads();
        int n;
        const int n_mine = sm.n_list, n_before = share_count(sm, cl, s, n_mine, &n);
        if (n > kList) {  // (after pass 0 alone)
            cl.sync();
            continue;
        }
        u64 *const to = cl.map_shared_rank(sm.l.all, 0) + n_before;
        for (int i = tid; i < n_mine; i += TH) to[i] = list[i];
        cl.sync();
        if (s.rank != 0) return;
        sort_keys<TH>(sm, n);
        if (pass < 2) n = min(n, k);
        // neighbours per thread: masses, their running sum, and how many pass the filters -- all keep a leading part
        constexpr int EACH = kList / TH;
        u64 m[EACH], sum = 0, whole;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int i = EACH * tid + j;
            m[j] = i < n ? row.mass(value_of(sm.l.all[i])) : 0;
            sm.l.mass[i] = m[j];
            sum += m[j];
        }
        u64 run = block_before<TH>(sum, sm.ws, &whole);
        const double target = by_p ? fmax((double)p * (double)(q.need ? whole : q.of), 1.0) : 0.0;
        unsigned stay = 0;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int i = EACH * tid + j;
            if (i < n) stay += i == 0 || ((!by_p || (double)run < target) && m[j] >= least);
            run += m[j];
        }
        unsigned kept;
        block_before<TH>(stay, sm.wc, &kept);
        u64 mine = 0, total;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if (EACH * tid + j < (int)kept) mine += m[j];
        block_before<TH>(mine, sm.ws, &total);
        const double aim = aim_at(total);
        for (int i = tid; i < (int)kept; i += TH) {  // mass of the kept ones with a lower index
            const unsigned at = (unsigned)sm.l.all[i];
            u64 below = 0;
            for (int j = 0; j < (int)kept; ++j)
                if ((unsigned)sm.l.all[j] < at) below += sm.l.mass[j];
            if ((double)below <= aim && (double)(below + sm.l.mass[i]) > aim) answer((int)at, value_of(sm.l.all[i]), total);
        }
        return;
    }

    // ---- the whole cluster: by index, the first at which the kept mass exceeds what u points at.  Warps own contiguous parts.
    auto kept_mass = [&](float v, int i) -> u64 {
        const u64 m = row.mass(v);
        return cut.keeps(v, s.first + i) && m >= least ? m : 0;
    };
    const int per = (s.n + (TH / 32) - 1) / (TH / 32), w0 = min(s.n, warp * per), w1 = min(s.n, w0 + per);
    u64 m = 0;
    if (cut.value == -INFINITY && least == 0) each(s, w0 + lane, w1, 32, [&](float v, int) { m += row.mass(v); });
    else if (least == 0) each(s, w0 + lane, w1, 32, [&](float v, int i) { if (cut.keeps(v, s.first + i)) m += row.mass(v); });
    else each(s, w0 + lane, w1, 32, [&](float v, int i) { m += kept_mass(v, i); });
    m = warp_add(m);
    if (lane == 0) sm.ws[warp] = m;
    __syncthreads();
    u64 all = 0, total = 0, before = 0;
    for (int w = 0; w < (TH / 32); ++w) all += sm.ws[w];
    if (tid < s.ranks) cl.map_shared_rank(sm.part, tid)[s.rank] = all;
    cl.sync();
    for (int c = 0; c < s.ranks; ++c) {
        if (c < s.rank) before += sm.part[c];
        total += sm.part[c];
    }
    const double aim = aim_at(total);
    if (!((double)before <= aim && (double)(before + all) > aim)) return;  // (one CTA goes on)
    int target = (TH / 32) - 1;
    for (int w = 0; w < (TH / 32); ++w) {
        if ((double)(before + sm.ws[w]) > aim) {
            target = w;
            break;
        }
        before += sm.ws[w];
    }
    __syncthreads();
    const int q0 = min(s.n, target * per), q1 = min(s.n, q0 + per);
    const int share = (q1 - q0 + TH - 1) / TH, i0 = min(q1, q0 + tid * share), i1 = min(q1, i0 + share);
    m = 0;
    for (int i = i0; i < i1; ++i) m += kept_mass(s[i], i);
    u64 run = before + block_before<TH>(m, sm.ws, &all);
    if ((double)run <= aim && (double)(run + m) > aim) {
        for (int i = i0; i < i1; ++i) {
            run += kept_mass(s[i], i);
            if ((double)run > aim) {
                answer(s.first + i, s[i], total);
                break;
            }
        }
    }
}

size_t sample_smem(int slice, bool bf16) { return (sizeof(SampleSmem) + 15) / 16 * 16 + (size_t)slice * (bf16 ? 2 : 4) + 16; }

}  // namespace

int launch_sample(const void *logits, int xdtype, int64_t batch, int64_t vocab, int64_t row_stride, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *u, int *tokens, float *prob, cudaStream_t s) {
    SampleArgs a;
    a.logits = logits;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.u = u;
    a.tokens = tokens;
    a.prob = prob;
    a.row_stride = row_stride;
    a.vocab = (int)vocab;
    // A larger cluster while slices are above 28 KiB, or while SMs would stay without a CTA and slices are above 2048 logits.
    const bool bf16 = xdtype == DMC_X_BF16;
    const int64_t few = bf16 ? 14336 : 7168;  // 28 KiB
    unsigned cluster = 1;
    while (cluster < kMaxCluster && (vocab > few * cluster || (vocab > (int64_t)2048 * cluster && batch * cluster <= ctx().sm_count)))
        cluster *= 2;
    a.slice = (int)((vocab + cluster - 1) / cluster + 7) / 8 * 8;
    const int threads = a.slice <= few ? 256 : 512;
    // More clusters than fit at once: the slow rows first, lest one of them begins last (64 rows of 128000, filters mixed: 71 us
    // in order, 60 so; 24 rows of 262144 f32, of which one slice fills an SM: 59 and 46; looking at the filters costs 2 us where
    // none is set: 256 rows of 50257 35 us in order, 37 so).  By registers 1024 threads fit on an SM, by shared memory (228 KiB,
    // of which each CTA takes 1 KiB more than it asks for) fewer once an f32 slice is above 100 KiB.
    const int64_t per_sm = std::min<int64_t>(1024 / threads, (228 << 10) / (int64_t)(sample_smem(a.slice, bf16) + 1024));
    const int64_t at_once = ctx().sm_count * per_sm / cluster;
    a.batch = batch > at_once && batch <= kRowsEach * threads && (top_k || top_p) ? (int)batch : 0;
    const void *fn = threads == 256 ? (bf16 ? (const void *)sample_kernel<256, true> : (const void *)sample_kernel<256, false>)
                                    : (bf16 ? (const void *)sample_kernel<512, true> : (const void *)sample_kernel<512, false>);
    DMC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sample_smem(kMaxSlice, bf16)));
    void *params[] = {&a};
    return launch_on(fn, dim3((unsigned)(batch * cluster)), dim3(threads), sample_smem(a.slice, bf16), s, params,
                     cluster);
}

}  // namespace dmc

using namespace dmc;

extern "C" int dmc_cuda_sample(const void *logits, int xdtype, int64_t batch, int64_t vocab, int64_t row_stride,
                               const float *temperature, const int *top_k, const float *top_p, const float *min_p, const float *u,
                               int *tokens, float *prob, void *stream) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    OnDevice on;
    if (xdtype != DMC_X_BF16 && xdtype != DMC_X_F32) return fail(DMC_CUDA_ERR_BAD_ARG, "sample: unknown xdtype %d", xdtype);
    if (batch < 0 || vocab < 1 || row_stride < vocab)
        return fail(DMC_CUDA_ERR_BAD_ARG, "sample: batch %lld, vocab %lld, row_stride %lld", (long long)batch, (long long)vocab,
                    (long long)row_stride);
    if (vocab > kSampleMaxVocab || batch > INT32_MAX / kMaxCluster)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "sample: vocab beyond %d or batch beyond %d", kSampleMaxVocab, INT32_MAX / kMaxCluster);
    if (batch == 0) return DMC_CUDA_OK;
    int rc = enter_device({{logits, (size_t)(xdtype == DMC_X_BF16 ? 2 : 4), "logits"}, {tokens, 4, "tokens"},
                           {temperature, 4, "temperature", true}, {top_k, 4, "top_k", true}, {top_p, 4, "top_p", true},
                           {min_p, 4, "min_p", true}, {u, 4, "u"}, {prob, 4, "prob", true}});
    if (rc) return rc;
    return launch_sample(logits, xdtype, batch, vocab, row_stride, temperature, top_k, top_p, min_p, u, tokens, prob, (cudaStream_t)stream);
}
