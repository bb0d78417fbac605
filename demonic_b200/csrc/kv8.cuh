// kv8.cuh -- device side of the 8-bit paged KV cache: append and attention.
//
// Codes are e4m3 [layers][pages][kv_heads][page_tokens][head_dim], one f32 scale per (layer, page, kv head); the
// pages of a sequence are named by its row of the table.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dmc_cuda.h"
#include "gemv.cuh"

namespace dmc {

namespace cg = cooperative_groups;

constexpr int kKv8MinExp = -40, kKv8MaxExp = 40;  // exponents of a page's scale

// One layer of a cache, as the kernels take it.
struct Kv8Layer {
    uint8_t *k, *v;
    float *ks, *vs;
    int pages, hk, page_shift;  // page_tokens = 1 << page_shift
};

struct Kv8Rows {  // which sequences a launch works on
    const int *table, *lens, *slot_ids;
    int *flags;
    long long table_stride;
    int slots, batch, tokens;
    int cap;  // tokens a row of the table can name
    int report;  // also set bits in *flags for bad rows (one kernel of a call does)
    const float *cos, *sin;  // [position][head_dim / 2]: rotate K and q on their way (the decode step); or null
};

// RoPE on 4 neighbouring elements of a head, pairs (2i, 2i + 1), dims d .. d + 3 (docs/STDLIB.md:185-202).
template <int HD>
__device__ __forceinline__ float4 kv8_rotate(const Kv8Rows &r, float4 x, int pos, int d) {
    const float2 c = *reinterpret_cast<const float2 *>(r.cos + (size_t)pos * (HD / 2) + d / 2);
    const float2 s = *reinterpret_cast<const float2 *>(r.sin + (size_t)pos * (HD / 2) + d / 2);
    return make_float4(x.x * c.x - x.y * s.x, x.x * s.x + x.y * c.x, x.z * c.y - x.w * s.y, x.z * s.y + x.w * c.y);
}

// Slot and length of row b; false if the row is skipped or bad.
__device__ __forceinline__ bool kv8_row(const Kv8Rows &r, int b, int *slot, int *len) {
    const int s = r.slot_ids ? r.slot_ids[b] : b;
    if (s < 0 || s >= r.slots) {
        if (s != -1 && r.report) atomicOr(r.flags, DMC_KV8_BAD_SLOT);
        return false;
    }
    const int n = r.lens[s];
    if (n > r.cap) {
        if (r.report) atomicOr(r.flags, DMC_KV8_TOO_LONG);
        return false;
    }
    *slot = s;
    *len = max(n, 0);
    return true;
}

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Four e4m3 codes to two pairs of f16 (exact: e4m3 is a subset of f16).
__device__ __forceinline__ void half4_of_e4m3(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
}

// ---- append ----------------------------------------------------------------------------------------------------

// Exponent of the smallest power of two s with amax / s <= 448 = 1.75 * 2^8, limited to what a page may have.
__device__ __forceinline__ int kv8_scale_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 135 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return min(max(e, kKv8MinExp), kKv8MaxExp);
}

template <bool BF16>
__device__ __forceinline__ float4 load_row4(const void *p, size_t at) {
    if constexpr (BF16) {
        const uint2 w = *(const uint2 *)((const uint16_t *)p + at);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xFFFF0000u));
    } else {
        return *(const float4 *)((const float *)p + at);
    }
}

// 16 bytes of a row: 8 bf16 or 4 f32.  (A plain load: the kernel before may have written the row, so it must not be a read-only
// one, which would take 17.2 us instead of 17.4 for the prompt below; streaming forms took 17.7.)
template <bool BF16>
__device__ __forceinline__ uint4 load_row16(const void *p, size_t at, bool vec) {
    if (vec) return *(const uint4 *)((const char *)p + at * (BF16 ? 2 : 4));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            const uint16_t *q = (const uint16_t *)p + at + 2 * i;
            w[i] = q[0] | (uint32_t)q[1] << 16;
        } else {
            w[i] = ((const uint32_t *)p)[at + i];
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// One (row, page it touches, kv head, K or V) per group of NTHR threads: its new tokens are read once, as they are, into
// registers, their maximum decides the scale, the codes go out.  A thread holds VPT pieces of 16 bytes.
//   few tokens   a warp each (NTHR = 32): nothing to wait for but its own lanes
//   prompts      256 threads each, a whole page in registers (16 of them for bf16, so that eight CTAs run on an SM)
// Prompts are bound by issue: 3 x 4001 tokens x 8 heads x 128, K and V bf16, 74 MB in 17.4 us = 4.2 TB/s, issue slots 79 % and ALU
// 53 % busy with scaling, converting and packing; f32 123 MB in 24.0 us = 5.1 TB/s.  Converting bf16 to f32 on arrival (32 registers,
// four CTAs) took 42.  At the 32 registers that eight CTAs leave, the bf16 builds spill 56 (head_dim 128) and 28 bytes.  A batch's
// single tokens are bound by latency (length -> page -> scale): 7 us.
template <int HD, int NTHR, int VPT, bool BF16>
__global__ void __launch_bounds__(256, NTHR == 256 && BF16 ? 8 : 4) kv8_append_kernel(Kv8Layer c, Kv8Rows r, const void *kx,
                                                                                    const void *vx, long long row_stride,
                                                                                    int touch, int vec) {
    constexpr int PER = 256 / NTHR, E = BF16 ? 8 : 4, PIECES = HD / E;
    __shared__ float red[8];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x % NTHR;
    const long long item = (long long)blockIdx.x * PER + threadIdx.x / NTHR;
    if (item >= (long long)r.batch * touch * c.hk * 2) return;  // (whole groups leave; NTHR == 256: whole CTAs)
    const int h = (int)(item % c.hk);
    const int kv = (int)(item / c.hk % 2);
    const int j = (int)(item / (2 * c.hk) % touch);
    const int b = (int)(item / ((long long)2 * c.hk * touch));
    const void *x = kv ? vx : kx;
    uint4 e[VPT];
    auto load = [&](size_t row0, int n) {
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            const int i = tid + u * NTHR;
            e[u] = make_uint4(0, 0, 0, 0);
            if (i < n) e[u] = load_row16<BF16>(x, (row0 + i / PIECES) * row_stride + (size_t)h * HD + (i % PIECES) * E, vec);
        }
    };
    // a single token's values do not depend on where it goes: asked for before the length and the page are known
    const bool single = NTHR == 32 && r.tokens == 1;
    if (single) load(b, PIECES);
    int s, len;
    if (!kv8_row(r, b, &s, &len)) return;
    const int pos0 = len - r.tokens;                       // position of token 0; negative: padding on the left
    const int page = (max(pos0, 0) >> c.page_shift) + j;   // position of the page in the sequence
    const int p0 = page << c.page_shift, p1 = p0 + (1 << c.page_shift);
    const int i0 = max(max(pos0, 0), p0), i1 = min(len, p1);  // positions of the new tokens in this page
    if (i0 >= i1) return;
    const int id = r.table[(size_t)s * r.table_stride + page];
    if ((unsigned)id >= (unsigned)c.pages) {
        if (tid == 0) atomicOr(r.flags, DMC_KV8_BAD_PAGE);
        return;
    }
    const int had = i0 - p0, n = (i1 - i0) * PIECES;
    if (!single) load((size_t)b * r.tokens + (i0 - pos0), n);
    if constexpr (!BF16)
        if (r.cos && !kv) {
#pragma unroll
            for (int u = 0; u < VPT; ++u) {
                const int i = tid + u * NTHR;
                if (i >= n) break;
                float4 &y = *reinterpret_cast<float4 *>(&e[u]);
                y = kv8_rotate<HD>(r, y, i0 + i / PIECES, i % PIECES * E);
            }
        }
    float *scale_at = (kv ? c.vs : c.ks) + (size_t)id * c.hk + h;
    const float was = had ? *scale_at : 0.0f;
    float amax = 0.0f;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {  // (a maximum passes over NaN)
        const uint32_t w[4] = {e[u].x, e[u].y, e[u].z, e[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (BF16) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xFFFF0000u))));
            else amax = fmaxf(amax, fabsf(__uint_as_float(w[k])));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if constexpr (NTHR > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
        __syncthreads();
        amax = red[0];
#pragma unroll
        for (int w = 1; w < NTHR / 32; ++w) amax = fmaxf(amax, red[w]);
    }
    const float scale = fmaxf(was, __uint_as_float((uint32_t)(kv8_scale_exp(amax) + 127) << 23));
    uint32_t *codes = (uint32_t *)((kv ? c.v : c.k) + ((((size_t)id * c.hk + h) << c.page_shift) + had) * HD);
    auto store = [&](auto quot) {
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            const int i = tid + u * NTHR;
            if (i >= n) break;
            const uint32_t w[4] = {e[u].x, e[u].y, e[u].z, e[u].w};
            uint32_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (BF16) q[k] = e4m3x2(quot(__uint_as_float(w[k] << 16)), quot(__uint_as_float(w[k] & 0xFFFF0000u)));
                else q[k] = __float_as_uint(quot(__uint_as_float(w[k])));
            }
            if constexpr (BF16) *reinterpret_cast<uint2 *>(codes + 2 * i) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
            else codes[i] = e4m3x2(__uint_as_float(q[0]), __uint_as_float(q[1])) | (uint32_t)e4m3x2(__uint_as_float(q[2]), __uint_as_float(q[3])) << 16;
        }
    };
    // a power of two, but for a scale that the caller put there: dividing by it is multiplying by its inverse
    if ((__float_as_uint(scale) & 0x7FFFFFu) == 0) {
        const float inv = 1.0f / scale;
        store([&](float v) { return v * inv; });
    } else {
        store([&](float v) { return v / scale; });
    }
    if (had && scale > was) {  // the tokens that were there before go to the larger scale
        const float f = was / scale;
        uint32_t *old = codes - had * (HD / 4);
        for (int i = tid; i < had * (HD / 4); i += NTHR) {
            uint32_t lo, hi;
            half4_of_e4m3(old[i], lo, hi);
            const float2 a = __half22float2(*(const __half2 *)&lo), d = __half22float2(*(const __half2 *)&hi);
            old[i] = e4m3x2(a.x * f, a.y * f) | (uint32_t)e4m3x2(d.x * f, d.y * f) << 16;
        }
    }
    if (scale != was || !had) {
        if constexpr (NTHR > 32) __syncthreads();  // every thread has read the old scale
        else __syncwarp();
        if (tid == 0) *scale_at = scale;
    }
}

// ---- attention -------------------------------------------------------------------------------------------------
//
// S' = K . Q' and O' = V' . P' on the tensor cores by mma.sync, keys (then dims) as the 16 rows and up to 8 query rows
// (tokens x heads of the group) as the 8 columns, so that a group of 8 heads wastes nothing and a warp takes each code once.
// (tcgen05 would need 128 rows of one operand and both in one type; here one side is 8 wide and the kernel is bound by memory.
// m16n8k32 on the codes themselves is no way out: it was measured at 0.23 a clock and SM with new operands, against 0.47 for
// m16n8k16.)  The codes are converted to f16, which is exact; f32 q and
// probabilities enter as two f16 terms each (22 bits), bf16 q as one, which holds it exactly down to 2^-22 of the row's
// largest element, and its probabilities as one (11 bits).
//
// The scores of 16 keys x 8 rows leave the first product with keys on g = lane / 4 and rows on t = lane % 4; movmatrix
// transposes the f16 probabilities into the operand of the second.  K comes from shared memory by ldmatrix, V by its form
// that transposes bytes, so that a word holds four keys of one dim.  The page's K scale multiplies the scores; the exponent
// of its V scale joins the score's, so that probabilities times V scale stay in range whatever the scales are, and the
// rest (1 for a power of two) multiplies the probability.
//
// Bound by HBM for few rows: 64 sequences of 8001-16000 keys x 8 heads, 8 query heads each, 1.58 GB in 254-266 us = 6.0-6.2
// TB/s (0.91-0.95 of a plain copy's rate); the copies alone, without a product, took 255.  One sequence of 200001 keys x 4 heads: 47 us
// for 205 MB, of which 5 the join and 4 the way to the first key.  Many f32 rows are bound by issue and
// latency: 5 tokens x 4 heads as two f16 terms each, over 400 warp instructions per 16 keys x 64 dims, issue slots 43 % and
// the tensor pipe 38 % busy with the 11 warps that the registers allow, 62 us for 117 MB.
//
// A tile's rows are as many as one warp's registers carry (16, or 32 of head_dim 64; the widest builds spill 24 to 68 bytes), and each
// further tile of a head reads its keys again: 2 tokens of the 64 sequences above (16 rows) take 254 us in bf16 and 350 in f32, 5
// tokens (40 rows, three tiles) 714 and 998.  A bf16 prompt of 1000 tokens, 32 heads over 8 x 128, takes 135 us, one of 4001 1330.
constexpr int kKv8Warps = 4, kKv8MaxCluster = 8;
constexpr int kKv8Unit = 16 * kKv8Warps;  // keys that a CTA takes at a time, 16 to a warp
constexpr int kKv8Batch = 16;             // tiles of 16 keys whose places a warp looks up together
constexpr int kKv8Shift = 10;             // probabilities are kept times 2^10: f16 holds them down to 2^-34 of the reference
constexpr float kKv8Lazy = 4.0f;          // the reference maximum is renewed when a score passes it by 2^4 (2^14 < 65504)
constexpr float kKv8NoRef = 3e38f;        // before a row's first key
// A piece of a sequence costs about as much as this many units more: its look-ups, q, and joining the warps.
constexpr int kKv8Piece = 5;

struct Kv8AttnArgs {
    Kv8Layer c;
    Kv8Rows r;
    const void *q;
    void *out;
    long long q_stride, out_stride;
    float *part_o;      // [ctas][2][8 NT][HD] sums of probability x value, not divided yet
    float2 *part_ml;    // [ctas][2][8 NT] reference maximum, sum of probabilities
    int2 *segs;         // [batch][kv heads][row tiles]: first part (CTA * 2 + which) or -1, last CTA
    float scale_log2;   // softmax scale * log2(e)
    int group;          // query heads per kv head
    int row_tiles;
    int ctas;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// 16 rows x 32 bytes as they lie: lane (g, t) gets bytes 4t.. of rows g and g + 8, then bytes 16 + 4t..
__device__ __forceinline__ void load_rows(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
// Twice 16 rows x 16 bytes, transposed: lane (g, t) gets column g of rows 4t.., column g + 8, then the same of the second
__device__ __forceinline__ void load_columns(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t *)&h;
}
// The part of (a, b) that their f16 pair `hi` leaves.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*(const __half2 *)&hi);
    return pack_half2(a - f.x, b - f.y);
}
template <bool BF16>
__device__ __forceinline__ void store_row4(void *p, size_t at, float4 z) {
    if constexpr (BF16) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(z.x, z.y), hi = __floats2bfloat162_rn(z.z, z.w);
        *reinterpret_cast<uint2 *>((uint16_t *)p + at) = make_uint2(*(const uint32_t *)&lo, *(const uint32_t *)&hi);
    } else {
        *reinterpret_cast<float4 *>((float *)p + at) = z;
    }
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void *src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's tiles (16 keys) come through a ring of its own in shared memory, filled by 16-byte asynchronous copies: what is in
// flight costs no registers, so an SM holds enough warps.  Chunks are stored permuted (chunk ^ some bits of the row) so that
// neither the K reads (rows 0-7 of a chunk) nor the V reads (rows 0, 1, 8, 9, 2, 3, 10, 11) meet in a bank.
template <int HD>
struct Kv8Ring {
    static constexpr int kTile = 16 * HD;  // bytes, K or V
    static constexpr int kStages = HD == 128 ? 3 : 4;
    static constexpr int ctas_per_sm(int nt) { return HD == 128 ? (nt == 1 ? 4 : 3) : (nt <= 2 ? 4 : 3); }
    // byte offset of 16-byte chunk c of row r
    __device__ static __forceinline__ int at(int r, int c) {
        const int b0 = r & 1, b1 = r >> 1 & 1, b2 = r >> 2 & 1, b3 = r >> 3 & 1;
        return HD == 128 ? r * 128 + ((c ^ (r & 3) ^ (b2 ^ b3) << 2) << 4)
                         : (r >> 1) * 128 + ((b0 << 2 | (c ^ b1 ^ (b2 ^ b3) << 1)) << 4);
    }
};

template <int HD, int NT, bool BF16>
struct Kv8Smem {
    using Ring = Kv8Ring<HD>;
    static constexpr int NR = 8 * NT;
    uint4 q[BF16 ? 1 : 2][NT][HD / 32][32];  // B fragments of 32 dims, high and low terms
    float fac[NR];                           // what a row's products are multiplied by
    float m[kKv8Warps][NR], l[kKv8Warps][NR];
    float2 ml[NR];                           // of the CTA's part of a row, for the others of its cluster
    // of the warps' tiles, two batches: K scale, exponent e of the V scale, 2^-e, V scale times 2^-e; first code, or -1
    float4 scale[kKv8Warps][2 * kKv8Batch];
    long long at[kKv8Warps][2 * kKv8Batch];
    union alignas(128) {
        unsigned char ring[kKv8Warps][Ring::kStages][2][Ring::kTile];
        float o[kKv8Warps][NR][HD + 4];  // the warps' results, once their rings are empty
    };
};

// Two arrangements.  CLUSTER = false: a fixed number of CTAs share all segments evenly, whatever the lengths, and a second kernel
// joins the parts of a row.  CLUSTER = true: a segment to a cluster, its keys cut evenly among the CTAs, which join their parts
// through distributed shared memory: one launch and no partial results in memory, for few and short segments.
template <int HD, int NT, bool BF16, bool CLUSTER>
__global__ void __launch_bounds__(128, Kv8Ring<HD>::ctas_per_sm(NT)) kv8_attn_kernel(Kv8AttnArgs a) {
    using Ring = Kv8Ring<HD>;
    constexpr int NR = 8 * NT, MT = HD / 16, S = Ring::kStages, TERMS = BF16 ? 1 : 2, UNIT = kKv8Unit;
    constexpr int COPIES = HD / 32;  // 16-byte copies per lane for a tile of K or V
    constexpr float SHIFT = (float)kKv8Shift;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Kv8Smem<HD, NT, BF16> &sm = *reinterpret_cast<Kv8Smem<HD, NT, BF16> *>(smem_raw);
    __shared__ long long sh_at, wsum[kKv8Warps];
    __shared__ int sh_row;
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int per = a.c.hk * a.row_tiles;  // segments (kv head, row tile) per row of the batch

    // ---- this CTA's share: all segments in a line, each as long as its units and kPiece more, cut into equal parts
    auto units_of = [&](int b, int *slot, int *len) -> int {
        if (!kv8_row(a.r, b, slot, len)) return 0;
        return max(1, (*len + UNIT - 1) / UNIT);  // (an empty sequence has one, to write its zeros)
    };
    auto length_of = [&](int b) -> long long {
        int slot, len;
        const int n = units_of(b, &slot, &len);
        return n ? (long long)(n + kKv8Piece) * per : 0;
    };
    long long total = 0, u0 = 0, u1 = 1, G = a.ctas;
    int b = 0;
    long long row_at = 0;
    if constexpr (!CLUSTER) {
    if (a.r.batch > 128) {
        for (int b = tid; b < a.r.batch; b += 128) total += length_of(b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) wsum[warp] = total;
        __syncthreads();
        total = wsum[0] + wsum[1] + wsum[2] + wsum[3];
        __syncthreads();
    }
    long long base = 0;
    for (int b0 = 0; b0 < a.r.batch; b0 += 128) {  // the row of the batch that the share starts in
        const int b = b0 + tid;
        const long long n = b < a.r.batch ? length_of(b) : 0;
        long long inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        for (int w = 0; w < warp; ++w) inc += wsum[w];
        inc += base;
        base += wsum[0] + wsum[1] + wsum[2] + wsum[3];
        if (a.r.batch <= 128) total = base;
        G = min((long long)a.ctas, total);  // nobody is left without a share in the middle
        if (blockIdx.x >= G) return;
        u0 = total * blockIdx.x / G;
        if (n && inc - n <= u0 && u0 < inc) {
            sh_row = b;
            sh_at = inc - n;
        }
        __syncthreads();
        if (base > u0) break;
    }
    u1 = total * (blockIdx.x + 1) / G;
    b = sh_row;
    row_at = sh_at;
    }
    bool first = true;

    // where this lane's chunks go in a tile and where its fragments come from
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(&sm.ring[warp][0][0][0]);
    const int crow = lane / (HD / 16), cchunk = lane % (HD / 16);  // its first chunk; the next ones 512 bytes on
    int put[COPIES], kat[HD / 32], vat[HD / 32];
#pragma unroll
    for (int j = 0; j < COPIES; ++j) put[j] = Ring::at(crow + j * (512 / HD), cchunk);
    // K: lanes 0-7 name rows 0-7 of an even chunk, 8-15 rows 8-15, 16-31 the same of the odd chunk.  V: lanes 0-15 name the rows
    // of an even chunk in the order in which the transposed probabilities come, 4t + i being key 2t, 2t + 1, 2t + 8, 2t + 9.
    const int vrow = 2 * (lane >> 2 & 3) + (lane & 1) + 8 * (lane >> 1 & 1);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        kat[i] = Ring::at(lane & 15, 2 * i + (lane >> 4));
        vat[i] = Ring::kTile + Ring::at(vrow, 2 * i + (lane >> 4));
    }

    for (long long u = u0; u < u1;) {
        int slot = 0, len = 0, units, seg, a0, a1;  // seg: (head, row tile); units a0 .. a1 - 1 of it are done here
        if constexpr (CLUSTER) {
            const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
            b = blockIdx.x / ranks / per;
            seg = blockIdx.x / ranks % per;
            units = units_of(b, &slot, &len);
            if (units == 0) return;  // (the whole cluster)
            a0 = (int)((long long)units * rank / ranks);
            a1 = (int)((long long)units * (rank + 1) / ranks);
            u = u1;
        } else {
            units = units_of(b, &slot, &len);
            while (units == 0 || u >= row_at + (long long)(units + kKv8Piece) * per) {
                if (units) row_at += (long long)(units + kKv8Piece) * per;
                units = units_of(++b, &slot, &len);
            }
            const int span = units + kKv8Piece;
            seg = (int)((u - row_at) / span);
            const long long seg0 = row_at + (long long)seg * span;
            a0 = max(0, (int)(u - seg0) - kKv8Piece);
            a1 = max(0, (int)min((long long)span, u1 - seg0) - kKv8Piece);
            u = min(u1, seg0 + span);
            if (a1 <= a0) continue;
        }
        const int h = seg / a.row_tiles, rt = seg % a.row_tiles;
        const int T = a.r.tokens, rows = T * a.group;
        const int *ids = a.r.table + (size_t)slot * a.r.table_stride;

        // ---- this warp's tiles: 16 keys from key_first, key_first + UNIT, ...  Where they are and their scales are fetched
        // kKv8Batch at a time, one tile per lane, and left in shared memory half a batch later.
        // No key is fetched that no row of the tile sees.
        const int seen = len - T + (min(rows, (rt + 1) * NR) - 1) / a.group + 1;
        const int key_first = a0 * UNIT + warp * 16, end = min(min(len, seen), a1 * UNIT);
        const int tiles = key_first < end ? (end - key_first + UNIT - 1) / UNIT : 0;
        struct Pages {
            long long at;
            float ks, vs;
        };
        auto pages_of = [&](int tile0) {
            Pages p{-1, 0.0f, 0.0f};
            const int key0 = key_first + (tile0 + lane) * UNIT;
            if (lane < kKv8Batch && tile0 + lane < tiles) {
                const int id = ids[key0 >> a.c.page_shift];
                if ((unsigned)id < (unsigned)a.c.pages) {
                    const size_t head = (size_t)id * a.c.hk + h;
                    p.at = (long long)(((head << a.c.page_shift) + (key0 & ((1 << a.c.page_shift) - 1))) * HD);
                    p.ks = a.c.ks[head];
                    p.vs = a.c.vs[head];
                } else {
                    atomicOr(a.r.flags, DMC_KV8_BAD_PAGE);
                }
            }
            return p;
        };
        auto keep_pages = [&](const Pages &p, int tile0) {
            if (lane < kKv8Batch) {
                const int i = (tile0 & kKv8Batch) + lane;
                // (exponent 0 for a scale of 0)
                const int e = p.vs != 0.0f ? min(max((int)(__float_as_uint(p.vs) >> 23 & 255) - 127, -48), 48) : 0;
                const float back = __uint_as_float((uint32_t)(127 - e) << 23);
                sm.at[warp][i] = p.at;
                sm.scale[warp][i] = make_float4(p.ks, (float)e, back, p.vs * back);
            }
            __syncwarp();
        };
        int stage_in = 0;  // ring slot that the next fetch fills
        // A tile without a page is not fetched, and passed over below.
        auto fetch = [&](int tile) {
            const long long from = tile < tiles ? sm.at[warp][tile % (2 * kKv8Batch)] : -1;
            if (from >= 0) {
                const int key0 = key_first + tile * UNIT;
                const uint8_t *kp = a.c.k + from + lane * 16, *vp = a.c.v + from + lane * 16;
                const uint32_t to = ring + stage_in * (2 * Ring::kTile);
#pragma unroll
                for (int j = 0; j < COPIES; ++j) copy16(to + put[j], kp + j * 512);
                if (key0 + 16 <= len) {
#pragma unroll
                    for (int j = 0; j < COPIES; ++j) copy16(to + Ring::kTile + put[j], vp + j * 512);
                } else {  // values behind the end may be anything, NaN too, and 0 * NaN would reach the sums
#pragma unroll
                    for (int j = 0; j < COPIES; ++j)
                        copy16_or_zero(to + Ring::kTile + put[j], vp + j * 512, key0 + crow + j * (512 / HD) < len);
                }
            }
            copy_commit();
            stage_in = stage_in == S - 1 ? 0 : stage_in + 1;
        };
        __syncthreads();  // the rings' memory held the last segment's results
        keep_pages(pages_of(0), 0);
        Pages ahead = pages_of(kKv8Batch);
#pragma unroll
        for (int i = 0; i < S - 1; ++i) fetch(i);

        // ---- Q rows of the tile as B fragments in shared memory, each row times a power of two
        for (int i = warp; i < NR; i += kKv8Warps) {
            const int row = rt * NR + i;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < rows && lane < HD / 4) {
                const size_t at = ((size_t)b * T + row / a.group) * a.q_stride + (size_t)(h * a.group + row % a.group) * HD + lane * 4;
                x = load_row4<BF16>(a.q, at);
                if (!BF16 && a.r.cos) x = kv8_rotate<HD>(a.r, x, max(0, len - T + row / a.group), lane * 4);
            }
            float mx = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            // 2^(7 - exponent): the largest element lands in [2^7, 2^8)
            const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -119), 127);
            const float f = __uint_as_float((uint32_t)(127 + 7 - e) << 23), back = __uint_as_float((uint32_t)(127 + e - 7) << 23);
            if (lane < HD / 4) {
                x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
                // dims 4 lane ..: lane t of chunk lane / 4
                uint2 *to = reinterpret_cast<uint2 *>(&sm.q[0][i / 8][lane / 8][(i % 8) * 4 + lane % 4]) + (lane >> 2 & 1);
                const uint2 hi = make_uint2(pack_half2(x.x, x.y), pack_half2(x.z, x.w));
                *to = hi;
                if (!BF16) to[NT * (HD / 32) * 64] = make_uint2(pack_rest(x.x, x.y, hi.x), pack_rest(x.z, x.w, hi.y));
            }
            if (lane == 0) sm.fac[i] = back * a.scale_log2;
        }
        __syncthreads();

        // ref: kShift minus the reference maximum (in units of log2) of a column
        float fac[NT][2], ref[NT][2], lsum[NT][2];
        int lim[NT][2];  // keys a row sees
        float o[NT][MT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = n * 8 + 2 * t + x, row = rt * NR + i;
                fac[n][x] = sm.fac[i];
                ref[n][x] = kKv8NoRef;
                lsum[n][x] = 0.0f;
                lim[n][x] = row < rows ? len - T + row / a.group + 1 : 0;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        }
        const int whole = len - T + 1;  // keys that every row of the sequence sees

        auto compute = [&](uint32_t mem, int key0, const float4 &scale) {
            const bool edge = key0 + 16 > whole;
            // The low terms' products by themselves, as far as the registers go: the tensor core cuts off what lies below a sum's
            // last place (16 heads x 513 keys: 3.6e-7 off in all, against 7.5e-7 in one sum; 24 rows: 4 us of 64 more apart).
            constexpr bool APART = !BF16 && NT <= 2;
            float s[NT][4], low[APART ? NT : 1][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][i] = 0.0f;
                    if (APART) low[n][i] = 0.0f;
                }
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                uint32_t w[4], c[8];
                load_rows(w, mem + kat[i]);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    half4_of_e4m3(w[2 * k], c[4 * k], c[4 * k + 2]);
                    half4_of_e4m3(w[2 * k + 1], c[4 * k + 1], c[4 * k + 3]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
                        const uint4 q = sm.q[k][n][i][lane];
                        float(&sum)[4] = APART && k ? low[APART ? n : 0] : s[n];
                        mma_f16(sum, c[0], c[1], c[2], c[3], q.x, q.y);
                        mma_f16(sum, c[4], c[5], c[6], c[7], q.z, q.w);
                    }
            }
            if constexpr (APART) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][i] += low[n][i];
            }
            // A score (with the V scale's exponent) is s kf + ev; it is rounded only once the reference has been taken off.
            float kf[NT][2], ev = scale.y, z[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) kf[n][i] = scale.x * fac[n][i];
            if (edge) {  // the score itself, -inf where it is not seen
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[n][i] = key0 + g + (i >> 1) * 8 >= lim[n][i & 1] ? -INFINITY : fmaf(s[n][i], kf[n][i & 1], ev);
                    kf[n][0] = kf[n][1] = 1.0f;
                }
                ev = 0.0f;
            }
            auto exponents = [&]() {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        z[n][i] = fmaf(s[n][i], kf[n][i & 1], ev + ref[n][i & 1]);
                        top = fmaxf(top, z[n][i]);
                    }
                return top;
            };
            if (__any_sync(0xffffffffu, exponents() > SHIFT + kKv8Lazy)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float m = fmaxf(fmaf(s[n][i], kf[n][i], ev), fmaf(s[n][i + 2], kf[n][i], ev));
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
                        const float r = fminf(ref[n][i], SHIFT - m), down = exp2_approx(r - ref[n][i]);
                        ref[n][i] = r;
                        lsum[n][i] *= down;
#pragma unroll
                        for (int j = 0; j < MT; ++j) o[n][j][i] *= down, o[n][j][i + 2] *= down;
                    }
                exponents();
            }
            uint32_t p[NT][TERMS][2];  // the probabilities as B fragments: keys 2t, 2t + 1, then 2t + 8, 2t + 9 of row g
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float pr = exp2_approx(z[n][i]);
                    lsum[n][i & 1] = fmaf(pr, scale.z, lsum[n][i & 1]);
                    s[n][i] = pr * scale.w;
                }
                const uint32_t h0 = pack_half2(s[n][0], s[n][1]), h1 = pack_half2(s[n][2], s[n][3]);
                p[n][0][0] = movmatrix(h0), p[n][0][1] = movmatrix(h1);
                if constexpr (!BF16) {
                    p[n][1][0] = movmatrix(pack_rest(s[n][0], s[n][1], h0));
                    p[n][1][1] = movmatrix(pack_rest(s[n][2], s[n][3], h1));
                }
            }
            auto product = [&](float (&acc)[4], const uint32_t *c, int n) {
#pragma unroll
                for (int k = 0; k < TERMS; ++k) mma_f16(acc, c[0], c[1], c[2], c[3], p[n][k][0], p[n][k][1]);
            };
            // dims 32 i + g, + 8, + 16, + 24: bytes of keys 2t, 2t + 1, 2t + 8, 2t + 9
            auto fragments = [&](const uint32_t (&w)[4], uint32_t (&c)[8]) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    half4_of_e4m3(w[2 * k], c[4 * k], c[4 * k + 2]);
                    half4_of_e4m3(w[2 * k + 1], c[4 * k + 1], c[4 * k + 3]);
                }
            };
            // A NaN that only later rows see must not reach the earlier ones as 0 * NaN.
            bool nan = false;
            if (T > 1 && edge) {
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    uint32_t w[4];
                    load_columns(w, mem + vat[i]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) nan |= (((w[k] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
                }
                nan = __any_sync(0xffffffffu, nan);
            }
            if (nan) {
#pragma unroll 1
                for (int seen = 1; seen <= 16; ++seen) {  // the columns that see so many of the tile's keys, with those alone
                    uint32_t keep = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (2 * t + (j & 1) + (j >> 1) * 8 < seen) keep |= 0xFFu << (8 * j);
#pragma unroll
                    for (int i = 0; i < HD / 32; ++i) {
                        uint32_t w[4], c[8];
                        load_columns(w, mem + vat[i]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] &= keep;
                        fragments(w, c);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                product(acc, c + 4 * j, n);
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (min(lim[n][k & 1] - key0, 16) == seen) o[n][2 * i + j][k] += acc[k];
                            }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    uint32_t w[4], c[8];
                    load_columns(w, mem + vat[i]);
                    fragments(w, c);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int n = 0; n < NT; ++n) product(o[n][2 * i + j], c + 4 * j, n);
                }
            }
        };

        int stage = 0;
        for (int tile = 0; tile < tiles; ++tile) {
            if (tile % kKv8Batch == kKv8Batch / 2) keep_pages(ahead, tile + kKv8Batch / 2);
            else if (tile % kKv8Batch == 0 && tile) ahead = pages_of(tile + kKv8Batch);
            copy_wait<S - 2>();
            __syncwarp();  // everybody's copies of this tile are there; everybody is done with the tile before it
            fetch(tile + S - 1);
            const int i = tile % (2 * kKv8Batch);
            if (sm.at[warp][i] >= 0) compute(ring + stage * (2 * Ring::kTile), key_first + tile * UNIT, sm.scale[warp][i]);
            stage = stage == S - 1 ? 0 : stage + 1;
        }
        copy_wait<0>();
        // Not before: the next kernel's CTAs would take the places of finished ones and, with another partition of the SM's
        // memory, keep this kernel's successor from getting all of its own at once (64 x 12000 keys: 355 us a call against 263).
        if (u >= u1) griddep_launch_dependents();
        __syncthreads();  // the rings are empty

        // ---- the four warps' results
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = n * 8 + 2 * t + x;
                float l = lsum[n][x];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
                if (g == 0) sm.m[warp][i] = ref[n][x] == kKv8NoRef ? -INFINITY : -ref[n][x], sm.l[warp][i] = l;
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    float *to = &sm.o[warp][i][0];
                    to[16 * j + g] = o[n][j][x];
                    to[16 * j + g + 8] = o[n][j][x + 2];
                }
            }
        __syncthreads();
        const bool complete = a0 == 0 && a1 == units;
        const int which = blockIdx.x * 2 + (first ? 0 : 1);
        if (!CLUSTER && tid == 0) {
            int2 *s = a.segs + (size_t)b * per + seg;
            if (a0 == 0) s->x = complete ? -1 : which;
            if (a1 == units) s->y = blockIdx.x;
        }
        for (int i = tid / (HD / 4); i < NR; i += 128 / (HD / 4)) {
            const int d = tid % (HD / 4) * 4, row = rt * NR + i;
            if (row >= rows) break;
            float M = -INFINITY, L = 0.0f;
            float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kKv8Warps; ++w) M = fmaxf(M, sm.m[w][i]);
#pragma unroll
            for (int w = 0; w < kKv8Warps; ++w) {
                const float f = sm.m[w][i] == -INFINITY ? 0.0f : exp2_approx(sm.m[w][i] - M);
                const float4 y = *reinterpret_cast<const float4 *>(&sm.o[w][i][d]);
                L = fmaf(sm.l[w][i], f, L);
                z.x = fmaf(y.x, f, z.x), z.y = fmaf(y.y, f, z.y), z.z = fmaf(y.z, f, z.z), z.w = fmaf(y.w, f, z.w);
            }
            if constexpr (CLUSTER) {
                *reinterpret_cast<float4 *>(&sm.o[0][i][d]) = z;  // (this thread alone has read it)
                if (d == 0) sm.ml[i] = make_float2(M, L);
            } else if (complete) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                const size_t at = ((size_t)b * T + row / a.group) * a.out_stride + (size_t)(h * a.group + row % a.group) * HD + d;
                store_row4<BF16>(a.out, at, make_float4(z.x * inv, z.y * inv, z.z * inv, z.w * inv));
            } else {
                *reinterpret_cast<float4 *>(a.part_o + ((size_t)which * NR + i) * HD + d) = z;
                if (d == 0) a.part_ml[(size_t)which * NR + i] = make_float2(M, L);
            }
        }
        first = false;
        if constexpr (CLUSTER) {
            cg::cluster_group cl = cg::this_cluster();
            const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
            cl.sync();
            // rows are shared out among the CTAs
            for (int i = rank + ranks * (tid / (HD / 4)); i < NR; i += ranks * (128 / (HD / 4))) {
                const int d = tid % (HD / 4) * 4, row = rt * NR + i;
                if (row >= rows) break;
                float2 ml[kKv8MaxCluster];
                float4 y[kKv8MaxCluster];
#pragma unroll
                for (int c = 0; c < kKv8MaxCluster; ++c) {
                    if (c >= ranks) break;
                    const Kv8Smem<HD, NT, BF16> *o = cl.map_shared_rank(&sm, c);
                    ml[c] = o->ml[i];
                    y[c] = *reinterpret_cast<const float4 *>(&o->o[0][i][d]);
                }
                float M = -INFINITY, L = 0.0f;
                float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int c = 0; c < kKv8MaxCluster; ++c)
                    if (c < ranks) M = fmaxf(M, ml[c].x);
#pragma unroll
                for (int c = 0; c < kKv8MaxCluster; ++c) {
                    if (c >= ranks) break;
                    const float f = ml[c].x == -INFINITY ? 0.0f : exp2_approx(ml[c].x - M);
                    L = fmaf(ml[c].y, f, L);
                    z.x = fmaf(y[c].x, f, z.x), z.y = fmaf(y[c].y, f, z.y), z.z = fmaf(y[c].z, f, z.z), z.w = fmaf(y[c].w, f, z.w);
                }
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                const size_t at = ((size_t)b * T + row / a.group) * a.out_stride + (size_t)(h * a.group + row % a.group) * HD + d;
                store_row4<BF16>(a.out, at, make_float4(z.x * inv, z.y * inv, z.z * inv, z.w * inv));
            }
            cl.sync();  // (the others have read this CTA's part)
        }
    }
}

// Rows whose keys were split over several CTAs: one CTA per `rpc` rows of a segment.  The parts' maxima and sums first, a warp
// per row, then their values weighted, HD / 4 threads per part and row, several parts of a row side by side.
constexpr int kKv8MaxCtas = 1024, kKv8JoinRows = 8;

template <int HD, bool BF16>
__global__ void __launch_bounds__(256) kv8_attn_join_kernel(Kv8AttnArgs a, int nr, int rpc) {
    constexpr int LANES = HD / 4, SETS = 256 / LANES;
    __shared__ float weight[kKv8JoinRows * kKv8MaxCtas], total[kKv8JoinRows];
    __shared__ float4 sums[SETS][LANES];
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, T = a.r.tokens, rows = T * a.group;
    const int groups = (nr + rpc - 1) / rpc;
    const int i0 = blockIdx.x % groups * rpc;
    const int seg = blockIdx.x / groups, rt = seg % a.row_tiles, h = seg / a.row_tiles % a.c.hk, b = seg / a.row_tiles / a.c.hk;
    const int n_rows = min(rpc, min(nr, rows - rt * nr) - i0);
    const int2 span = a.segs[seg];
    int slot, len;
    if (n_rows <= 0 || !kv8_row(a.r, b, &slot, &len) || span.x < 0) return;
    const int c0 = span.x >> 1, parts = span.y - c0 + 1;
    // the first CTA may have come to this segment after another one; the rest start with it
    auto part_of = [&](int k) { return (size_t)(k == 0 ? span.x : (c0 + k) * 2) * nr + i0; };
    for (int r = warp; r < n_rows; r += 8) {
        float M = -INFINITY, L = 0.0f;
        for (int k = lane; k < parts; k += 32) M = fmaxf(M, weight[r * parts + k] = a.part_ml[part_of(k) + r].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        for (int k = lane; k < parts; k += 32) {
            const float m = weight[r * parts + k], f = m == -INFINITY ? 0.0f : exp2_approx(m - M);
            weight[r * parts + k] = f;
            L = fmaf(a.part_ml[part_of(k) + r].y, f, L);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane == 0) total[r] = L;
    }
    __syncthreads();
    // sets of threads: `side` of them share a row
    const int d = tid % LANES, set = tid / LANES, side = max(1, SETS / rpc);
    for (int r0 = 0; r0 < n_rows; r0 += SETS / side) {
        const int r = r0 + set / side;
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n_rows) {
#pragma unroll 8
            for (int k = set % side; k < parts; k += side) {
                const float f = weight[r * parts + k];
                const float4 y = __ldcg(reinterpret_cast<const float4 *>(a.part_o + (part_of(k) + r) * HD) + d);
                z.x = fmaf(y.x, f, z.x), z.y = fmaf(y.y, f, z.y), z.z = fmaf(y.z, f, z.z), z.w = fmaf(y.w, f, z.w);
            }
        }
        sums[set][d] = z;
        __syncthreads();
        if (r < n_rows && set % side == 0) {
            for (int k = 1; k < side; ++k) {
                const float4 y = sums[set + k][d];
                z.x += y.x, z.y += y.y, z.z += y.z, z.w += y.w;
            }
            const int row = rt * nr + i0 + r;
            const float inv = total[r] == 0.0f ? 0.0f : 1.0f / total[r];
            const size_t at = ((size_t)b * T + row / a.group) * a.out_stride + (size_t)(h * a.group + row % a.group) * HD + d * 4;
            store_row4<BF16>(a.out, at, make_float4(z.x * inv, z.y * inv, z.z * inv, z.w * inv));
        }
        __syncthreads();
    }
}

}  // namespace dmc
