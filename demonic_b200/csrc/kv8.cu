// kv8.cu -- entry points of the 8-bit paged KV cache: append and attention (declared in include/dmc_cuda.h, kernels in
// kv8.cuh).  The page operations are in kv8_pages.cu.
#include <algorithm>

#include "kv8.cuh"
#include "kv8_host.h"

namespace dmc {

int check_kv8(const dmc_kv8_cache *c, const dmc_kv8_seqs *q, const char *who) {
    if (!c || !q) return fail(DMC_CUDA_ERR_BAD_ARG, "%s: null descriptor", who);
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "%s: page_tokens must be 16, 32 or 64 (got %d)", who, c->page_tokens);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %d)", who, c->head_dim);
    if (c->layers < 1 || c->kv_heads < 1 || c->pages < 1 || q->slots < 1 || q->table_stride < 1)
        return fail(DMC_CUDA_ERR_BAD_ARG, "%s: layers, kv_heads, pages, slots and table_stride must be positive", who);
    if (c->pages > kKv8MaxPages || q->slots > kKv8MaxSlots || c->kv_heads > 4096 ||
        q->table_stride > (1 << 30) / c->page_tokens)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "%s: more than %d pages, %d slots, 4096 kv heads or 2^30 tokens per slot", who,
                    kKv8MaxPages, kKv8MaxSlots);
    return DMC_CUDA_OK;
}

namespace {

Kv8Layer layer_of(const dmc_kv8_cache &c, int layer) {
    Kv8Layer l;
    const size_t heads = (size_t)layer * c.pages * c.kv_heads, at = heads * c.page_tokens * c.head_dim;
    l.k = (uint8_t *)c.k + at;
    l.v = (uint8_t *)c.v + at;
    l.ks = c.k_scale + heads;
    l.vs = c.v_scale + heads;
    l.pages = (int)c.pages;
    l.hk = c.kv_heads;
    l.page_shift = c.page_tokens == 16 ? 4 : c.page_tokens == 32 ? 5 : 6;
    return l;
}

Kv8Rows rows_of(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, const int *slot_ids, int batch, int tokens, const Kv8Rope &rope) {
    Kv8Rows r;
    r.cos = rope.cos;
    r.sin = rope.sin;
    r.table = q.table;
    r.lens = q.lens;
    r.slot_ids = slot_ids;
    r.flags = q.flags;
    r.table_stride = q.table_stride;
    r.slots = q.slots;
    r.batch = batch;
    r.tokens = tokens;
    r.cap = (int)(q.table_stride * c.page_tokens);
    r.report = 1;
    return r;
}

int check_rows(const dmc_kv8_cache *c, const dmc_kv8_seqs *q, int layer, int xdtype, const int *slot_ids, int batch, int tokens,
               const char *who) {
    if (layer < 0 || layer >= c->layers) return fail(DMC_CUDA_ERR_BAD_ARG, "%s: layer %d of %d", who, layer, c->layers);
    if (xdtype != DMC_X_BF16 && xdtype != DMC_X_F32) return fail(DMC_CUDA_ERR_BAD_ARG, "%s: unknown xdtype %d", who, xdtype);
    if (batch < 0 || tokens < 0) return fail(DMC_CUDA_ERR_BAD_ARG, "%s: negative batch or tokens", who);
    if (batch > kKv8MaxSlots || tokens > kKv8MaxTokens)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "%s: batch %d or tokens %d beyond %d and %d", who, batch, tokens, kKv8MaxSlots,
                    kKv8MaxTokens);
    if (!slot_ids && batch > q->slots)
        return fail(DMC_CUDA_ERR_BAD_ARG, "%s: batch %d of %d slots without slot_ids", who, batch, q->slots);
    return DMC_CUDA_OK;
}

template <int HD, bool BF16>
const void *append_fn(int nthr) {
    constexpr int E = BF16 ? 8 : 4;
    return nthr == 32 ? (const void *)kv8_append_kernel<HD, 32, 512 / 32 / E, BF16>
                      : (const void *)kv8_append_kernel<HD, 256, 64 * HD / 256 / E, BF16>;
}

// How an attention call is cut: query rows per tile, tiles, CTAs.
struct AttnPlan {
    int nt, row_tiles, ctas;
    size_t parts, bytes;  // partial rows; workspace: their values, their (maximum, sum), the segments' parts
    int rpc;              // rows per CTA of the join
};

template <int HD, int NT>
const void *attn_fn(bool bf16, bool cluster, size_t *smem) {
    *smem = bf16 ? sizeof(Kv8Smem<HD, NT, true>) : sizeof(Kv8Smem<HD, NT, false>);
    return bf16 ? (cluster ? (const void *)kv8_attn_kernel<HD, NT, true, true> : (const void *)kv8_attn_kernel<HD, NT, true, false>)
                : (cluster ? (const void *)kv8_attn_kernel<HD, NT, false, true> : (const void *)kv8_attn_kernel<HD, NT, false, false>);
}
const void *attn_fn(int hd, int nt, bool bf16, bool cluster, size_t *smem) {
#define PICK(HD, NT) \
    if (hd == HD && nt == NT) return attn_fn<HD, NT>(bf16, cluster, smem);
    PICK(64, 1) PICK(64, 2) PICK(64, 3) PICK(64, 4) PICK(128, 1) PICK(128, 2)
#undef PICK
    return nullptr;
}

AttnPlan plan_attention(int hd, int hk, int q_heads, int batch, int tokens, int sms) {
    AttnPlan p;
    const int rows = tokens * (q_heads / hk);
    // 8 rows per tile, or as many as the registers carry: a second tile reads the keys again (what that costs: kv8.cuh)
    p.nt = std::min((rows + 7) / 8, hd == 128 ? 2 : 4);
    p.row_tiles = (rows + 8 * p.nt - 1) / (8 * p.nt);
    const int per_sm = hd == 128 ? Kv8Ring<128>::ctas_per_sm(p.nt) : Kv8Ring<64>::ctas_per_sm(p.nt);
    p.ctas = std::min(sms * per_sm, kKv8MaxCtas);
    p.parts = (size_t)p.ctas * 2 * 8 * p.nt;
    p.bytes = p.parts * (hd * 4 + 8) + (size_t)batch * hk * p.row_tiles * 8;
    // enough joining CTAs to fill the device, and no more rows each than needed for that
    p.rpc = 1;
    while (p.rpc < std::min(kKv8JoinRows, 8 * p.nt) && (int64_t)batch * tokens * q_heads > (int64_t)sms * 4 * p.rpc) p.rpc *= 2;
    return p;
}

}  // namespace

int64_t kv8_attention_bytes(const dmc_kv8_cache &c, int q_heads, int batch, int tokens) {
    return (int64_t)plan_attention(c.head_dim, c.kv_heads, q_heads, batch, std::max(tokens, 1), ctx().sm_count).bytes;
}

int launch_kv8_append(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, int layer, const void *k, const void *v, int xdtype,
                      int64_t row_stride, const int *slot_ids, int batch, int tokens, cudaStream_t s, Kv8Rope rope) {
    Kv8Layer l = layer_of(c, layer);
    Kv8Rows r = rows_of(c, q, slot_ids, batch, tokens, rope);
    const bool bf16 = xdtype == DMC_X_BF16;
    const size_t esz = bf16 ? 2 : 4;
    // pages that `tokens` consecutive positions can touch
    int touch = (tokens + c.page_tokens - 2) / c.page_tokens + 1;
    int vec = ((uintptr_t)k | (uintptr_t)v | (uintptr_t)(row_stride * (int64_t)esz)) % 16 == 0;
    const int nthr = std::min(tokens, c.page_tokens) * c.head_dim <= 512 ? 32 : 256;
    const int64_t items = (int64_t)batch * touch * c.kv_heads * 2, ctas = (items * nthr + 255) / 256;
    if (ctas > INT32_MAX) return fail(DMC_CUDA_ERR_UNSUPPORTED, "kv8_append: batch * tokens * kv_heads is too large");
    long long stride = row_stride;
    void *params[] = {&l, &r, (void *)&k, (void *)&v, &stride, &touch, &vec};
    const void *fn = c.head_dim == 64 ? (bf16 ? append_fn<64, true>(nthr) : append_fn<64, false>(nthr))
                                      : (bf16 ? append_fn<128, true>(nthr) : append_fn<128, false>(nthr));
    return launch_on(fn, dim3((unsigned)ctas), dim3(256), 0, s, params);
}

int launch_kv8_attention(const dmc_kv8_cache &c, const dmc_kv8_seqs &q, int layer, const void *x, int64_t q_stride, void *out,
                         int64_t out_stride, int xdtype, int q_heads, const int *slot_ids, int batch, int tokens, float scale,
                         void *workspace, cudaStream_t s, Kv8Rope rope) {
    const bool bf16 = xdtype == DMC_X_BF16;
    const AttnPlan p = plan_attention(c.head_dim, c.kv_heads, q_heads, batch, tokens, ctx().sm_count);
    Kv8AttnArgs a;
    a.c = layer_of(c, layer);
    a.r = rows_of(c, q, slot_ids, batch, tokens, rope);
    a.q = x;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.part_o = (float *)workspace;
    a.part_ml = (float2 *)(a.part_o + p.parts * c.head_dim);
    a.segs = (int2 *)(a.part_ml + p.parts);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.group = q_heads / c.kv_heads;
    a.row_tiles = p.row_tiles;
    const int64_t segs = (int64_t)batch * c.kv_heads * p.row_tiles, units = (a.r.cap + kKv8Unit - 1) / kKv8Unit;
    // A cluster per segment, of as many CTAs as there can be units or as the device holds, while no CTA can get more than 16
    // units: the lengths are not known here, and longer ones are better shared out evenly.
    unsigned cluster = 1;
    while (cluster < kKv8MaxCluster && cluster < units && segs * cluster * 2 <= p.ctas) cluster *= 2;
    const bool few = segs <= p.ctas && units <= 16 * (int64_t)cluster;
    size_t smem = 0;
    const void *fn = attn_fn(c.head_dim, p.nt, bf16, few, &smem);
    DMC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    void *params[] = {&a};
    if (few) {
        a.ctas = (int)(segs * cluster);
        return launch_on(fn, dim3((unsigned)a.ctas), dim3(128), smem, s, params, cluster);
    }
    a.ctas = (int)std::min<int64_t>(p.ctas, segs * units);  // no more CTAs than there can be units
    int rc = launch_on(fn, dim3((unsigned)a.ctas), dim3(128), smem, s, params);
    if (rc) return rc;
    int nr = 8 * p.nt, rpc = p.rpc;
    a.r.report = 0;
    void *params2[] = {&a, &nr, &rpc};
    const void *join = c.head_dim == 64 ? (bf16 ? (const void *)kv8_attn_join_kernel<64, true> : (const void *)kv8_attn_join_kernel<64, false>)
                                        : (bf16 ? (const void *)kv8_attn_join_kernel<128, true> : (const void *)kv8_attn_join_kernel<128, false>);
    return launch_on(join, dim3((unsigned)(segs * ((nr + rpc - 1) / rpc))), dim3(256), 0, s, params2);
}

}  // namespace dmc

using namespace dmc;

extern "C" int dmc_kv8_append(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, int layer, const void *k, const void *v,
                              int xdtype, int64_t row_stride, const int *slot_ids, int batch, int tokens, void *stream) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    OnDevice on;
    int rc;
    if ((rc = check_kv8(cache, seqs, "kv8_append")) ||
        (rc = check_rows(cache, seqs, layer, xdtype, slot_ids, batch, tokens, "kv8_append")))
        return rc;
    if (batch == 0 || tokens == 0) return DMC_CUDA_OK;
    const size_t esz = xdtype == DMC_X_BF16 ? 2 : 4;
    if (row_stride < (int64_t)cache->kv_heads * cache->head_dim)
        return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_append: row_stride %lld below kv_heads * head_dim", (long long)row_stride);
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), {slot_ids, 4, "slot_ids", true}, {k, esz, "k"}, {v, esz, "v"}}))) return rc;
    return launch_kv8_append(*cache, *seqs, layer, k, v, xdtype, row_stride, slot_ids, batch, tokens, (cudaStream_t)stream);
}

extern "C" int64_t dmc_kv8_attention_workspace(const dmc_kv8_cache *cache, int q_heads, int batch, int tokens) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return -1;
    if (!cache || cache->kv_heads < 1 || q_heads < 1 || q_heads % cache->kv_heads || batch < 0 || tokens < 0 ||
        batch > kKv8MaxSlots || tokens > kKv8MaxTokens || (int64_t)batch * tokens > INT32_MAX / q_heads ||
        (cache->head_dim != 64 && cache->head_dim != 128)) {
        fail(DMC_CUDA_ERR_BAD_ARG, "kv8_attention_workspace: bad head counts, head_dim or sizes");
        return -1;
    }
    OnDevice on;
    if (ensure_init()) return -1;
    return kv8_attention_bytes(*cache, q_heads, batch, tokens);
}

extern "C" int dmc_kv8_attention(const dmc_kv8_cache *cache, const dmc_kv8_seqs *seqs, int layer, const void *q, int64_t q_stride,
                                 void *out, int64_t out_stride, int xdtype, int q_heads, const int *slot_ids, int batch,
                                 int tokens, float scale, void *workspace, int64_t workspace_bytes, void *stream) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    OnDevice on;
    int rc;
    if ((rc = check_kv8(cache, seqs, "kv8_attention")) ||
        (rc = check_rows(cache, seqs, layer, xdtype, slot_ids, batch, tokens, "kv8_attention")))
        return rc;
    if (q_heads < 1 || q_heads % cache->kv_heads)
        return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_attention: q_heads %d is not a multiple of kv_heads %d", q_heads, cache->kv_heads);
    if (batch == 0 || tokens == 0) return DMC_CUDA_OK;
    const int64_t width = (int64_t)q_heads * cache->head_dim;
    if (q_stride < width || out_stride < width)
        return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_attention: row strides %lld, %lld below q_heads * head_dim", (long long)q_stride,
                    (long long)out_stride);
    if (q_stride % 4 || out_stride % 4)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "kv8_attention: row strides have to be multiples of 4 elements");
    if ((int64_t)batch * tokens > INT32_MAX / q_heads)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "kv8_attention: batch * tokens * q_heads is too large");
    const size_t esz = xdtype == DMC_X_BF16 ? 2 : 4;
    if ((rc = enter_device({KV8_POINTERS(cache, seqs), {slot_ids, 4, "slot_ids", true}, {q, 4 * esz, "q"}, {out, 4 * esz, "out"},
                            {workspace, 16, "workspace"}})))
        return rc;
    const AttnPlan p = plan_attention(cache->head_dim, cache->kv_heads, q_heads, batch, tokens, ctx().sm_count);
    if (workspace_bytes < (int64_t)p.bytes)
        return fail(DMC_CUDA_ERR_BAD_ARG, "kv8_attention: workspace of %lld bytes, %zu are needed", (long long)workspace_bytes, p.bytes);
    return launch_kv8_attention(*cache, *seqs, layer, q, q_stride, out, out_stride, xdtype, q_heads, slot_ids, batch, tokens, scale,
                                workspace, (cudaStream_t)stream);
}
