// decode.cu -- one decode step of a decoder-only transformer, fully on the device: every
// projection goes through the GEMV path, the companions of decode_ops.cuh sit between them, and
// the whole step (43 launches in the fused arrangement) is captured once into a CUDA graph and replayed per token, so the
// per-call host<->device traffic the reference ABI forces (compiler/src/gpu.rs:528-531, 649-651)
// disappears: a token id goes in, a token id comes out.
#include <cstring>
#include <new>
#include <utility>
#include <vector>

#include "decode_ops.cuh"
#include "kv8_host.h"

namespace dmc {
namespace {

struct Layer {
    uint16_t *wqkv = nullptr, *wo = nullptr, *wgu = nullptr, *wd = nullptr;  // [3D,D] [D,D] [2F,D] [D,F] bf16, k contiguous
    float *g1 = nullptr, *g2 = nullptr;                                      // RMSNorm gains [D]
    float *kc = nullptr, *vc = nullptr;                                      // KV cache [H][cap][hd] f32
};

// What a step of the 8-bit cache takes from the host in one copy, and gives back.
struct StepIn {
    int token, slot, len;
    int top_k;
    float temperature, top_p, min_p, u;
};
struct StepOut {
    int token;
    float prob;
    int flags;
};

// The 8-bit paged cache of a decoder that holds several sequences (dmc_decoder_create_kv8).
struct Kv8State {
    dmc_kv8_cache cache = {};
    dmc_kv8_seqs seqs = {};
    void *workspace = nullptr;
    StepIn *in = nullptr, *h_in = nullptr;    // device; pinned
    StepOut *out = nullptr, *h_out = nullptr;
    int *pair = nullptr;                      // device: source and destination of a fork, or the slot of a release
    std::vector<int> lens;                    // the device's lens
    std::vector<char> shared;                 // a sequence whose last page another may hold
};

struct Decoder {
    dmc_decoder_config cfg;
    Kv8State *kv8 = nullptr;
    std::vector<Layer> layers;
    uint16_t *embed = nullptr, *lm_head = nullptr;  // [V,D] bf16
    float *gf = nullptr, *rope_cos = nullptr, *rope_sin = nullptr;
    float *h2 = nullptr;        // second residual-stream buffer (the fused RMSNorm ping-pongs between h and h2)
    unsigned *attn_cnt = nullptr;
    unsigned long long *am_key = nullptr;  // arg-max key the lm-head GEMV leaves (fused arrangement)
    float *am_val = nullptr;    // argmax per-CTA candidates (unfused arrangement)
    int *am_idx = nullptr;
    unsigned *am_cnt = nullptr;
    int fused = 1;              // 1: RMSNorm / SwiGLU fused into the GEMVs' staging, RoPE + append + combine into attention
    float *h = nullptr, *xn = nullptr, *qkv = nullptr, *ao = nullptr, *d1 = nullptr, *gu = nullptr, *act = nullptr,
          *d2 = nullptr, *logits = nullptr, *part = nullptr;
    int *d_token = nullptr, *d_pos = nullptr, *d_next = nullptr;
    int splits = 32;            // key ranges per head in the attention kernels
    cudaGraph_t graph = nullptr;
    cudaGraphExec_t exec = nullptr;
    int64_t launches_per_step = 0;
};

// Zeroed on the context's stream, which the first copies into it run on too: it does not wait for the default stream.
template <typename T>
int dalloc(T **p, size_t count) {
    DMC_CUDA_TRY(dmc_malloc((void **)p, count * sizeof(T)));
    DMC_CUDA_TRY(cudaMemsetAsync(*p, 0, count * sizeof(T), ctx().stream));
    return DMC_CUDA_OK;
}

template <typename... Args>
int launch_small(void (*fn)(Args...), dim3 grid, dim3 block, cudaStream_t s, Args... args) {
    void *params[] = {(void *)&args...};
    return launch_ex((const void *)fn, grid, block, 0, s, params);
}

// y = W . prologue(x) with the prologue fused into the GEMV's x staging (see GemvArgs::pro).
int gemv_pro(const void *W, const float *x, float *y, int64_t k, int64_t n, int pro, const float *add, const float *g,
             float *hout, float eps, cudaStream_t s) {
    Context &c = ctx();
    c.pro = pro;
    c.pro_add = add;
    c.pro_g = g;
    c.pro_hout = hout;
    c.pro_eps = eps;
    int rc = launch_gemv(W, x, y, 1, k, n, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s);
    c.pro = 0;
    c.pro_add = c.pro_g = nullptr;
    c.pro_hout = nullptr;
    return rc;
}

// One step over the 8-bit cache, 6 launches per layer -- qkv (RMSNorm in its staging) -> append (RoPE on K) ->
// attention (RoPE on q) -> Wo -> gate/up -> down; 7 where max_len is so large that the attention's parts are joined by a launch of
// their own -- then lm-head and the draw of the token.  The slot's length already counts the token.  8 layers x 2048, 513 tokens held:
// 51 launches, 351 us, against 42 and 283 over the f32 cache, whose attention appends too and whose lm-head takes the arg-max.
int enqueue_step_kv8(Decoder &d, cudaStream_t s) {
    const dmc_decoder_config &c = d.cfg;
    Kv8State &k = *d.kv8;
    const int D = c.d_model, H = c.heads, F = c.ffn, V = c.vocab;
    int rc;
    float *hin = d.h, *hout = d.h2;
    if ((rc = launch_small(embed_kernel, dim3(8), dim3(256), s, (const uint16_t *)d.embed, V, D, (const int *)&k.in->token, hin,
                           (unsigned long long *)nullptr)))
        return rc;
    const float *carry = nullptr;
    const Kv8Rope rope{d.rope_cos, d.rope_sin};
    for (int l = 0; l < c.layers; ++l) {
        Layer &L = d.layers[l];
        if ((rc = gemv_pro(L.wqkv, hin, d.qkv, D, 3 * D, 1, carry, L.g1, hout, c.eps, s))) return rc;
        std::swap(hin, hout);
        if ((rc = launch_kv8_append(k.cache, k.seqs, l, d.qkv + D, d.qkv + 2 * D, DMC_X_F32, D, &k.in->slot, 1, 1, s, rope))) return rc;
        if ((rc = launch_kv8_attention(k.cache, k.seqs, l, d.qkv, D, d.ao, D, DMC_X_F32, H, &k.in->slot, 1, 1,
                                       1.0f / sqrtf((float)c.head_dim), k.workspace, s, rope)))
            return rc;
        if ((rc = launch_gemv(L.wo, d.ao, d.d1, 1, D, D, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
        if ((rc = gemv_pro(L.wgu, hin, d.gu, D, 2 * F, 1, d.d1, L.g2, hout, c.eps, s))) return rc;
        std::swap(hin, hout);
        if ((rc = gemv_pro(L.wd, d.gu, d.d2, F, D, 2, nullptr, nullptr, nullptr, 0.0f, s))) return rc;
        carry = d.d2;
    }
    if ((rc = gemv_pro(d.lm_head, hin, d.logits, D, V, 1, carry, d.gf, nullptr, c.eps, s))) return rc;
    return launch_sample(d.logits, DMC_X_F32, 1, V, V, &k.in->temperature, &k.in->top_k, &k.in->top_p, &k.in->min_p, &k.in->u,
                         &k.out->token, &k.out->prob, s);
}

// All launches of one step, in order, on `s`: 5 per layer (43 in all for 8 layers).
int enqueue_step_fused(Decoder &d, cudaStream_t s) {
    const dmc_decoder_config &c = d.cfg;
    const int D = c.d_model, H = c.heads, F = c.ffn, V = c.vocab, cap = c.max_len;
    int rc;
    float *hin = d.h, *hout = d.h2;
    if ((rc = launch_small(embed_kernel, dim3(8), dim3(256), s, (const uint16_t *)d.embed, V, D, (const int *)d.d_token, hin,
                           d.am_key)))
        return rc;
    const float *carry = nullptr;
    const int chunk = (cap + d.splits - 1) / d.splits;
    for (int l = 0; l < c.layers; ++l) {
        Layer &L = d.layers[l];
        // qkv = Wqkv . rms_norm(h + carry);  h' = h + carry
        if ((rc = gemv_pro(L.wqkv, hin, d.qkv, D, 3 * D, 1, carry, L.g1, hout, c.eps, s))) return rc;
        std::swap(hin, hout);
        if ((rc = launch_small(attn_fused_kernel, dim3(H, d.splits), dim3(128), s, (const float *)d.qkv,
                               (const float *)d.rope_cos, (const float *)d.rope_sin, L.kc, L.vc, d.part, d.ao, d.attn_cnt, H,
                               cap, (const int *)d.d_pos, chunk)))
            return rc;
        if ((rc = launch_gemv(L.wo, d.ao, d.d1, 1, D, D, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
        // gu = Wgu . rms_norm(h + d1);  h' = h + d1
        if ((rc = gemv_pro(L.wgu, hin, d.gu, D, 2 * F, 1, d.d1, L.g2, hout, c.eps, s))) return rc;
        std::swap(hin, hout);
        // d2 = Wd . (silu(gate) * up)
        if ((rc = gemv_pro(L.wd, d.gu, d.d2, F, D, 2, nullptr, nullptr, nullptr, 0.0f, s))) return rc;
        carry = d.d2;
    }
    // logits = lm_head . rms_norm(h + carry), and their arg-max in the same kernel
    ctx().amax = d.am_key;
    rc = gemv_pro(d.lm_head, hin, d.logits, D, V, 1, carry, d.gf, nullptr, c.eps, s);
    ctx().amax = nullptr;
    return rc;
}

// The unfused sequence (9 launches per layer), kept as the reference arrangement of the same math.
int enqueue_step_plain(Decoder &d, cudaStream_t s) {
    const dmc_decoder_config &c = d.cfg;
    const int D = c.d_model, H = c.heads, hd = c.head_dim, F = c.ffn, V = c.vocab, cap = c.max_len;
    int rc;
    if ((rc = launch_small(embed_kernel, dim3(8), dim3(256), s, (const uint16_t *)d.embed, V, D, (const int *)d.d_token, d.h,
                           (unsigned long long *)nullptr)))
        return rc;
    const float *carry = nullptr;  // residual branch output waiting to be added to h
    const int chunk = (cap + d.splits - 1) / d.splits;
    for (int l = 0; l < c.layers; ++l) {
        Layer &L = d.layers[l];
        if ((rc = launch_small(rmsnorm_kernel, dim3(1), dim3(1024), s, d.h, carry, (const float *)L.g1, d.xn, D, c.eps))) return rc;
        if ((rc = launch_gemv(L.wqkv, d.xn, d.qkv, 1, D, 3 * D, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
        if ((rc = launch_small(rope_append_kernel, dim3(4), dim3(256), s, d.qkv, (const float *)d.rope_cos,
                               (const float *)d.rope_sin, L.kc, L.vc, H, hd, cap, (const int *)d.d_pos)))
            return rc;
        if ((rc = launch_small(attn_partial_kernel, dim3(H, d.splits), dim3(128), s, (const float *)d.qkv,
                               (const float *)L.kc, (const float *)L.vc, d.part, H, cap, (const int *)d.d_pos, chunk)))
            return rc;
        if ((rc = launch_small(attn_combine_kernel, dim3(H), dim3(128), s, (const float *)d.part, d.ao, d.splits))) return rc;
        if ((rc = launch_gemv(L.wo, d.ao, d.d1, 1, D, D, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
        if ((rc = launch_small(rmsnorm_kernel, dim3(1), dim3(1024), s, d.h, (const float *)d.d1, (const float *)L.g2, d.xn, D, c.eps)))
            return rc;
        if ((rc = launch_gemv(L.wgu, d.xn, d.gu, 1, D, 2 * F, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
        if ((rc = launch_small(swiglu_kernel, dim3(8), dim3(256), s, (const float *)d.gu, d.act, F))) return rc;
        if ((rc = launch_gemv(L.wd, d.act, d.d2, 1, F, D, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
        carry = d.d2;
    }
    if ((rc = launch_small(rmsnorm_kernel, dim3(1), dim3(1024), s, d.h, carry, (const float *)d.gf, d.xn, D, c.eps))) return rc;
    if ((rc = launch_gemv(d.lm_head, d.xn, d.logits, 1, D, V, 1, 0, 0, DMC_LAYOUT_NK, DMC_W_BF16, -1, s))) return rc;
    return launch_small(argmax_kernel, dim3(64), dim3(256), s, (const float *)d.logits, V, d.d_next, d.am_val, d.am_idx, d.am_cnt);
}

int enqueue_step(Decoder &d, cudaStream_t s) { return d.kv8 ? enqueue_step_kv8(d, s) : d.fused ? enqueue_step_fused(d, s) : enqueue_step_plain(d, s); }

int ensure_graph(Decoder &d) {
    if (d.exec) return DMC_CUDA_OK;
    Context &c = ctx();
    int rc = enqueue_step(d, c.stream);  // eager once: kernel attributes and scratch are set up outside capture
    if (rc) return rc;
    DMC_CUDA_TRY(cudaStreamSynchronize(c.stream));
    const int64_t before = c.launches;
    DMC_CUDA_TRY(cudaStreamBeginCapture(c.stream, cudaStreamCaptureModeThreadLocal));
    rc = enqueue_step(d, c.stream);
    cudaError_t ce = cudaStreamEndCapture(c.stream, &d.graph);
    if (rc) return rc;
    DMC_CUDA_TRY(ce);
    d.launches_per_step = c.launches - before;
    DMC_CUDA_TRY(cudaGraphInstantiate(&d.exec, d.graph, 0));
    return DMC_CUDA_OK;
}

void *weight_slot(Decoder &d, int which, int layer, size_t *bytes) {
    const dmc_decoder_config &c = d.cfg;
    const size_t D = c.d_model, F = c.ffn, V = c.vocab;
    if (which == DMC_DEC_EMBED) { *bytes = V * D * 2; return d.embed; }
    if (which == DMC_DEC_LM_HEAD) { *bytes = V * D * 2; return d.lm_head; }
    if (which == DMC_DEC_GAIN_FINAL) { *bytes = D * 4; return d.gf; }
    if (layer < 0 || layer >= c.layers) return nullptr;
    Layer &L = d.layers[layer];
    switch (which) {
        case DMC_DEC_WQKV: *bytes = 3 * D * D * 2; return L.wqkv;
        case DMC_DEC_WO: *bytes = D * D * 2; return L.wo;
        case DMC_DEC_WGU: *bytes = 2 * F * D * 2; return L.wgu;
        case DMC_DEC_WD: *bytes = D * F * 2; return L.wd;
        case DMC_DEC_GAIN1: *bytes = D * 4; return L.g1;
        case DMC_DEC_GAIN2: *bytes = D * 4; return L.g2;
        default: return nullptr;
    }
}

bool decoder_config_ok(const dmc_decoder_config *cfg) {
    return cfg && cfg->layers >= 1 && cfg->d_model >= 8 && cfg->heads >= 1 && cfg->head_dim == 128 &&
           cfg->heads * cfg->head_dim == cfg->d_model && cfg->ffn >= 8 && cfg->vocab >= 1 && cfg->max_len >= 1 &&
           cfg->d_model % 8 == 0 && cfg->ffn % 8 == 0;
}

void free_kv8(Kv8State *k) {
    if (!k) return;
    void *dev[] = {k->cache.k, k->cache.v, k->cache.k_scale, k->cache.v_scale, k->seqs.table, k->seqs.lens, k->seqs.refs,
                   k->seqs.free_list, k->seqs.free_count, k->seqs.flags, k->seqs.scratch, k->workspace, k->in, k->out, k->pair};
    for (void *p : dev)
        if (p) cudaFree(p);
    if (k->h_in) cudaFreeHost(k->h_in);
    if (k->h_out) cudaFreeHost(k->h_out);
    delete k;
}

// Everything that a decoder owns, its 8-bit cache included; one that was only partly allocated too.
void free_decoder(Decoder *d) {
    if (!d) return;
    if (d->exec) cudaGraphExecDestroy(d->exec);
    if (d->graph) cudaGraphDestroy(d->graph);
    void *singles[] = {d->embed, d->lm_head, d->gf, d->rope_cos, d->rope_sin, d->h, d->xn, d->qkv, d->ao, d->d1, d->gu,
                       d->act, d->d2, d->logits, d->part, d->d_token, d->d_pos, d->d_next, d->h2, d->attn_cnt, d->am_val, d->am_idx, d->am_cnt,
                       d->am_key};
    for (void *p : singles)
        if (p) cudaFree(p);
    for (Layer &L : d->layers) {
        void *ps[] = {L.wqkv, L.wo, L.wgu, L.wd, L.g1, L.g2, L.kc, L.vc};
        for (void *p : ps)
            if (p) cudaFree(p);
    }
    free_kv8(d->kv8);
    delete d;
}

int create_kv8(Kv8State &k, const dmc_decoder_config &cfg, int sequences, int64_t pages, int page_tokens) {
    dmc_kv8_cache &c = k.cache;
    dmc_kv8_seqs &q = k.seqs;
    c.pages = pages;
    c.layers = cfg.layers;
    c.kv_heads = cfg.heads;
    c.page_tokens = page_tokens;
    c.head_dim = cfg.head_dim;
    q.slots = sequences;
    q.table_stride = (cfg.max_len + page_tokens - 1) / page_tokens;
    const size_t heads = (size_t)cfg.layers * pages * cfg.heads, codes = heads * page_tokens * cfg.head_dim;
    int rc = dalloc((uint8_t **)&c.k, codes) || dalloc((uint8_t **)&c.v, codes) || dalloc(&c.k_scale, heads) || dalloc(&c.v_scale, heads) ||
             dalloc(&q.table, (size_t)sequences * q.table_stride) || dalloc(&q.lens, sequences) || dalloc(&q.refs, pages) ||
             dalloc(&q.free_list, pages) || dalloc(&q.free_count, 1) || dalloc(&q.flags, 1) ||
             dalloc((uint8_t **)&q.scratch, dmc_kv8_scratch_bytes(pages, sequences)) ||
             dalloc((uint8_t **)&k.workspace, kv8_attention_bytes(c, cfg.heads, 1, 1)) || dalloc(&k.in, 1) || dalloc(&k.out, 1) ||
             dalloc(&k.pair, 2);
    if (rc) return dmc::status();
    DMC_CUDA_TRY(dmc_malloc_host((void **)&k.h_in, sizeof(StepIn)));
    DMC_CUDA_TRY(dmc_malloc_host((void **)&k.h_out, sizeof(StepOut)));
    std::vector<int> free_list(pages);
    for (int64_t i = 0; i < pages; ++i) free_list[i] = (int)(pages - 1 - i);
    const int count = (int)pages;
    DMC_CUDA_TRY(cudaMemcpyAsync(q.free_list, free_list.data(), pages * 4, cudaMemcpyHostToDevice, ctx().stream));
    DMC_CUDA_TRY(cudaMemcpyAsync(q.free_count, &count, 4, cudaMemcpyHostToDevice, ctx().stream));
    DMC_CUDA_TRY(cudaStreamSynchronize(ctx().stream));
    k.lens.assign(sequences, 0);
    k.shared.assign(sequences, 0);
    return DMC_CUDA_OK;
}

// The decoder of a call on the 8-bit cache and its state, or null and a status.
Kv8State *kv8_of(void *dec, const char *who) {
    Decoder *d = static_cast<Decoder *>(dec);
    if (d && d->kv8) return d->kv8;
    fail(DMC_CUDA_ERR_BAD_ARG, "%s: not a decoder with an 8-bit cache", who);
    return nullptr;
}
bool kv8_slot_ok(const Kv8State &k, int seq) { return seq >= 0 && seq < k.seqs.slots; }

}  // namespace
}  // namespace dmc

using namespace dmc;

static int create_decoder(const dmc_decoder_config *cfg, bool kv8, Decoder **out);

extern "C" int dmc_decoder_create(const dmc_decoder_config *cfg, void **out) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    if (!decoder_config_ok(cfg) || !out)
        return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_create: unsupported configuration (head_dim must be 128, "
                                          "heads*head_dim == d_model, d_model and ffn multiples of 8)");
    int rc = ensure_init();
    if (rc) return rc;
    Decoder *d = nullptr;
    if ((rc = create_decoder(cfg, false, &d))) return rc;
    *out = d;
    return DMC_CUDA_OK;
}

// What every decoder has, and the f32 cache of one without an 8-bit cache.  The caller frees what a throw leaves in *d.
static int alloc_decoder(const dmc_decoder_config *cfg, bool kv8, Decoder *d) {
    int rc;
    d->cfg = *cfg;
    const size_t D = cfg->d_model, F = cfg->ffn, V = cfg->vocab, H = cfg->heads, hd = cfg->head_dim, cap = cfg->max_len;
    d->layers.resize(cfg->layers);
    rc = dalloc(&d->embed, V * D) || dalloc(&d->lm_head, V * D) || dalloc(&d->gf, D) || dalloc(&d->rope_cos, cap * hd / 2) ||
         dalloc(&d->rope_sin, cap * hd / 2) || dalloc(&d->h, D) || dalloc(&d->xn, D) || dalloc(&d->qkv, 3 * D) ||
         dalloc(&d->ao, D) || dalloc(&d->d1, D) || dalloc(&d->gu, 2 * F) || dalloc(&d->act, F) || dalloc(&d->d2, D) ||
         dalloc(&d->logits, V) || dalloc(&d->part, H * (size_t)d->splits * (hd + 2)) || dalloc(&d->d_token, 1) ||
         dalloc(&d->d_pos, 1) || dalloc(&d->d_next, 1) || dalloc(&d->h2, D) || dalloc(&d->attn_cnt, H) ||
         dalloc(&d->am_val, 64) || dalloc(&d->am_idx, 64) || dalloc(&d->am_cnt, 1) || dalloc(&d->am_key, 1);
    d->fused = tuning().decode_fused;
    for (Layer &L : d->layers)
        rc = rc || dalloc(&L.wqkv, 3 * D * D) || dalloc(&L.wo, D * D) || dalloc(&L.wgu, 2 * F * D) || dalloc(&L.wd, D * F) ||
             dalloc(&L.g1, D) || dalloc(&L.g2, D) || (!kv8 && (dalloc(&L.kc, H * cap * hd) || dalloc(&L.vc, H * cap * hd)));
    return rc ? dmc::status() : DMC_CUDA_OK;
}

static int create_decoder(const dmc_decoder_config *cfg, bool kv8, Decoder **out) {
    Decoder *d = nullptr;
    int rc;
    try {
        d = new Decoder();
        rc = alloc_decoder(cfg, kv8, d);
    } catch (const std::bad_alloc &) {  // not across the C boundary
        rc = fail(DMC_CUDA_ERR_OOM, "decoder_create: host memory");
    }
    if (rc) free_decoder(d);
    else *out = d;
    return rc;
}

extern "C" int dmc_decoder_create_kv8(const dmc_decoder_config *cfg, int sequences, int64_t pages, int page_tokens, void **out) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    if (!decoder_config_ok(cfg) || !out || sequences < 1 || sequences > kKv8MaxSlots || pages < 1 || pages > kKv8MaxPages ||
        (page_tokens != 16 && page_tokens != 32 && page_tokens != 64))
        return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_create_kv8: unsupported configuration (head_dim must be 128, heads*head_dim == d_model, "
                                          "d_model and ffn multiples of 8, page_tokens 16, 32 or 64, sequences and pages positive)");
    if (cfg->vocab > kSampleMaxVocab || cfg->max_len > 1 << 30 || cfg->heads > 4096)
        return fail(DMC_CUDA_ERR_UNSUPPORTED, "decoder_create_kv8: more than %d words, 2^30 tokens or 4096 heads", kSampleMaxVocab);
    int rc = ensure_init();
    if (rc) return rc;
    Kv8State *k = nullptr;
    Decoder *d = nullptr;
    try {
        k = new Kv8State();
        rc = create_kv8(*k, *cfg, sequences, pages, page_tokens);
        if (!rc) rc = create_decoder(cfg, true, &d);
    } catch (const std::bad_alloc &) {  // not across the C boundary
        rc = fail(DMC_CUDA_ERR_OOM, "decoder_create_kv8: host memory");
    }
    if (rc) {
        free_kv8(k);
        return rc;
    }
    d->kv8 = k;
    *out = d;
    return DMC_CUDA_OK;
}

extern "C" int dmc_decoder_step_kv8(void *dec, int seq, int token, const dmc_sampling *how, int *next_token, float *prob,
                                    float *logits_out) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    Kv8State *k = kv8_of(dec, "decoder_step_kv8");
    if (!k) return dmc::status();
    Decoder *d = static_cast<Decoder *>(dec);
    if (!kv8_slot_ok(*k, seq)) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_step_kv8: sequence %d of %d", seq, k->seqs.slots);
    const int len = k->lens[seq] + 1;
    if (len > d->cfg.max_len) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_step_kv8: sequence %d is full (%d tokens)", seq, len - 1);
    int rc = ensure_init();
    if (rc) return rc;
    cudaStream_t s = ctx().stream;
    const dmc_sampling greedy = {0.0f, 0, 1.0f, 0.0f, 0.0f}, &h = how ? *how : greedy;
    *k->h_in = StepIn{token, seq, len, h.top_k, h.temperature, h.top_p, h.min_p, h.u};
    DMC_CUDA_TRY(cudaMemcpyAsync(k->in, k->h_in, sizeof(StepIn), cudaMemcpyHostToDevice, s));
    if ((len - 1) % k->cache.page_tokens == 0 || k->shared[seq]) {
        // the token may need a page: known only on the device, and nothing may be written without one
        if ((rc = launch_kv8_reserve(k->cache, k->seqs, &k->in->slot, nullptr, 1, 1, s))) return rc;
        DMC_CUDA_TRY(cudaMemcpyAsync(&k->h_out->flags, k->seqs.flags, 4, cudaMemcpyDeviceToHost, s));
        DMC_CUDA_TRY(cudaStreamSynchronize(s));
        stream_drained();
        if (k->h_out->flags) {
            DMC_CUDA_TRY(cudaMemsetAsync(k->seqs.flags, 0, 4, s));
            DMC_CUDA_TRY(cudaStreamSynchronize(s));
            return fail(DMC_CUDA_ERR_OOM, "decoder_step_kv8: no page is left for sequence %d (flags %d)", seq, k->h_out->flags);
        }
        k->shared[seq] = 0;
    } else {
        DMC_CUDA_TRY(cudaMemcpyAsync(k->seqs.lens + seq, &k->h_in->len, 4, cudaMemcpyHostToDevice, s));
    }
    k->lens[seq] = len;
    // (the first call also runs the step once eagerly before capturing it: the same token at the same place)
    if ((rc = ensure_graph(*d))) return rc;
    DMC_CUDA_TRY(cudaGraphLaunch(d->exec, s));
    ctx().launches += d->launches_per_step;
    DMC_CUDA_TRY(cudaMemcpyAsync(k->h_out, k->out, 8, cudaMemcpyDeviceToHost, s));
    if (logits_out) DMC_CUDA_TRY(cudaMemcpyAsync(logits_out, d->logits, (size_t)d->cfg.vocab * 4, cudaMemcpyDeviceToHost, s));
    DMC_CUDA_TRY(cudaStreamSynchronize(s));
    stream_drained();
    if (next_token) *next_token = k->h_out->token;
    if (prob) *prob = k->h_out->prob;
    return dmc::status();
}

extern "C" int dmc_decoder_fork(void *dec, int src, int dst) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    Kv8State *k = kv8_of(dec, "decoder_fork");
    if (!k) return dmc::status();
    if (!kv8_slot_ok(*k, src) || !kv8_slot_ok(*k, dst) || src == dst || k->lens[dst] != 0)
        return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_fork: from sequence %d into %d (of %d; the second has to be empty)", src, dst, k->seqs.slots);
    int rc = ensure_init();
    if (rc) return rc;
    const int pair[2] = {src, dst};
    DMC_CUDA_TRY(cudaMemcpyAsync(k->pair, pair, 8, cudaMemcpyHostToDevice, ctx().stream));
    if ((rc = launch_kv8_fork(k->cache, k->seqs, k->pair, k->pair + 1, 1, ctx().stream))) return rc;
    DMC_CUDA_TRY(cudaStreamSynchronize(ctx().stream));  // pair lives on this stack frame
    stream_drained();
    k->lens[dst] = k->lens[src];
    if (k->lens[src]) k->shared[src] = k->shared[dst] = 1;  // (a full last page too: the benchmark writes into it again)
    return DMC_CUDA_OK;
}

extern "C" int dmc_decoder_release(void *dec, int seq) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    Kv8State *k = kv8_of(dec, "decoder_release");
    if (!k) return dmc::status();
    if (!kv8_slot_ok(*k, seq)) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_release: sequence %d of %d", seq, k->seqs.slots);
    int rc = ensure_init();
    if (rc) return rc;
    DMC_CUDA_TRY(cudaMemcpyAsync(k->pair, &seq, 4, cudaMemcpyHostToDevice, ctx().stream));
    if ((rc = launch_kv8_release(k->cache, k->seqs, k->pair, 1, ctx().stream))) return rc;
    DMC_CUDA_TRY(cudaStreamSynchronize(ctx().stream));  // seq lives on this stack frame
    stream_drained();
    k->lens[seq] = 0;
    k->shared[seq] = 0;
    return DMC_CUDA_OK;
}

extern "C" int dmc_decoder_compact(void *dec) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    Kv8State *k = kv8_of(dec, "decoder_compact");
    if (!k) return dmc::status();
    int rc = ensure_init();
    if (rc || (rc = launch_kv8_compact(k->cache, k->seqs, nullptr, ctx().stream))) return rc;
    DMC_CUDA_TRY(cudaStreamSynchronize(ctx().stream));
    stream_drained();
    return DMC_CUDA_OK;
}

extern "C" int dmc_decoder_length(void *dec, int seq) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    Decoder *d = static_cast<Decoder *>(dec);
    return d && d->kv8 && kv8_slot_ok(*d->kv8, seq) ? d->kv8->lens[seq] : -1;
}

extern "C" int64_t dmc_decoder_free_pages(void *dec) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return -1;
    Kv8State *k = kv8_of(dec, "decoder_free_pages");
    int n = -1;
    auto body = [&]() -> int {
        DMC_CUDA_TRY(cudaMemcpyAsync(&n, k->seqs.free_count, 4, cudaMemcpyDeviceToHost, ctx().stream));
        DMC_CUDA_TRY(cudaStreamSynchronize(ctx().stream));
        stream_drained();
        return DMC_CUDA_OK;
    };
    return k && body() == DMC_CUDA_OK ? n : -1;
}

extern "C" int dmc_decoder_load(void *dec, int which, int layer, const void *host, int64_t bytes) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    Decoder *d = static_cast<Decoder *>(dec);
    size_t want = 0;
    void *dst = nullptr;
    if (which == DMC_DEC_ROPE_COS || which == DMC_DEC_ROPE_SIN) {
        want = (size_t)d->cfg.max_len * d->cfg.head_dim / 2 * 4;
        dst = which == DMC_DEC_ROPE_COS ? d->rope_cos : d->rope_sin;
    } else if (which == DMC_DEC_KCACHE || which == DMC_DEC_VCACHE) {
        if (layer < 0 || layer >= d->cfg.layers) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_load: bad layer %d", layer);
        if (d->kv8) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_load: an 8-bit cache is filled by steps");
        want = (size_t)d->cfg.heads * d->cfg.max_len * d->cfg.head_dim * 4;
        dst = which == DMC_DEC_KCACHE ? d->layers[layer].kc : d->layers[layer].vc;
    } else {
        dst = weight_slot(*d, which, layer, &want);
    }
    if (!dst || !host || (size_t)bytes != want)
        return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_load: tensor %d layer %d wants %zu bytes, got %lld", which, layer, want,
                    (long long)bytes);
    DMC_CUDA_TRY(cudaMemcpyAsync(dst, host, want, cudaMemcpyHostToDevice, ctx().stream));
    DMC_CUDA_TRY(cudaStreamSynchronize(ctx().stream));
    return DMC_CUDA_OK;
}

extern "C" int dmc_decoder_step(void *dec, int token, int pos, int *next_token, float *logits_out) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return dmc::status();
    Decoder *d = static_cast<Decoder *>(dec);
    if (d->kv8) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_step: a decoder with an 8-bit cache is stepped by dmc_decoder_step_kv8");
    if (pos < 0 || pos >= d->cfg.max_len) return fail(DMC_CUDA_ERR_BAD_ARG, "decoder_step: pos %d outside the cache", pos);
    cudaStream_t s = ctx().stream;
    const int tp[2] = {token, pos};
    DMC_CUDA_TRY(cudaMemcpyAsync(d->d_token, &tp[0], 4, cudaMemcpyHostToDevice, s));
    DMC_CUDA_TRY(cudaMemcpyAsync(d->d_pos, &tp[1], 4, cudaMemcpyHostToDevice, s));
    DMC_CUDA_TRY(cudaStreamSynchronize(s));  // tp lives on this stack frame
    // (the first call also runs the step once eagerly before capturing it: token and pos are already
    // in place, so that run writes the same cache slot with the same values)
    int rc = ensure_graph(*d);
    if (rc) return rc;
    DMC_CUDA_TRY(cudaGraphLaunch(d->exec, s));
    ctx().launches += d->launches_per_step;
    int next = 0;
    unsigned long long key = 0ull;
    if (d->fused) DMC_CUDA_TRY(cudaMemcpyAsync(&key, d->am_key, 8, cudaMemcpyDeviceToHost, s));
    else DMC_CUDA_TRY(cudaMemcpyAsync(&next, d->d_next, 4, cudaMemcpyDeviceToHost, s));
    if (logits_out) DMC_CUDA_TRY(cudaMemcpyAsync(logits_out, d->logits, (size_t)d->cfg.vocab * 4, cudaMemcpyDeviceToHost, s));
    DMC_CUDA_TRY(cudaStreamSynchronize(s));
    stream_drained();
    if (d->fused) next = key ? (int)(0xFFFFFFFFu - (unsigned)(key & 0xFFFFFFFFull)) : 0;  // low half: 0xFFFFFFFF - row
    if (next_token) *next_token = next;
    return dmc::status();
}

extern "C" double dmc_decoder_bench(void *dec, int token, int pos, int steps, int warmup) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    if (dmc::status()) return -1.0;
    Decoder *d = static_cast<Decoder *>(dec);
    cudaStream_t s = ctx().stream;
    if (steps < 1 || warmup < 0 || pos < 0 || pos >= d->cfg.max_len) {
        fail(DMC_CUDA_ERR_BAD_ARG, "decoder_bench: bad steps/warmup/pos");
        return -1.0;
    }
    if (d->kv8 && pos != d->kv8->lens[0] - 1) {
        fail(DMC_CUDA_ERR_BAD_ARG, "decoder_bench: sequence 0 holds %d tokens: its last position has to be repeated", d->kv8->lens[0]);
        return -1.0;
    }
    if (d->kv8 && d->kv8->shared[0]) {
        fail(DMC_CUDA_ERR_BAD_ARG, "decoder_bench: another sequence may hold the last page of sequence 0, which would be written to");
        return -1.0;
    }
    cudaEvent_t e0 = nullptr, e1 = nullptr;
    double us = -1.0;
    auto body = [&]() -> int {
        const int tp[2] = {token, pos};
        if (d->kv8) {
            *d->kv8->h_in = StepIn{token, 0, pos + 1, 0, 0.0f, 1.0f, 0.0f, 0.0f};
            DMC_CUDA_TRY(cudaMemcpyAsync(d->kv8->in, d->kv8->h_in, sizeof(StepIn), cudaMemcpyHostToDevice, s));
        }
        DMC_CUDA_TRY(cudaMemcpyAsync(d->d_token, &tp[0], 4, cudaMemcpyHostToDevice, s));
        DMC_CUDA_TRY(cudaMemcpyAsync(d->d_pos, &tp[1], 4, cudaMemcpyHostToDevice, s));
        DMC_CUDA_TRY(cudaStreamSynchronize(s));
        int rc = ensure_graph(*d);
        if (rc) return rc;
        DMC_CUDA_TRY(cudaEventCreate(&e0));
        DMC_CUDA_TRY(cudaEventCreate(&e1));
        for (int i = 0; i < warmup; ++i) DMC_CUDA_TRY(cudaGraphLaunch(d->exec, s));
        DMC_CUDA_TRY(cudaStreamSynchronize(s));
        DMC_CUDA_TRY(cudaEventRecord(e0, s));
        for (int i = 0; i < steps; ++i) DMC_CUDA_TRY(cudaGraphLaunch(d->exec, s));
        DMC_CUDA_TRY(cudaEventRecord(e1, s));
        DMC_CUDA_TRY(cudaStreamSynchronize(s));
        ctx().launches += d->launches_per_step * (warmup + steps);
        float ms = 0.0f;
        DMC_CUDA_TRY(cudaEventElapsedTime(&ms, e0, e1));
        us = (double)ms * 1000.0 / steps;
        return DMC_CUDA_OK;
    };
    body();
    if (e0) cudaEventDestroy(e0);
    if (e1) cudaEventDestroy(e1);
    return dmc::status() ? -1.0 : us;
}

extern "C" int64_t dmc_decoder_launches_per_step(void *dec) { return static_cast<Decoder *>(dec)->launches_per_step; }

extern "C" void dmc_decoder_destroy(void *dec) {
    std::lock_guard<std::mutex> lock(ctx_mutex());
    Decoder *d = static_cast<Decoder *>(dec);
    if (!d) return;
    if (ctx().ready) cudaStreamSynchronize(ctx().stream);
    free_decoder(d);
}
