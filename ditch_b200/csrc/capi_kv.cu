// The C entries of the paged 8-bit key / value cache and of windowed
// attention: the checks of their arguments and the launches.
#include <algorithm>

#include "device.cuh"
#include "kvcache.cuh"

using namespace ditch;

namespace {

#define REQUIRE(cond, ...)              \
    do {                                \
        if (!(cond)) {                  \
            set_error(__VA_ARGS__);     \
            return DITCH_CUDA_INVALID;  \
        }                               \
    } while (0)

constexpr size_t kMaxCount = 1u << 30;  // rows, tokens and sequences of one call

int log2_of(int v) {
    int n = 0;
    while ((1 << n) < v) n++;
    return n;
}

size_t type_bytes(int dtype) { return dtype == DITCH_DTYPE_F32 ? 4 : 2; }

int take_cache(const ditch_cuda_kv_cache *c, kv::Cache *out) {
    REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "kv cache: null pool");
    REQUIRE(c->format == DITCH_KV_INT8 || c->format == DITCH_KV_FP8, "kv cache: unknown format %d", c->format);
    REQUIRE(c->kv_heads > 0 && c->kv_heads <= 65535, "kv cache: bad head count %d", c->kv_heads);
    REQUIRE(c->head_dim > 0, "kv cache: bad head size %d", c->head_dim);
    if (c->head_dim % 16 || c->head_dim > 128) {
        set_error("kv cache: head size %d (multiples of 16 up to 128 are taken)", c->head_dim);
        return DITCH_CUDA_UNSUPPORTED;
    }
    const int p = c->page_tokens, b = c->block_tokens;
    REQUIRE(p >= 16 && p <= 256 && (p & (p - 1)) == 0, "kv cache: pages of %d tokens", p);
    REQUIRE((b == 16 || b == 32 || b == 64) && b <= p, "kv cache: blocks of %d tokens in pages of %d", b, p);
    REQUIRE(c->n_pages > 0 && c->n_pages <= 0x7fffffff, "kv cache: %zu pages", c->n_pages);
    REQUIRE(!((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15),
            "kv cache: codes must be 16-byte aligned");
    REQUIRE(!((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3),
            "kv cache: scales must be 4-byte aligned");
    out->k = static_cast<uint8_t *>(c->k);
    out->v = static_cast<uint8_t *>(c->v);
    out->ks = c->k_scale;
    out->vs = c->v_scale;
    out->n_pages = static_cast<long long>(c->n_pages);
    out->fp8 = c->format == DITCH_KV_FP8;
    out->heads = c->kv_heads;
    out->dim = c->head_dim;
    out->page_shift = log2_of(p);
    out->block_shift = log2_of(b);
    return DITCH_CUDA_OK;
}

int take_batch(const ditch_cuda_kv_batch *b, kv::Batch *out) {
    REQUIRE(b->n_seqs < kMaxCount && b->n_tokens < kMaxCount && b->max_new < kMaxCount && b->max_len < kMaxCount &&
                b->max_pages < kMaxCount,
            "kv batch: a count is too large");
    REQUIRE(b->n_seqs == 0 || (b->offsets && b->lens && b->pages), "kv batch: null argument");
    REQUIRE(b->max_new <= b->n_tokens && b->max_new <= b->max_len, "kv batch: max_new %zu exceeds n_tokens or max_len",
            b->max_new);
    REQUIRE(b->n_tokens == 0 || (b->n_seqs > 0 && b->max_new > 0 && b->n_tokens <= b->n_seqs * b->max_new),
            "kv batch: %zu tokens in %zu sequences of at most %zu", b->n_tokens, b->n_seqs, b->max_new);
    out->offsets = b->offsets;
    out->lens = b->lens;
    out->pages = b->pages;
    out->n_seqs = static_cast<int>(b->n_seqs);
    out->n_tokens = static_cast<int>(b->n_tokens);
    out->max_new = static_cast<int>(b->max_new);
    out->max_len = static_cast<int>(b->max_len);
    out->max_pages = static_cast<int>(b->max_pages);
    return DITCH_CUDA_OK;
}

// A null `r` (or data) gives p = null.
int take_rows(const ditch_cuda_rows *r, const char *name, int dim, kv::Rows *out) {
    *out = kv::Rows{};
    if (!r) return DITCH_CUDA_OK;
    REQUIRE(r->data, "%s: null rows", name);
    if (r->dtype != DITCH_DTYPE_F32 && r->dtype != DITCH_DTYPE_F16 && r->dtype != DITCH_DTYPE_BF16) {
        set_error("%s: dtype %d (f32, f16 and bf16 rows are taken)", name, r->dtype);
        return DITCH_CUDA_UNSUPPORTED;
    }
    REQUIRE(r->heads > 0 && r->heads <= 65535, "%s: bad head count %d", name, r->heads);
    const size_t e = type_bytes(r->dtype);
    REQUIRE(!(reinterpret_cast<uintptr_t>(r->data) & (e - 1)), "%s: rows must be aligned to their elements", name);
    REQUIRE(r->token_stride < (1ull << 40) && r->head_stride < (1ull << 40), "%s: a stride is too large", name);
    REQUIRE(r->heads == 1 || r->head_stride >= static_cast<size_t>(dim), "%s: heads overlap", name);
    out->p = r->data;
    out->dtype = r->dtype;
    out->heads = r->heads;
    out->ts = static_cast<long long>(r->token_stride);
    out->hs = static_cast<long long>(r->head_stride);
    out->vec = !((reinterpret_cast<uintptr_t>(r->data) | r->token_stride * e | r->head_stride * e) & 15);
    return DITCH_CUDA_OK;
}

}  // namespace

#define TAKE(expr)            \
    do {                      \
        int _s = (expr);      \
        if (_s) return _s;    \
    } while (0)

extern "C" {

int ditch_cuda_kv_append(ditch_cuda_device *dev, const ditch_cuda_kv_cache *cache, const ditch_cuda_kv_batch *batch,
                         const ditch_cuda_rope *rope, const ditch_cuda_rows *q, const ditch_cuda_rows *q_out,
                         const ditch_cuda_rows *k, const ditch_cuda_rows *v, const ditch_cuda_rows *k_out,
                         const ditch_cuda_rows *v_out, void *stream) {
    clear_error();
    REQUIRE(dev && cache && batch && k && v, "kv_append: null argument");
    kv::AppendParams p{};
    TAKE(take_cache(cache, &p.c));
    TAKE(take_batch(batch, &p.b));
    const int d = p.c.dim;
    TAKE(take_rows(q, "kv_append: q", d, &p.q));
    TAKE(take_rows(q_out, "kv_append: q_out", d, &p.qo));
    TAKE(take_rows(k, "kv_append: k", d, &p.k));
    TAKE(take_rows(v, "kv_append: v", d, &p.v));
    TAKE(take_rows(k_out, "kv_append: k_out", d, &p.ko));
    TAKE(take_rows(v_out, "kv_append: v_out", d, &p.vo));
    REQUIRE((q != nullptr) == (q_out != nullptr), "kv_append: q and q_out go together");
    REQUIRE(!q || q->heads == q_out->heads, "kv_append: q and q_out have different heads");
    REQUIRE(k->heads == p.c.heads && v->heads == p.c.heads && (!k_out || k_out->heads == p.c.heads) &&
                (!v_out || v_out->heads == p.c.heads),
            "kv_append: the rows' heads are not the cache's %d", p.c.heads);
    REQUIRE(k->dtype == v->dtype && (!q || q->dtype == k->dtype), "kv_append: q, k and v have different dtypes");
    if (rope) {
        REQUIRE(rope->cos_t && rope->sin_t, "kv_append: null RoPE tables");
        REQUIRE(!((reinterpret_cast<uintptr_t>(rope->cos_t) | reinterpret_cast<uintptr_t>(rope->sin_t)) & 15),
                "kv_append: the RoPE tables must be 16-byte aligned");
        REQUIRE(rope->style == 0 || rope->style == 1, "kv_append: style must be 0 (neox) or 1 (gptj)");
        REQUIRE(rope->half > 0 && 2 * rope->half <= static_cast<size_t>(d), "kv_append: rotated half exceeds the head");
        REQUIRE(rope->table_len >= batch->max_len && rope->table_len < kMaxCount,
                "kv_append: RoPE tables of %zu positions for %zu tokens", rope->table_len, batch->max_len);
        if (rope->half % 8) {
            set_error("kv_append: half %zu (multiples of 8 are taken)", rope->half);
            return DITCH_CUDA_UNSUPPORTED;
        }
        p.r.cos_t = rope->cos_t;
        p.r.sin_t = rope->sin_t;
        p.r.len = static_cast<int>(rope->table_len);
        p.r.half = static_cast<int>(rope->half);
        p.r.style = rope->style;
    }
    if (p.b.n_tokens == 0) return DITCH_CUDA_OK;
    std::lock_guard<std::mutex> lk(dev->mu);
    DITCH_CUDA(cudaSetDevice(dev->ordinal));
    p.status = dev->status;
    DITCH_LAUNCH(dev, kv::append(p, static_cast<cudaStream_t>(stream)));
    return DITCH_CUDA_OK;
}

int ditch_cuda_kv_read(ditch_cuda_device *dev, const ditch_cuda_kv_cache *cache, const ditch_cuda_kv_batch *batch,
                       const ditch_cuda_rows *k_out, const ditch_cuda_rows *v_out, void *stream) {
    clear_error();
    REQUIRE(dev && cache && batch && k_out && v_out, "kv_read: null argument");
    kv::ReadParams p{};
    TAKE(take_cache(cache, &p.c));
    TAKE(take_batch(batch, &p.b));
    TAKE(take_rows(k_out, "kv_read: k_out", p.c.dim, &p.ko));
    TAKE(take_rows(v_out, "kv_read: v_out", p.c.dim, &p.vo));
    REQUIRE(k_out->heads == p.c.heads && v_out->heads == p.c.heads, "kv_read: the rows' heads are not the cache's %d",
            p.c.heads);
    if (p.b.n_tokens == 0) return DITCH_CUDA_OK;
    std::lock_guard<std::mutex> lk(dev->mu);
    DITCH_CUDA(cudaSetDevice(dev->ordinal));
    p.status = dev->status;
    DITCH_LAUNCH(dev, kv::read_back(p, static_cast<cudaStream_t>(stream)));
    return DITCH_CUDA_OK;
}

size_t ditch_cuda_kv_attention_workspace(ditch_cuda_device *dev, const ditch_cuda_kv_cache *cache,
                                         const ditch_cuda_kv_batch *batch, size_t q_heads) {
    clear_error();
    kv::Cache c;
    kv::Batch b;
    if (!dev || !cache || !batch) {
        set_error("kv_attention_workspace: null argument");
        return 0;
    }
    if (take_cache(cache, &c) || take_batch(batch, &b)) return 0;
    if (q_heads == 0 || q_heads % c.heads || q_heads > 65535 || b.n_tokens == 0) return 0;
    return kv::attend_workspace(c, b, static_cast<int>(q_heads), dev->sms);
}

int ditch_cuda_kv_attention(ditch_cuda_device *dev, const ditch_cuda_kv_cache *cache, const ditch_cuda_kv_batch *batch,
                            const ditch_cuda_rows *q, const ditch_cuda_rows *out, float scale, size_t window,
                            size_t sinks, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    REQUIRE(dev && cache && batch && q && out, "kv_attention: null argument");
    kv::AttendParams p{};
    TAKE(take_cache(cache, &p.c));
    TAKE(take_batch(batch, &p.b));
    TAKE(take_rows(q, "kv_attention: q", p.c.dim, &p.q));
    TAKE(take_rows(out, "kv_attention: out", p.c.dim, &p.out));
    REQUIRE(q->heads == out->heads, "kv_attention: q and out have different heads");
    REQUIRE(q->heads % p.c.heads == 0, "kv_attention: %d query heads over %d kv heads", q->heads, p.c.heads);
    REQUIRE(scale > 0.0f && scale < 1e30f, "kv_attention: scale must be positive");
    REQUIRE(sinks == 0 || window > 0, "kv_attention: sinks without a window");
    if (p.b.n_tokens == 0) return DITCH_CUDA_OK;
    const size_t need = kv::attend_workspace(p.c, p.b, q->heads, dev->sms);
    REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "kv_attention: a workspace of %zu bytes is needed, %zu given",
            need, workspace ? workspace_bytes : 0);
    REQUIRE(!(reinterpret_cast<uintptr_t>(workspace) & 15), "kv_attention: the workspace must be 16-byte aligned");
    p.scale = scale;
    p.window = window >= kMaxCount ? 0 : static_cast<int>(window);
    p.sinks = static_cast<int>(std::min(sinks, kMaxCount));
    p.ws = workspace;
    std::lock_guard<std::mutex> lk(dev->mu);
    DITCH_CUDA(cudaSetDevice(dev->ordinal));
    p.status = dev->status;
    DITCH_LAUNCH(dev, kv::attend(p, dev->sms, static_cast<cudaStream_t>(stream)));
    return DITCH_CUDA_OK;
}

int ditch_cuda_window_attention(ditch_cuda_device *dev, const ditch_cuda_ragged *seqs, size_t head_dim,
                                const ditch_cuda_rows *q, const ditch_cuda_rows *k, const ditch_cuda_rows *v,
                                const ditch_cuda_rows *out, float scale, size_t window, size_t sinks, void *stream) {
    clear_error();
    REQUIRE(dev && seqs && q && k && v && out, "window_attention: null argument");
    REQUIRE(seqs->n_seqs < kMaxCount && seqs->n_q < kMaxCount && seqs->n_kv < kMaxCount && seqs->max_q <= seqs->n_q &&
                seqs->max_kv <= seqs->n_kv && seqs->n_q <= seqs->n_seqs * seqs->max_q,
            "window_attention: bad counts");
    REQUIRE(seqs->n_seqs <= kv::kTiledSeqs, "window_attention: %zu sequences (at most %d)", seqs->n_seqs, kv::kTiledSeqs);
    REQUIRE(seqs->n_seqs == 0 || (seqs->q_offsets && seqs->kv_offsets), "window_attention: null offsets");
    REQUIRE(head_dim > 0, "window_attention: bad head size");
    if (head_dim % 8 || head_dim > 128) {
        set_error("window_attention: head size %zu (multiples of 8 up to 128 are taken)", head_dim);
        return DITCH_CUDA_UNSUPPORTED;
    }
    kv::WindowParams p{};
    const int d = static_cast<int>(head_dim);
    TAKE(take_rows(q, "window_attention: q", d, &p.q));
    TAKE(take_rows(k, "window_attention: k", d, &p.k));
    TAKE(take_rows(v, "window_attention: v", d, &p.v));
    TAKE(take_rows(out, "window_attention: out", d, &p.out));
    REQUIRE(q->heads == out->heads && k->heads == v->heads && q->heads % k->heads == 0,
            "window_attention: %d query, %d key, %d value and %d output heads", q->heads, k->heads, v->heads, out->heads);
    REQUIRE(q->dtype == k->dtype && q->dtype == v->dtype && q->dtype == out->dtype,
            "window_attention: the rows have different dtypes");
    if (q->dtype == DITCH_DTYPE_F32) {
        set_error("window_attention: f16 and bf16 rows are taken");
        return DITCH_CUDA_UNSUPPORTED;
    }
    REQUIRE(scale > 0.0f && scale < 1e30f, "window_attention: scale must be positive");
    REQUIRE(sinks == 0 || window > 0, "window_attention: sinks without a window");
    if (seqs->n_q == 0) return DITCH_CUDA_OK;
    p.b.qo = seqs->q_offsets;
    p.b.ko = seqs->kv_offsets;
    p.b.n_seqs = static_cast<int>(seqs->n_seqs);
    p.b.n_q = static_cast<int>(seqs->n_q);
    p.b.n_kv = static_cast<int>(seqs->n_kv);
    p.b.max_q = static_cast<int>(seqs->max_q);
    p.b.max_kv = static_cast<int>(seqs->max_kv);
    p.dim = d;
    p.scale = scale;
    p.window = window >= kMaxCount ? 0 : static_cast<int>(window);
    p.sinks = static_cast<int>(std::min(sinks, kMaxCount));
    std::lock_guard<std::mutex> lk(dev->mu);
    DITCH_CUDA(cudaSetDevice(dev->ordinal));
    p.status = dev->status;
    DITCH_LAUNCH(dev, kv::window_attention(p, dev->sms, static_cast<cudaStream_t>(stream)));
    return DITCH_CUDA_OK;
}

}  // extern "C"
