// C entries of the operators over a paged cache (include/timestral_b200.h): every check that the
// host can make, before any device work.
#include "paged.cuh"
#include "timestral_b200.h"

#include <climits>
#include <cmath>
#include <cstdio>
#include <string>

namespace tsb {
void set_thread_error(const char* message);
}

namespace {

struct Refusal {
    const char* call;
    char text[224];
    int code = TSB_OK;
    explicit Refusal(const char* name) : call(name) { text[0] = 0; }
    // false (and the first message kept) when `ok` does not hold
    template <class... A>
    bool need(bool ok, const char* fmt, A... args) {
        if (ok || code != TSB_OK) return ok;
        char what[160];
        if constexpr (sizeof...(A) == 0) std::snprintf(what, sizeof(what), "%s", fmt);
        else std::snprintf(what, sizeof(what), fmt, args...);
        std::snprintf(text, sizeof(text), "%s: %s", call, what);
        code = TSB_ERR_ARG;
        return false;
    }
    int report() const {
        if (code != TSB_OK) tsb::set_thread_error(text);
        return code;
    }
};

// Memory of the current device: a host pointer, or one of another device, would fault in the
// kernel, so it is refused here.
bool on_device(Refusal& r, const void* p, const char* name, int dev) {
    if (!r.need(p != nullptr, "%s is NULL", name)) return false;
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return r.need(false, "%s is not device memory", name);
    }
    return r.need(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged, "%s is not device memory", name) &&
           r.need(at.type == cudaMemoryTypeManaged || at.device == dev, "%s is memory of device %d, the current device is %d", name,
                  at.device, dev);
}

bool aligned(Refusal& r, const void* p, const char* name, unsigned bytes) {
    return r.need(reinterpret_cast<uintptr_t>(p) % bytes == 0, "%s is not %u-byte aligned", name, bytes);
}

bool values_type(Refusal& r, int type) {
    return r.need(type == TSB_TYPE_F16 || type == TSB_TYPE_BF16, "type %d is neither f16 (1) nor bf16 (30)", type);
}

// Shapes and strides alone: what needs no device.
bool heads_shape(Refusal& r, const tsb_heads& h, const char* name, int heads, int head_dim) {
    return aligned(r, h.data, name, 16) &&
           r.need(h.token_stride % 8 == 0 && h.head_stride % 8 == 0, "%s has a stride that is not a multiple of 8 elements", name) &&
           r.need(h.token_stride >= 0 && h.head_stride >= (heads > 1 ? head_dim : 0), "%s has heads that overlap", name);
}
// An output also must not have tokens that share memory.
bool output_shape(Refusal& r, const tsb_heads& h, const char* name, int tokens, int heads, int head_dim) {
    const int64_t token = (heads > 1 ? h.head_stride * (heads - 1) : 0) + head_dim;
    const bool apart = tokens <= 1 || h.token_stride >= token ||
                       (h.token_stride >= head_dim && h.head_stride >= h.token_stride * (tokens - 1) + head_dim) || (heads == 1 && h.token_stride >= head_dim);
    return heads_shape(r, h, name, heads, head_dim) && r.need(apart, "%s has tokens that overlap", name);
}
// An output in its input's place has its layout: a block would write what another has not read yet.
bool in_place_shape(Refusal& r, const tsb_heads& in, const tsb_heads& out, const char* name, int tokens, int heads) {
    return r.need(in.data != out.data || ((tokens <= 1 || in.token_stride == out.token_stride) && (heads <= 1 || in.head_stride == out.head_stride)),
                  "%s is its input with other strides", name);
}

bool rotation_shape(Refusal& r, const tsb_rotation& t, int head_dim, bool positions_needed) {
    if (!t.cos && !t.sin) return true;
    return r.need(t.cos && t.sin, "one of cos and sin is NULL") &&
           r.need(t.rope_dim >= 16 && t.rope_dim <= head_dim && t.rope_dim % 16 == 0,
                  "rope_dim %d is not a multiple of 16 up to head_dim %d", t.rope_dim, head_dim) &&
           r.need(t.rows > 0, "the rotation tables have %d rows", t.rows) &&
           r.need(t.stride >= t.rope_dim / 2 && t.stride % 4 == 0, "the rotation tables' stride must be a multiple of 4 of at least rope_dim / 2") &&
           aligned(r, t.cos, "cos", 16) && aligned(r, t.sin, "sin", 16) &&
           r.need(t.positions || !positions_needed, "positions is NULL");
}

bool cache_shape(Refusal& r, const tsb_paged_cache* c) {
    return r.need(c != nullptr, "cache is NULL") && values_type(r, c->type) &&
           r.need(c->head_dim == 64 || c->head_dim == 128, "head_dim %d is neither 64 nor 128", c->head_dim) &&
           r.need(c->page_size >= 8 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
                  "page_size %d is not a power of two from 8 to 1024", c->page_size) &&
           r.need(c->num_pages > 0 && c->kv_heads > 0, "the cache has %d pages of %d heads", c->num_pages, c->kv_heads) &&
           r.need(c->table_width >= 0 && c->table_stride >= 0, "the page table's width or stride is negative") &&
           aligned(r, c->k, "cache k", 16) && aligned(r, c->v, "cache v", 16) && aligned(r, c->table, "table", 4) &&
           r.need(c->k_page_stride % 8 == 0 && c->k_head_stride % 8 == 0 && c->k_slot_stride % 8 == 0 && c->v_page_stride % 8 == 0 &&
                      c->v_head_stride % 8 == 0 && c->v_slot_stride % 8 == 0,
                  "the cache has a stride that is not a multiple of 8 elements") &&
           r.need(c->k_page_stride >= 0 && c->v_page_stride >= 0 && c->k_slot_stride >= c->head_dim && c->v_slot_stride >= c->head_dim &&
                      c->k_head_stride >= (c->kv_heads > 1 ? c->head_dim : 0) && c->v_head_stride >= (c->kv_heads > 1 ? c->head_dim : 0),
                  "the cache has strides that overlap");
}

bool batch_shape(Refusal& r, const tsb_paged_batch* b, const tsb_paged_cache* c, int tokens) {
    return r.need(b != nullptr, "batch is NULL") &&
           r.need(b->seqs >= 0 && b->max_chunk >= 0 && b->max_length >= 0 && tokens >= 0, "a size is negative") &&
           aligned(r, b->q_start, "q_start", 4) && aligned(r, b->lengths, "lengths", 4) &&
           r.need(b->max_length <= INT_MAX - 1024, "max_length %d is above 2^31 - 1025", b->max_length) &&
           r.need(int64_t(b->max_length) <= int64_t(c->table_width) * c->page_size,
                  "max_length %d is more than the page table holds (%d pages of %d)", b->max_length, c->table_width, c->page_size);
}

tsb::PagedHeads view(const tsb_heads& h) {
    tsb::PagedHeads v;
    v.data = h.data; v.token = h.token_stride; v.head = h.head_stride;
    return v;
}
tsb::PagedRotation view(const tsb_rotation& t) {
    tsb::PagedRotation v;
    if (!t.cos) return v;
    v.cos = t.cos; v.sin = t.sin; v.stride = t.stride; v.rows = t.rows; v.dim = t.rope_dim; v.positions = t.positions;
    return v;
}
tsb::PagedCache view(const tsb_paged_cache& c) {
    tsb::PagedCache v;
    v.k = c.k; v.v = c.v;
    v.k_page = c.k_page_stride; v.k_head = c.k_head_stride; v.k_slot = c.k_slot_stride;
    v.v_page = c.v_page_stride; v.v_head = c.v_head_stride; v.v_slot = c.v_slot_stride;
    v.table = c.table; v.table_stride = c.table_stride; v.num_pages = c.num_pages;
    v.kv_heads = c.kv_heads; v.head_dim = c.head_dim;
    while ((1 << v.page_shift) < c.page_size) ++v.page_shift;
    return v;
}
tsb::PagedBatch view(const tsb_paged_batch& b, int tokens) {
    tsb::PagedBatch v;
    v.q_start = b.q_start; v.lengths = b.lengths; v.seqs = b.seqs; v.max_length = b.max_length;
    v.max_chunk = b.max_chunk < tokens ? b.max_chunk : tokens;      // more than there are cannot be
    v.tokens = tokens;
    return v;
}

bool cache_on_device(Refusal& r, const tsb_paged_cache& c, const tsb_paged_batch& b, int dev) {
    return on_device(r, c.k, "cache k", dev) && on_device(r, c.v, "cache v", dev) && on_device(r, c.table, "table", dev) &&
           on_device(r, b.q_start, "q_start", dev) && on_device(r, b.lengths, "lengths", dev);
}
bool rotation_on_device(Refusal& r, const tsb_rotation& t, int dev) {
    return !t.cos || (on_device(r, t.cos, "cos", dev) && on_device(r, t.sin, "sin", dev) &&
                      (!t.positions || (aligned(r, t.positions, "positions", 4) && on_device(r, t.positions, "positions", dev))));
}
bool error_word(Refusal& r, int32_t* error, int dev) {
    return !error || (aligned(r, error, "error", 4) && on_device(r, error, "error", dev));
}

int launched(Refusal& r, cudaError_t e) {
    if (e == cudaSuccess) return TSB_OK;
    std::snprintf(r.text, sizeof(r.text), "%s: %s", r.call, e == cudaErrorInvalidValue ? "a size or stride that does not fit a launch or a tensor map" : cudaGetErrorString(e));
    cudaGetLastError();
    r.code = e == cudaErrorInvalidValue ? TSB_ERR_ARG : TSB_ERR_CUDA;
    return r.report();
}

bool current_device(Refusal& r, int* dev) {
    const cudaError_t e = cudaGetDevice(dev);
    if (e == cudaSuccess) return true;
    cudaGetLastError();
    r.need(false, "no usable CUDA device");
    r.code = TSB_ERR_CUDA;
    return false;
}

bool attention_shape(Refusal& r, const tsb_paged_attention_args* a, bool pointers) {
    if (!r.need(a != nullptr, "args is NULL") || !cache_shape(r, a->cache) || !batch_shape(r, a->batch, a->cache, a->tokens)) return false;
    const tsb_paged_cache& c = *a->cache;
    if (!r.need(a->q_heads > 0 && a->q_heads % c.kv_heads == 0, "q_heads %d is not a multiple of kv_heads %d", a->q_heads, c.kv_heads) ||
        !r.need(int64_t(a->tokens) * a->q_heads <= INT_MAX, "%d tokens of %d heads are more than 2^31 - 1 rows", a->tokens, a->q_heads) ||
        !r.need(a->window >= 0, "window %d is negative", a->window))
        return false;
    return !pointers ||
           (heads_shape(r, a->q, "q", a->q_heads, c.head_dim) && output_shape(r, a->out, "out", a->tokens, a->q_heads, c.head_dim) &&
            in_place_shape(r, a->q, a->out, "out", a->tokens, a->q_heads) &&
            (!a->gate.data || heads_shape(r, a->gate, "gate", a->q_heads, c.head_dim)) &&
            r.need(std::isfinite(a->scale), "scale is not finite") &&
            r.need(!a->key_valid || (a->key_valid_positions >= 0 && a->key_valid_stride >= (int64_t(a->key_valid_positions) + 31) / 32),
                   "key_valid_stride holds fewer bits than key_valid_positions") &&
            aligned(r, a->key_valid, "key_valid", 4) && aligned(r, a->workspace, "workspace", 16));
}

tsb::PagedAttention attention_of(const tsb_paged_attention_args& a) {
    tsb::PagedAttention p;
    p.cache = view(*a.cache);
    p.batch = view(*a.batch, a.tokens);
    p.q = view(a.q); p.out = view(a.out);
    if (a.gate.data) p.gate = view(a.gate);
    p.q_heads = a.q_heads; p.group = a.q_heads / a.cache->kv_heads;
    p.window = a.window; p.self_visible = a.self_visible != 0;
    const double scale = a.scale != 0.f ? double(a.scale) : 1.0 / std::sqrt(double(a.cache->head_dim));
    p.scale_log2 = float(scale * 1.4426950408889634);
    p.key_valid = reinterpret_cast<const uint32_t*>(a.key_valid);
    p.key_valid_stride = a.key_valid_stride;
    p.key_valid_positions = a.key_valid ? a.key_valid_positions : 0;
    p.err = a.error;
    return p;
}

}  // namespace

extern "C" TIMESTRAL_API int tsb_norm_rope(const tsb_norm_rope_args* a, void* stream) {
    Refusal r("tsb_norm_rope");
    if (!r.need(a != nullptr, "args is NULL") || !values_type(r, a->type) ||
        !r.need(a->head_dim >= 16 && a->head_dim <= 256 && a->head_dim % 16 == 0, "head_dim %d is not a multiple of 16 up to 256", a->head_dim) ||
        !r.need(a->tokens >= 0 && a->q_heads >= 0 && a->k_heads >= 0, "a size is negative") ||
        !r.need(std::isfinite(a->eps) && a->eps >= 0, "eps is negative or not finite") ||
        !rotation_shape(r, a->rotation, a->head_dim, a->tokens > 0))       // (no token: an empty array may have no address)
        return r.report();
    const struct { const tsb_heads &in, &out; const float* w; int heads; const char *name, *out_name, *w_name; } side[2] = {
        {a->q, a->q_out, a->q_weight, a->q_heads, "q", "q_out", "q_weight"}, {a->k, a->k_out, a->k_weight, a->k_heads, "k", "k_out", "k_weight"}};
    for (const auto& s : side)
        if (s.heads && (!heads_shape(r, s.in, s.name, s.heads, a->head_dim) || !output_shape(r, s.out, s.out_name, a->tokens, s.heads, a->head_dim) ||
                        !in_place_shape(r, s.in, s.out, s.out_name, a->tokens, s.heads) ||
                        !aligned(r, s.w, s.w_name, 16)))
            return r.report();
    if (!a->tokens || (!a->q_heads && !a->k_heads)) return TSB_OK;
    int dev = 0;
    if (!current_device(r, &dev)) return r.report();
    for (const auto& s : side)
        if (s.heads && (!on_device(r, s.in.data, s.name, dev) || (s.out.data != s.in.data && !on_device(r, s.out.data, s.out_name, dev)) ||
                        (s.w && !on_device(r, s.w, s.w_name, dev))))
            return r.report();
    if (!rotation_on_device(r, a->rotation, dev) || !error_word(r, a->error, dev)) return r.report();
    tsb::NormRope n;
    tsb::NormRopeSide* to[2] = {&n.q, &n.k};
    for (int i = 0; i < 2; ++i) {
        to[i]->in = view(side[i].in); to[i]->out = view(side[i].out);
        to[i]->weight = side[i].w; to[i]->heads = side[i].heads;
    }
    n.rot = view(a->rotation);
    n.tokens = a->tokens; n.head_dim = a->head_dim; n.eps = a->eps; n.err = a->error;
    return launched(r, tsb::norm_rope(n, a->type == TSB_TYPE_BF16, static_cast<cudaStream_t>(stream)));
}

extern "C" TIMESTRAL_API int tsb_paged_append(const tsb_paged_append_args* a, void* stream) {
    Refusal r("tsb_paged_append");
    if (!r.need(a != nullptr, "args is NULL") || !cache_shape(r, a->cache) || !batch_shape(r, a->batch, a->cache, a->tokens) ||
        !heads_shape(r, a->k, "k", a->cache->kv_heads, a->cache->head_dim) || !heads_shape(r, a->v, "v", a->cache->kv_heads, a->cache->head_dim) ||
        !aligned(r, a->k_weight, "k_weight", 16) || !r.need(std::isfinite(a->eps) && a->eps >= 0, "eps is negative or not finite") ||
        !rotation_shape(r, a->rotation, a->cache->head_dim, false))
        return r.report();
    if (!a->tokens || !a->batch->seqs || !a->batch->max_chunk) return TSB_OK;
    int dev = 0;
    if (!current_device(r, &dev) || !cache_on_device(r, *a->cache, *a->batch, dev) || !on_device(r, a->k.data, "k", dev) ||
        !on_device(r, a->v.data, "v", dev) || (a->k_weight && !on_device(r, a->k_weight, "k_weight", dev)) ||
        !rotation_on_device(r, a->rotation, dev) || !error_word(r, a->error, dev))
        return r.report();
    tsb::PagedAppend p;
    p.cache = view(*a->cache);
    p.batch = view(*a->batch, a->tokens);
    p.k = view(a->k); p.v = view(a->v);
    p.k_weight = a->k_weight; p.eps = a->eps; p.rot = view(a->rotation); p.err = a->error;
    return launched(r, tsb::paged_append(p, a->cache->type == TSB_TYPE_BF16, static_cast<cudaStream_t>(stream)));
}

extern "C" TIMESTRAL_API size_t tsb_paged_attention_workspace(const tsb_paged_attention_args* a) {
    Refusal r("tsb_paged_attention_workspace");
    if (!attention_shape(r, a, false)) { r.report(); return 0; }
    if (!a->tokens || !a->batch->seqs || !a->batch->max_chunk) return 0;
    const tsb::PagedPlan p = tsb::paged_plan(attention_of(*a));
    return p.splits > 1 && p.splits > p.cluster ? size_t(p.splits) * p.split_bytes : 0;
}

extern "C" TIMESTRAL_API int tsb_paged_attention(const tsb_paged_attention_args* a, void* stream) {
    Refusal r("tsb_paged_attention");
    if (!attention_shape(r, a, true)) return r.report();
    if (!a->tokens || !a->batch->seqs || !a->batch->max_chunk) return TSB_OK;
    int dev = 0;
    if (!current_device(r, &dev) || !cache_on_device(r, *a->cache, *a->batch, dev) || !on_device(r, a->q.data, "q", dev) ||
        (a->out.data != a->q.data && !on_device(r, a->out.data, "out", dev)) || (a->gate.data && !on_device(r, a->gate.data, "gate", dev)) ||
        (a->key_valid && !on_device(r, a->key_valid, "key_valid", dev)) ||
        (a->workspace_bytes && !on_device(r, a->workspace, "workspace", dev)) || !error_word(r, a->error, dev))
        return r.report();
    tsb::PagedAttention p = attention_of(*a);
    tsb::paged_workspace(&p, a->workspace, a->workspace_bytes);
    return launched(r, tsb::paged_attention(p, a->cache->type == TSB_TYPE_BF16, static_cast<cudaStream_t>(stream)));
}
