// Attention of the newest tokens of some sequences over a caller-owned cache (prism_cuda_cache_attention_dev).
#include <cmath>
#include <stdexcept>

#include "cache_attn.cuh"

namespace prism {

// A warp per (row, query head), position by position.
template <int KIND, int HD>
__global__ void __launch_bounds__(128) cache_attn_plain_kernel(const CacheAttnDev a) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 5), token = unit / a.heads, head = unit % a.heads;
    CacheEntry x;
    if (!cache_entry(a, blockIdx.y, x) || token >= x.n) return;
    cache_plain_row<KIND, HD>(a, x, token, head, threadIdx.x & 31);
}

template <int KIND>
static void launch_plain(prism_cuda_ctx *ctx, uint32_t hd, const CacheAttnDev &a) {
    const dim3 grid((uint32_t)(((uint64_t)a.max_tokens * a.heads + 3) / 4), a.n_entries), block(128);
    switch (hd) {
    case 32: return launch_pdl(ctx, "cache_attn_plain_kernel", cache_attn_plain_kernel<KIND, 32>, grid, block, 0, a);
    case 64: return launch_pdl(ctx, "cache_attn_plain_kernel", cache_attn_plain_kernel<KIND, 64>, grid, block, 0, a);
    case 128: return launch_pdl(ctx, "cache_attn_plain_kernel", cache_attn_plain_kernel<KIND, 128>, grid, block, 0, a);
    default: return launch_pdl(ctx, "cache_attn_plain_kernel", cache_attn_plain_kernel<KIND, 256>, grid, block, 0, a);
    }
}

static int cache_attention(prism_cuda_ctx *ctx, const prism_cache *c, const prism_cache_attention *p) {
    if (!ctx || !c || !p) return fail(ctx, PRISM_E_NULL, "cache_attention: null argument");
    CacheAttnDev a{};
    int kind;
    PRISM_TRY(kv_check(ctx, c, &a.c, &kind));
    if (p->num_heads == 0 || p->num_heads > 65536 || p->num_heads % c->kv_heads)
        return fail(ctx, PRISM_E_ARG, "cache_attention: num_heads must be a multiple of kv_heads, at most 65536");
    if (p->n_entries > 65535) return fail(ctx, PRISM_E_ARG, "cache_attention: at most 65535 entries a call");
    if (p->n_rows > 0x7FFFFFFFu || p->max_tokens > (1u << 24) || (uint64_t)p->max_tokens * p->num_heads > (1u << 30))
        return fail(ctx, PRISM_E_ARG, "cache_attention: too many rows");
    if (p->tree && (p->tree_words == 0 || (uint64_t)p->tree_words * 64 < p->max_tokens))
        return fail(ctx, PRISM_E_ARG, "cache_attention: a row's mask needs a bit for each of max_tokens tokens");
    if (p->tree && p->window && !p->q_pos) return fail(ctx, PRISM_E_NULL, "cache_attention: a tree under a window needs the rows' positions");
    if (!std::isfinite(p->scale)) return fail(ctx, PRISM_E_ARG, "cache_attention: the scale of the scores must be finite");
    if (p->n_entries == 0 || p->n_rows == 0 || p->max_tokens == 0) return PRISM_OK;
    if (!p->q || !p->out || !p->seq || !p->q_start || !p->length) return fail(ctx, PRISM_E_NULL, "cache_attention: null argument");
    const uint64_t width = (uint64_t)p->num_heads * c->head_dim;
    if (p->q_stride < width || p->out_stride < width || p->q_stride % 8 || p->out_stride % 8 ||
        ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out)) & 15))
        return fail(ctx, PRISM_E_ARG, "cache_attention: rows must be 16-byte aligned and at least num_heads * head_dim values apart");
    if (reinterpret_cast<uintptr_t>(p->tree) & 7) return fail(ctx, PRISM_E_ARG, "cache_attention: masks must be 8-byte aligned");
    DeviceGuard on(ctx->device);
    if (on.err != cudaSuccess) return cuda_fail(ctx, on.err, "cudaSetDevice");
    a.q = static_cast<const uint16_t *>(p->q);
    a.out = static_cast<uint16_t *>(p->out);
    a.q_stride = p->q_stride;
    a.out_stride = p->out_stride;
    a.n_rows = p->n_rows;
    a.n_entries = p->n_entries;
    a.seq = p->seq;
    a.q_start = p->q_start;
    a.length = p->length;
    a.max_tokens = p->max_tokens;
    a.heads = p->num_heads;
    a.group = p->num_heads / c->kv_heads;
    a.window = p->window;
    a.sinks = p->window ? p->sinks : 0;
    a.scale = p->scale != 0.0f ? p->scale : 1.0f / sqrtf((float)c->head_dim);
    a.tree = p->tree;
    a.tree_words = p->tree_words;
    a.q_pos = p->q_pos;
    switch (kind) {
    case KV_F16: launch_plain<KV_F16>(ctx, c->head_dim, a); break;
    case KV_BF16: launch_plain<KV_BF16>(ctx, c->head_dim, a); break;
    case KV_INT8: launch_plain<KV_INT8>(ctx, c->head_dim, a); break;
    case KV_E4M3: launch_plain<KV_E4M3>(ctx, c->head_dim, a); break;
    default: launch_plain<KV_INT4>(ctx, c->head_dim, a); break;
    }
    return after_launch(ctx, "cache_attn_plain_kernel");
}

}  // namespace prism

using namespace prism;

extern "C" int prism_cuda_cache_attention_dev(prism_cuda_ctx *ctx, const prism_cache *cache, const prism_cache_attention *a) {
    try {
        return cache_attention(ctx, cache, a);
    } catch (const std::exception &) {
        return PRISM_E_STATE;  // no memory for a message
    }
}
