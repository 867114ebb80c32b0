// hq_attn_api.cu -- C entry points of attention and the cache's device calls
// (include/hq.h): argument checks and dispatch.  Nothing throws or allocates.
#include "hq.h"
#include "hq_attn.h"
#include "hq_common.cuh"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <vector>

using namespace hq;

namespace {

hq_status fail(hq_status s, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);
    return s;
}

hq_status cuda_fail(cudaError_t e, const char* what) {
    return fail(HQ_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

hq_status check_device(int* dev_out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    const DeviceInfo& di = device_info(dev);
    if (di.cc_major != 10)
        return fail(HQ_ERR_UNSUPPORTED_DEVICE, "device %d is sm_%d%d; this library is built for sm_100a", dev, di.cc_major,
                    di.cc_minor);
    *dev_out = dev;
    return HQ_OK;
}

// Sizes and types; strides and pointers are checked per tensor below.
hq_status check_shape(const hq_attn_shape* s, bool attention) {
    if (!s) return fail(HQ_ERR_INVALID_ARG, "null shape");
    if (s->n_tokens < 0 || s->n_seqs < 0 || s->max_q_len < 0) return fail(HQ_ERR_INVALID_ARG, "negative size");
    if (s->dtype != HQ_F16 && s->dtype != HQ_BF16) return fail(HQ_ERR_INVALID_ARG, "dtype must be HQ_F16 or HQ_BF16");
    if (s->n_kv_heads <= 0 || s->n_kv_heads > 65535) return fail(HQ_ERR_INVALID_ARG, "n_kv_heads=%d", s->n_kv_heads);
    if (s->head_dim <= 0 || s->head_dim % 8 || s->head_dim > 128)
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "head_dim=%d must be a multiple of 8 up to 128", s->head_dim);
    if (!attention) return HQ_OK;
    if (s->n_heads <= 0 || s->n_heads % s->n_kv_heads)
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "n_heads=%d must be a multiple of n_kv_heads=%d", s->n_heads, s->n_kv_heads);
    if (s->n_heads / s->n_kv_heads > 128)
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "%d query heads a key/value head, more than 128", s->n_heads / s->n_kv_heads);
    if ((long long)s->n_tokens * s->n_heads > 0x7fffffffLL || (long long)s->n_seqs * s->n_heads > 0x7fffffffLL)
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "n_tokens * n_heads and n_seqs * n_heads must fit 31 bits");
    if (!(s->scale > 0.f) || !std::isfinite(s->scale)) return fail(HQ_ERR_INVALID_ARG, "scale must be positive and finite");
    return HQ_OK;
}

hq_status check_rows(const hq_rows* r, const char* name) {
    if (!r || !r->p) return fail(HQ_ERR_INVALID_ARG, "null %s", name);
    if (!aligned16(r->p)) return fail(HQ_ERR_MISALIGNED, "%s must be 16-byte aligned", name);
    if (r->stride_token < 0 || r->stride_head < 0 || r->stride_token % 8 || r->stride_head % 8)
        return fail(HQ_ERR_MISALIGNED, "%s: strides must be non-negative multiples of 8 elements", name);
    return HQ_OK;
}

hq_status check_pages(const hq_pages* r, const char* name) {
    if (!r->p) return fail(HQ_ERR_INVALID_ARG, "null %s pages", name);
    if (!aligned16(r->p)) return fail(HQ_ERR_MISALIGNED, "%s pages must be 16-byte aligned", name);
    if (r->stride_page < 0 || r->stride_token < 0 || r->stride_head < 0 || r->stride_page % 8 || r->stride_token % 8 ||
        r->stride_head % 8)
        return fail(HQ_ERR_MISALIGNED, "%s pages: strides must be non-negative multiples of 8 elements", name);
    return HQ_OK;
}

hq_status check_cache(const hq_kv_view* c, int n_seqs) {
    if (!c) return fail(HQ_ERR_INVALID_ARG, "null cache");
    hq_status st;
    if ((st = check_pages(&c->k, "key")) != HQ_OK || (st = check_pages(&c->v, "value")) != HQ_OK) return st;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "page_size=%d must be a power of two from 16 to 256", c->page_size);
    if (c->num_pages <= 0 || c->max_pages < 0 || c->table_stride < 0) return fail(HQ_ERR_INVALID_ARG, "bad cache size");
    if ((long long)c->max_pages * c->page_size > 0x7fffffffLL || (long long)c->num_pages * c->page_size > 0x7fffffffLL)
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "more than 2^31 - 1 keys");
    if (n_seqs > 0 && (!c->kv_lens || (c->max_pages > 0 && !c->page_table)))
        return fail(HQ_ERR_INVALID_ARG, "null page_table or kv_lens");
    return HQ_OK;
}

void fill_shape(AttnArgs& a, const hq_attn_shape* s, const hq_rows* q, const hq_rows* out, float* lse) {
    a.dtype = (DType)s->dtype;
    a.T = s->n_tokens;
    a.B = s->n_seqs;
    a.max_q = s->max_q_len;
    a.Hq = s->n_heads;
    a.Hk = s->n_kv_heads;
    a.G = a.Hq / a.Hk;
    a.D = s->head_dim;
    a.scale = s->scale;
    a.q = q->p;
    a.q_st = q->stride_token;
    a.q_sh = q->stride_head;
    a.o = out->p;
    a.o_st = out->stride_token;
    a.o_sh = out->stride_head;
    a.lse = lse;
}

// 0 for what the call refuses anyway.
size_t workspace_bytes(const hq_attn_shape* s, bool paged, int max_kv, int prefix_len) {
    if (check_shape(s, true) != HQ_OK || s->n_tokens == 0 || s->n_seqs == 0 || max_kv < 0 || prefix_len < 0) return 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
    return attn_plan(s->n_tokens, s->n_seqs, s->max_q_len, s->n_heads, s->n_kv_heads, s->head_dim, paged, max_kv, prefix_len,
                     device_info(dev).sm_count)
        .bytes;
}

hq_status check_workspace(const void* ws, size_t bytes, size_t need) {
    if (need && !ws) return fail(HQ_ERR_INVALID_ARG, "null workspace (%zu bytes required)", need);
    if (!aligned16(ws)) return fail(HQ_ERR_MISALIGNED, "workspace must be 16-byte aligned");
    if (bytes < need) return fail(HQ_ERR_WORKSPACE_TOO_SMALL, "workspace %zu bytes < required %zu", bytes, need);
    return HQ_OK;
}

// Queries, keys and values are read through tensor maps: positive strides below 2^40 bytes.
hq_status check_map(long long stride, long long count, const char* what) {
    if (count > 1 && (stride <= 0 || stride >= (1LL << 39)))
        return fail(HQ_ERR_UNSUPPORTED_SHAPE, "%s stride %lld", what, stride);
    return HQ_OK;
}

}  // namespace

extern "C" {

HQ_API size_t hq_attn_prompt_workspace_size(const hq_attn_shape* shape) {
    return shape ? workspace_bytes(shape, false, shape->max_q_len, 0) : 0;
}

HQ_API size_t hq_attn_paged_workspace_size(const hq_attn_shape* shape, int max_kv_len, int prefix_len) {
    return shape ? workspace_bytes(shape, true, max_kv_len, prefix_len) : 0;
}

HQ_API hq_status hq_attn_prompt(const hq_attn_shape* shape, const hq_rows* q, const hq_rows* k, const hq_rows* v,
                                const int32_t* cu_seqlens, int causal, const hq_rows* out, float* lse, void* workspace,
                                size_t ws_bytes, hq_stream_t stream) {
    hq_status st = check_shape(shape, true);
    if (st != HQ_OK) return st;
    if (shape->n_tokens == 0 || shape->n_seqs == 0) return HQ_OK;
    if ((st = check_rows(q, "q")) != HQ_OK || (st = check_rows(k, "k")) != HQ_OK || (st = check_rows(v, "v")) != HQ_OK ||
        (st = check_rows(out, "out")) != HQ_OK)
        return st;
    if (!cu_seqlens) return fail(HQ_ERR_INVALID_ARG, "null cu_seqlens");
    for (const hq_rows* r : {q, k, v})
        if ((st = check_map(r->stride_token, shape->n_tokens, "token")) != HQ_OK ||
            (st = check_map(r->stride_head, r == q ? shape->n_heads : shape->n_kv_heads, "head")) != HQ_OK)
            return st;
    if ((st = check_workspace(workspace, ws_bytes, hq_attn_prompt_workspace_size(shape))) != HQ_OK) return st;
    int dev = 0;
    if ((st = check_device(&dev)) != HQ_OK) return st;
    AttnArgs a{};
    fill_shape(a, shape, q, out, lse);
    a.causal = causal != 0;
    a.cu_q = cu_seqlens;
    a.k = k->p;
    a.k_st = k->stride_token;
    a.k_sh = k->stride_head;
    a.v = v->p;
    a.v_st = v->stride_token;
    a.v_sh = v->stride_head;
    a.max_kv = a.max_q;
    a.err = device_error_word(dev);
    a.ws = static_cast<uint8_t*>(workspace);
    a.dev = dev;
    a.sm_count = device_info(dev).sm_count;
    a.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = launch_attn(a);
    return e == cudaSuccess ? HQ_OK : cuda_fail(e, "attention launch");
}

HQ_API hq_status hq_attn_paged(const hq_attn_shape* shape, const hq_rows* q, const hq_kv_view* cache,
                               const int32_t* cu_q, int max_kv_len, const int32_t* prefix_table, int prefix_len,
                               const hq_rows* out, float* lse, void* workspace, size_t ws_bytes, hq_stream_t stream) {
    hq_status st = check_shape(shape, true);
    if (st != HQ_OK) return st;
    if (shape->n_tokens == 0 || shape->n_seqs == 0) return HQ_OK;
    if ((st = check_rows(q, "q")) != HQ_OK || (st = check_rows(out, "out")) != HQ_OK ||
        (st = check_cache(cache, shape->n_seqs)) != HQ_OK)
        return st;
    if (max_kv_len < 0 || prefix_len < 0) return fail(HQ_ERR_INVALID_ARG, "negative length");
    if (prefix_len > 0 && !prefix_table) return fail(HQ_ERR_INVALID_ARG, "null prefix_table");
    if (!cu_q && shape->n_tokens < shape->n_seqs)
        return fail(HQ_ERR_INVALID_ARG, "%d sequences of one row in %d rows", shape->n_seqs, shape->n_tokens);
    if ((st = check_map(q->stride_token, shape->n_tokens, "token")) != HQ_OK ||
        (st = check_map(q->stride_head, shape->n_heads, "head")) != HQ_OK)
        return st;
    for (const hq_pages* r : {&cache->k, &cache->v})
        if ((st = check_map(r->stride_token, cache->page_size, "token")) != HQ_OK ||
            (st = check_map(r->stride_head, shape->n_kv_heads, "head")) != HQ_OK ||
            (st = check_map(r->stride_page, cache->num_pages, "page")) != HQ_OK)
            return st;
    if ((st = check_workspace(workspace, ws_bytes, hq_attn_paged_workspace_size(shape, max_kv_len, prefix_len))) != HQ_OK)
        return st;
    int dev = 0;
    if ((st = check_device(&dev)) != HQ_OK) return st;
    AttnArgs a{};
    fill_shape(a, shape, q, out, lse);
    a.causal = 1;
    a.cu_q = cu_q;
    a.k = cache->k.p;
    a.k_sp = cache->k.stride_page;
    a.k_st = cache->k.stride_token;
    a.k_sh = cache->k.stride_head;
    a.v = cache->v.p;
    a.v_sp = cache->v.stride_page;
    a.v_st = cache->v.stride_token;
    a.v_sh = cache->v.stride_head;
    a.page_size = cache->page_size;
    a.num_pages = cache->num_pages;
    a.max_pages = cache->max_pages;
    a.table = cache->page_table;
    a.table_stride = cache->table_stride;
    a.kv_lens = cache->kv_lens;
    a.max_kv = max_kv_len;
    a.prefix_table = prefix_table;
    a.prefix_len = prefix_len;
    a.err = device_error_word(dev);
    a.ws = static_cast<uint8_t*>(workspace);
    a.dev = dev;
    a.sm_count = device_info(dev).sm_count;
    a.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = launch_attn(a);
    return e == cudaSuccess ? HQ_OK : cuda_fail(e, "attention launch");
}

HQ_API hq_status hq_kv_append(const hq_attn_shape* shape, const hq_rows* k, const hq_rows* v, const hq_kv_view* cache,
                              const int32_t* cu_q, hq_stream_t stream) {
    hq_status st = check_shape(shape, false);
    if (st != HQ_OK) return st;
    if (shape->n_tokens == 0 || shape->n_seqs == 0) return HQ_OK;
    if ((st = check_rows(k, "k")) != HQ_OK || (st = check_rows(v, "v")) != HQ_OK ||
        (st = check_cache(cache, shape->n_seqs)) != HQ_OK)
        return st;
    if (!cu_q && shape->n_tokens < shape->n_seqs)
        return fail(HQ_ERR_INVALID_ARG, "%d sequences of one row in %d rows", shape->n_seqs, shape->n_tokens);
    int dev = 0;
    if ((st = check_device(&dev)) != HQ_OK) return st;
    KvAppendArgs a{};
    a.T = shape->n_tokens;
    a.B = shape->n_seqs;
    a.Hk = shape->n_kv_heads;
    a.D = shape->head_dim;
    a.k = k->p;
    a.k_st = k->stride_token;
    a.k_sh = k->stride_head;
    a.v = v->p;
    a.v_st = v->stride_token;
    a.v_sh = v->stride_head;
    a.kp = cache->k.p;
    a.kp_sp = cache->k.stride_page;
    a.kp_st = cache->k.stride_token;
    a.kp_sh = cache->k.stride_head;
    a.vp = cache->v.p;
    a.vp_sp = cache->v.stride_page;
    a.vp_st = cache->v.stride_token;
    a.vp_sh = cache->v.stride_head;
    a.page_size = cache->page_size;
    a.num_pages = cache->num_pages;
    a.max_pages = cache->max_pages;
    a.table = cache->page_table;
    a.table_stride = cache->table_stride;
    a.kv_lens = cache->kv_lens;
    a.cu_q = cu_q;
    a.err = device_error_word(dev);
    cudaError_t e = launch_kv_append(a, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? HQ_OK : cuda_fail(e, "append launch");
}

HQ_API hq_status hq_kv_copy_pages(void* const* bases, int n_bases, size_t page_stride_bytes, size_t page_bytes,
                                  int num_pages, const hq_page_move* moves, int n_moves, hq_stream_t stream) {
    if (n_bases < 0 || n_moves < 0 || num_pages <= 0) return fail(HQ_ERR_INVALID_ARG, "bad size");
    if (n_bases == 0 || n_moves == 0) return HQ_OK;
    if (!bases || !moves) return fail(HQ_ERR_INVALID_ARG, "null pointer argument");
    if (page_bytes == 0 || page_bytes % 16 || page_stride_bytes % 16 || page_stride_bytes < page_bytes)
        return fail(HQ_ERR_MISALIGNED, "page_bytes=%zu and page_stride_bytes=%zu must be multiples of 16, the stride no less",
                    page_bytes, page_stride_bytes);
    for (int b = 0; b < n_bases; ++b) {
        if (!bases[b]) return fail(HQ_ERR_INVALID_ARG, "null page array %d", b);
        if (!aligned16(bases[b])) return fail(HQ_ERR_MISALIGNED, "page array %d must be 16-byte aligned", b);
    }
    try {
        std::vector<uint8_t> use((size_t)num_pages, 0);  // 1 read, 2 written
        for (int i = 0; i < n_moves; ++i) {
            const int s = moves[i].src, d = moves[i].dst;
            if (s < 0 || s >= num_pages || d < 0 || d >= num_pages)
                return fail(HQ_ERR_INVALID_ARG, "move %d: %d -> %d outside %d pages", i, s, d, num_pages);
            if (s == d || use[d] || use[s] == 2)
                return fail(HQ_ERR_INVALID_ARG, "move %d: %d -> %d writes a page that another move reads or writes", i, s, d);
            use[s] = 1;
            use[d] = 2;
        }
    } catch (const std::bad_alloc&) {
        return fail(HQ_ERR_OUT_OF_MEMORY, "no host memory for %d pages", num_pages);
    }
    int dev = 0;
    hq_status st = check_device(&dev);
    if (st != HQ_OK) return st;
    static_assert(sizeof(hq_page_move) == sizeof(PageMove), "same two ints");
    cudaError_t e = launch_kv_copy_pages(bases, n_bases, page_stride_bytes, page_bytes,
                                         reinterpret_cast<const PageMove*>(moves), n_moves,
                                         reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? HQ_OK : cuda_fail(e, "page copy launch");
}

}  // extern "C"
