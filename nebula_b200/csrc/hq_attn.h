// hq_attn.h -- internal interface of the attention kernels.
#pragma once

#include "hq_internal.h"

namespace hq {

struct AttnArgs {
    DType dtype;
    int T, B, max_q;        // rows, sequences, bound of a sequence's rows
    int Hq, Hk, G, D;       // G = Hq / Hk
    float scale;
    int causal;             // row i of n sees keys 0 .. len - n + i, else all len
    const void* q;
    long long q_st, q_sh;   // strides in elements: per token, per head
    void* o;
    long long o_st, o_sh;
    float* lse;             // nullable, [T][Hq]
    const int* cu_q;        // nullable: row s is sequence s
    // Keys and values: pages (page_size > 0), or packed rows like q's (0).
    const void *k, *v;
    long long k_sp, k_st, k_sh, v_sp, v_st, v_sh;
    int page_size, num_pages, max_pages;
    const int* table;
    long long table_stride;
    const int* kv_lens;
    int max_kv;             // bound of kv_lens that sizes the launch
    const int* prefix_table;
    int prefix_len;         // 0: no shared prefix
    unsigned* err;
    uint8_t* ws;
    int sm_count, dev;
    cudaStream_t stream;
};

// Sequences of at most kDecodeRows rows (tokens x G) over pages are the decode
// kernel's, where it is launched; all others the tile kernel's.
constexpr int kDecodeRows = 16;

// What a call launches, and the workspace that its partial results take.
struct AttnPlan {
    bool decode, tile;
    int prefix;         // key splits of the shared prefix (0: none)
    int own;            // key splits of the tile kernel
    int ctas, whole;    // decode kernel: CTAs; no (sequence, head) is split
    size_t planes;      // partials of every (row, head): prefix, tile, decode
    size_t bytes;
};
AttnPlan attn_plan(int T, int B, int max_q, int Hq, int Hk, int D, bool paged, int max_kv, int prefix_len, int sms);
cudaError_t launch_attn(const AttnArgs& a);

// The decode kernel's partial results and those of the prefix that they join.
struct DecodeParts {
    int ctas, whole, only;
    float *slot_o, *slot_l;  // [ctas][2][16][D], [ctas][2][16]
    float *own_o, *own_l;    // [T * Hq][D], [T * Hq]; null without a prefix
    const float *pre_o, *pre_l;
    int prefix_splits;
};
int decode_ctas(int B, int Hk, int max_kv, int sms);
cudaError_t launch_attn_decode(const AttnArgs& a, const DecodeParts& parts);
cudaError_t launch_attn_join(const AttnArgs& a, const DecodeParts& parts);

struct KvAppendArgs {
    int T, B, Hk, D;
    const void *k, *v;
    long long k_st, k_sh, v_st, v_sh;  // rows
    void *kp, *vp;
    long long kp_sp, kp_st, kp_sh, vp_sp, vp_st, vp_sh;  // pages
    int page_size, num_pages, max_pages;
    const int* table;
    long long table_stride;
    const int* kv_lens;
    const int* cu_q;
    unsigned* err;
};
cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s);

struct PageMove {
    int src, dst;
};
cudaError_t launch_kv_copy_pages(void* const* bases, int n_bases, size_t stride, size_t bytes, const PageMove* moves,
                                 int n_moves, cudaStream_t s);

}  // namespace hq
