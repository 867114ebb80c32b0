// hq_attn.h -- internal interface of the attention kernels.
#pragma once

#include "hq_internal.h"

#include <cuda.h>

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

// Sequences of at most AttnPlan::dec_rows rows (tokens x G) over pages are the decode
// kernel's, all others the tile kernel's.  Alone, the decode kernel takes up to
// kDecodeRows; beside the tile kernel up to 8, the fewest that it computes, if they
// hold a token.
constexpr int kDecodeRows = 16;

// Launches a kernel; with `overlap` it may start while the kernel before it on the
// stream still runs (programmatic dependent launch), for whose results it then waits
// itself.
template <typename P>
cudaError_t launch_overlapped(void (*fn)(P), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, bool overlap,
                              const P& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, p);
}

// Tensor maps of the keys and values, boxes of 64 dims x box_rows tokens.
cudaError_t kv_maps(const AttnArgs& a, int box_rows, CUtensorMap* k_map, CUtensorMap* v_map);
// Pages of 128 dims with the dims as two blocks of 64, both in a box: {64, token, block,
// head, page}; the boxes lie in shared memory as two of kv_maps'.
cudaError_t kv_maps_128(const AttnArgs& a, int box_rows, CUtensorMap* k_map, CUtensorMap* v_map);

// How the decode kernel's CTAs share the items, the (sequence, key/value head)s.
enum DecodeMode : int { kFlat = 0, kWhole = 1, kCluster = 2 };
struct DecodePlan {
    int mode, ctas, cluster;
    int group;  // warps of an item
};
DecodePlan decode_plan(int B, int Hk, int max_q, int max_kv, int sms);

// What a call launches, and the workspace that its partial results take.
struct AttnPlan {
    bool decode, tile;
    int prefix;          // key splits of the shared prefix (0: none)
    int own;             // key splits of the tile kernel
    int tile_blocks, tile_sms;  // its row blocks, as far as the sizes tell, and SMs
    DecodePlan dec;
    int dec_rows;
    bool join;           // partials of the decode kernel are joined by a kernel
    size_t planes;       // partials of every (row, head): prefix, tile, decode
    size_t slots;        // rows of the decode kernel's slots
    size_t bytes;
};
AttnPlan attn_plan(int T, int B, int max_q, int Hq, int Hk, int D, bool paged, int max_kv, int prefix_len, int sms);
cudaError_t launch_attn(const AttnArgs& a);

// The decode kernel's partial results and those of the prefix that they join.
struct DecodeParts {
    DecodePlan plan;
    int rows, only, overlap;
    float *slot_o, *slot_l;  // [ctas][2][16][D], [ctas][2][16]
    float *own_o, *own_l;    // [T * Hq][D], [T * Hq]: with a prefix and kFlat
    const float *pre_o, *pre_l;
    int prefix_splits;
};
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
    int per_head, page_shift;  // set by the launch: 16-byte vectors of a head, and
    unsigned head_mul;         // 2^32 / per_head rounded up
};
cudaError_t launch_kv_append(KvAppendArgs a, cudaStream_t s);

struct PageMove {
    int src, dst;
};
cudaError_t launch_kv_copy_pages(void* const* bases, int n_bases, size_t stride, size_t bytes, const PageMove* moves,
                                 int n_moves, cudaStream_t s);

}  // namespace hq
