// hq_kv.cu -- device calls of the paged key/value cache: a step's rows into
// their pages, and pages over other pages.  Both move bytes once: bound by HBM,
// or by the launch where there is little to move.
#include "hq_attn.cuh"

#include <algorithm>

namespace hq {

namespace {

// One warp a row: its keys and values are requested, 16 bytes a lane and eight
// requests at a time, before its place is looked up (three dependent loads), so the
// two latencies overlap.
// Measured (prompts of 17,408 tokens in all, 8 heads of 128, bf16: 143 MB): 25.6 us,
// 5.6 TB/s; with one block a row that looked its place up first, 37.5 us. One row of
// each of 64 sequences: 3.1 us, a launch's own time.
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs a) {
    const int lane = threadIdx.x & 31, t = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= a.T) return;
    const int n = a.Hk * (a.D / 8);  // vectors of a row of keys
    const uint16_t* src[2] = {static_cast<const uint16_t*>(a.k) + t * a.k_st, static_cast<const uint16_t*>(a.v) + t * a.v_st};
    long long to_k = -1, to_v = -1;
#pragma unroll 1
    for (int i0 = 0; i0 < 2 * n; i0 += 256) {
        uint4 x[8];
        long long off[8];  // of the vector within its row of the page
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + 32 * j + lane, kv = i >= n, r = kv ? i - n : i;
            const int h = a.per_head == 1 ? r : (int)__umulhi((unsigned)r, a.head_mul), c = (r - h * a.per_head) * 8;
            if (i < 2 * n) x[j] = ldg128_nc(src[kv] + h * (kv ? a.v_sh : a.k_sh) + c);
            off[j] = h * (kv ? a.vp_sh : a.kp_sh) + c;
        }
        if (i0 == 0) {  // the row's place
            int pos = -1, s = -1;
            for (int s0 = 0; s0 < a.B && s < 0; s0 += 32) {
                int first = 0, m = 0, p = -1;
                bool mine = false;
                if (s0 + lane < a.B) {
                    if (!seq_rows(a.cu_q, s0 + lane, a.T, first, m)) bad_index(a.err);
                    else if (t >= first && t < first + m) {
                        mine = true;
                        const int len = a.kv_lens[s0 + lane];
                        p = len_ok(len, a.max_pages, a.page_size) ? len - m + (t - first) : -1;
                    }
                }
                const unsigned hit = __ballot_sync(~0u, mine);
                if (hit) {
                    s = s0 + __ffs(hit) - 1;
                    pos = __shfl_sync(~0u, p, __ffs(hit) - 1);
                }
            }
            if (s < 0) return;  // a row of no sequence
            const int page = pos >= 0 ? a.table[s * a.table_stride + (pos >> a.page_shift)] : -1;
            if (!page_ok(page, a.num_pages)) {
                bad_index(a.err);
                return;
            }
            const int slot = pos & (a.page_size - 1);
            to_k = page * a.kp_sp + slot * a.kp_st;
            to_v = page * a.vp_sp + slot * a.vp_st;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + 32 * j + lane;
            if (i >= 2 * n) continue;
            uint16_t* dst = i >= n ? static_cast<uint16_t*>(a.vp) + to_v : static_cast<uint16_t*>(a.kp) + to_k;
            *reinterpret_cast<uint4*>(dst + off[j]) = x[j];
        }
    }
}

constexpr int kMovesPerLaunch = 256;
constexpr int kBasesPerLaunch = 64;

// The lists travel as kernel parameters: no copy to the device, and a captured
// call keeps its own.
struct CopyParams {
    void* bases[kBasesPerLaunch];
    PageMove moves[kMovesPerLaunch];
    size_t stride, bytes;
};

// One block a page and array, one 16-byte load in flight a thread. 801 pages of 64 KB in
// 16 layers' keys and values: 557 us, 6.0 TB/s. A large page alone is bound by its
// block's round trips: one of 256 KB in 4 layers 14.8 us, eight 16.7 us (2.0 TB/s), 64 of
// them 57.8 us (4.6 TB/s); one of 32 KB 5.1 us.
__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const __grid_constant__ CopyParams p) {
    const PageMove mv = p.moves[blockIdx.x];
    uint8_t* base = static_cast<uint8_t*>(p.bases[blockIdx.y]);
    const uint4* src = reinterpret_cast<const uint4*>(base + mv.src * p.stride);
    uint4* dst = reinterpret_cast<uint4*>(base + mv.dst * p.stride);
    for (size_t i = threadIdx.x; i < p.bytes / 16; i += blockDim.x) dst[i] = src[i];
}

}  // namespace

cudaError_t launch_kv_append(KvAppendArgs a, cudaStream_t s) {
    a.per_head = a.D / 8;  // at most 16, and a row has fewer than 2^20 vectors: exact
    a.head_mul = a.per_head > 1 ? (unsigned)(((1ull << 32) + a.per_head - 1) / a.per_head) : 0u;
    a.page_shift = 0;
    while ((1 << a.page_shift) < a.page_size) ++a.page_shift;
    kv_append_kernel<<<(a.T + 7) / 8, 256, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_kv_copy_pages(void* const* bases, int n_bases, size_t stride, size_t bytes, const PageMove* moves,
                                 int n_moves, cudaStream_t s) {
    CopyParams p;
    p.stride = stride;
    p.bytes = bytes;
    for (int b0 = 0; b0 < n_bases; b0 += kBasesPerLaunch) {
        const int nb = std::min(kBasesPerLaunch, n_bases - b0);
        std::copy(bases + b0, bases + b0 + nb, p.bases);
        for (int m0 = 0; m0 < n_moves; m0 += kMovesPerLaunch) {
            const int nm = std::min(kMovesPerLaunch, n_moves - m0);
            std::copy(moves + m0, moves + m0 + nm, p.moves);
            kv_copy_pages_kernel<<<dim3(nm, nb), 256, 0, s>>>(p);
            cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace hq
