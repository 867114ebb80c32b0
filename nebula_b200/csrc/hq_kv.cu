// hq_kv.cu -- device calls of the paged key/value cache: a step's rows into
// their pages, and pages over other pages.  Both move bytes once: bound by HBM,
// or by the launch where there is little to move.
#include "hq_attn.cuh"

#include <algorithm>

namespace hq {

namespace {

// One block per row: its place first, then 16 bytes a thread.
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs a) {
    const int t = blockIdx.x;
    __shared__ long long s_k, s_v;
    if (threadIdx.x == 0) {
        s_k = -1;
        int s = 0, first = 0, n = 0;
        for (; s < a.B; ++s) {
            if (!seq_rows(a.cu_q, s, a.T, first, n)) bad_index(a.err);
            else if (t >= first && t < first + n) break;
        }
        if (s < a.B) {
            const int len = a.kv_lens[s], pos = len - n + (t - first);
            int page = -1;
            if (len_ok(len, a.max_pages, a.page_size) && pos >= 0)
                page = a.table[s * a.table_stride + pos / a.page_size];
            if (!page_ok(page, a.num_pages)) {
                bad_index(a.err);
            } else {
                s_k = page * a.kp_sp + (pos % a.page_size) * a.kp_st;
                s_v = page * a.vp_sp + (pos % a.page_size) * a.vp_st;
            }
        }
    }
    __syncthreads();
    if (s_k < 0) return;
    const int per_head = a.D / 8, n = a.Hk * per_head;
    for (int i = threadIdx.x; i < 2 * n; i += blockDim.x) {
        const bool is_v = i >= n;
        const int r = is_v ? i - n : i;
        const int h = r / per_head, c = (r % per_head) * 8;
        if (is_v)
            *reinterpret_cast<uint4*>((uint16_t*)a.vp + s_v + h * a.vp_sh + c) =
                *reinterpret_cast<const uint4*>((const uint16_t*)a.v + t * a.v_st + h * a.v_sh + c);
        else
            *reinterpret_cast<uint4*>((uint16_t*)a.kp + s_k + h * a.kp_sh + c) =
                *reinterpret_cast<const uint4*>((const uint16_t*)a.k + t * a.k_st + h * a.k_sh + c);
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

__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const __grid_constant__ CopyParams p) {
    const PageMove mv = p.moves[blockIdx.x];
    uint8_t* base = static_cast<uint8_t*>(p.bases[blockIdx.y]);
    const uint4* src = reinterpret_cast<const uint4*>(base + mv.src * p.stride);
    uint4* dst = reinterpret_cast<uint4*>(base + mv.dst * p.stride);
    for (size_t i = threadIdx.x; i < p.bytes / 16; i += blockDim.x) dst[i] = src[i];
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s) {
    kv_append_kernel<<<a.T, 256, 0, s>>>(a);
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
