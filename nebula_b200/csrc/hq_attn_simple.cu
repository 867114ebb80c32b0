// hq_attn_simple.cu -- attention, one warp per (row, query head).
//
// One pass over the keys with a running maximum m and sum l: for a score s,
// m' = max(m, s), o = o e^(m - m') + e^(s - m') v, l likewise; out = o / l.
// Lane l holds elements 4l .. 4l + 3 of q, o and of each key and value.
#include "hq_attn.h"
#include "hq_attn_index.h"
#include "hq_common.cuh"

namespace hq {

namespace {

__device__ __forceinline__ void bad_index(unsigned* err) {
    if (err) atomicCAS(err, 0u, (unsigned)kDevBadIndex);
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, bool have, float (&f)[4]) {
    if (!have) {
        f[0] = f[1] = f[2] = f[3] = 0.f;
        return;
    }
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f32(e[i]);
}

template <typename T>
__global__ void __launch_bounds__(128) attn_simple_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(w / a.Hq), h = (int)(w % a.Hq);
    if (t >= a.T) return;
    // the sequence of row t
    int s = 0, first = 0, n = 0;
    for (; s < a.B; ++s) {
        if (!seq_rows(a.cu_q, s, a.T, first, n)) bad_index(a.err);
        else if (t >= first && t < first + n) break;
    }
    if (s == a.B) return;
    int len = n;
    if (a.page_size) {
        len = a.kv_lens[s];
        if (!len_ok(len, a.max_pages, a.page_size)) {
            bad_index(a.err);
            return;
        }
    }
    const int seen = keys_seen(len, n, t - first, a.causal);
    const bool have = 4 * lane < a.D;
    const int hk = h / a.G;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    load4((const T*)a.q + t * a.q_st + h * a.q_sh + 4 * lane, have, q);
    const float sl = a.scale * 1.44269504088896340736f;
    for (int part = a.prefix_len ? 0 : 1; part < 2; ++part) {
        const int lim = part ? seen : a.prefix_len;
        for (int j = 0; j < lim; ++j) {
            long long ko, vo;
            if (a.page_size) {
                const int pi = j / a.page_size, slot = j % a.page_size;
                const int page = part ? a.table[s * a.table_stride + pi] : a.prefix_table[pi];
                if (!page_ok(page, a.num_pages)) {
                    if (!lane) bad_index(a.err);
                    continue;
                }
                ko = page * a.k_sp + slot * a.k_st;
                vo = page * a.v_sp + slot * a.v_st;
            } else {
                ko = (first + j) * a.k_st;
                vo = (first + j) * a.v_st;
            }
            float k[4], v[4];
            load4((const T*)a.k + ko + hk * a.k_sh + 4 * lane, have, k);
            load4((const T*)a.v + vo + hk * a.v_sh + 4 * lane, have, v);
            float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
            for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
            x *= sl;
            const float m2 = fmaxf(m, x);
            const float base = m2 == -INFINITY ? 0.f : m2;
            const float c = exp2f(m - base), p = exp2f(x - base);
            m = m2;
            l = l * c + p;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = o[i] * c + p * v[i];
        }
    }
    // scores that are all -inf have no softmax: NaN, as 0 / 0; no keys at all: 0
    const float inv = l != 0.f ? 1.f / l : (seen + a.prefix_len > 0 ? NAN : 0.f);
    if (have) {
        T* p = (T*)a.o + t * a.o_st + h * a.o_sh + 4 * lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = from_f32<T>(o[i] * inv);
    }
    if (a.lse && lane == 0)
        a.lse[(size_t)t * a.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309417f;
}

}  // namespace

cudaError_t launch_attn_simple(const AttnArgs& a) {
    const long long warps = (long long)a.T * a.Hq;
    const unsigned grid = (unsigned)((warps + 3) / 4);
    if (a.dtype == DType::F16) attn_simple_kernel<__half><<<grid, 128, 0, a.stream>>>(a);
    else attn_simple_kernel<__nv_bfloat16><<<grid, 128, 0, a.stream>>>(a);
    return cudaGetLastError();
}

}  // namespace hq
