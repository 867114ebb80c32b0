// hq_attn.cuh -- device helpers that the attention and cache kernels share.
#pragma once

#include "hq_attn.h"
#include "hq_attn_index.h"
#include "hq_common.cuh"

namespace hq {

// 2^x within 2^-22 of its value, log2 within 2^-22 in all, 1 / x within 1 ulp: the error
// of a weight, far below the half step (2^-8 or 2^-11) by which it is rounded for P V.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t w;
    if (kBF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

__device__ __forceinline__ void bad_index(unsigned* err) {
    if (err) atomicCAS(err, 0u, (unsigned)kDevBadIndex);
}

// Not 0 where one of the eight 16-bit values of v is Inf or NaN: one step more in the
// exponent's last place then reaches the sign's.
template <bool kBF16>
__device__ __forceinline__ uint32_t not_finite(uint4 v) {
    constexpr uint32_t kStep = kBF16 ? 0x00800080u : 0x04000400u, kAbs = 0x7FFF7FFFu;
    return (((v.x & kAbs) + kStep) | ((v.y & kAbs) + kStep) | ((v.z & kAbs) + kStep) | ((v.w & kAbs) + kStep)) & 0x80008000u;
}

__device__ __forceinline__ float ld_dsmem_f1(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// mbar_wait (hq_common.cuh) in few instructions: kernels that wait in many places
// and run for microseconds are bound by fetching their code.  A wait of the block
// that gives up records kDevTimeout and sets *gave_up (shared memory); those that
// come after it give up at once where they would wait.
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, int* gave_up, unsigned* err) {
    unsigned long long t0 = 0;
#pragma unroll 1
    for (unsigned n = 1; !mbar_try_wait(bar, parity); ++n) {
        if (n & 63u) continue;
        if (*reinterpret_cast<volatile int*>(gave_up)) return;
        const unsigned long long t = globaltimer_ns();
        if (t0 == 0) t0 = t;
        else if (t - t0 > kWaitBudgetNs) {
            record_error(err, kDevTimeout);
            *reinterpret_cast<volatile int*>(gave_up) = 1;
            return;
        }
    }
}

__device__ __forceinline__ void tmap_prefetch(const void* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// A box of the tensor map into shared memory; its bytes count on `bar`.
__device__ __forceinline__ void tma_load_3d(void* dst, const void* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_5d(void* dst, const void* map, int c0, int c1, int c2, int c3, int c4, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

// One row's partial results on their way to the output: sums of 2^(x - top) v in
// acc (four dims d .. d + 3 of this lane) and of 2^(x - top) in sum.
struct Row {
    float acc[4], sum, top;
};

// Joins n partials to it: normalised outputs po[at(i)][D], log2 of their sums pl[at(i)].
// 32 sums at a time (a lane each), eight outputs requested at a time.
template <typename At>
__device__ __forceinline__ void join_parts(Row& x, int n, const float* po, const float* pl, int D, int d, At at) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int c = 0; c < n; c += 32) {
        const float l2 = c + lane < n ? pl[at(c + lane)] : -INFINITY;
        const float top = fmaxf(x.top, warp_max(l2));
        const float base = top == -INFINITY ? 0.f : top;
        const float f = ex2(x.top - base), w = ex2(l2 - base);
        x.top = top;
        x.sum = x.sum * f + warp_sum(w);
#pragma unroll
        for (int e = 0; e < 4; ++e) x.acc[e] *= f;
#pragma unroll 1
        for (int s = 0; s < min(32, n - c); s += 8) {
            float4 o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] = c + s + i < n && d < D ? *reinterpret_cast<const float4*>(po + at(c + s + i) * D + d)
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float ws = __shfl_sync(~0u, w, s + i);
                x.acc[0] += ws * o[i].x;
                x.acc[1] += ws * o[i].y;
                x.acc[2] += ws * o[i].z;
                x.acc[3] += ws * o[i].w;
            }
        }
    }
}

// Normalises it; log2 of its sum.  A row without any weight is 0 where it sees no key,
// and NaN (0 / 0) where its scores are all -inf.
__device__ __forceinline__ float finish_row(Row& x, bool sees) {
    const bool some = x.sum != 0.f;
    const float inv = some ? rcp(x.sum) : sees ? NAN : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) x.acc[e] = some ? x.acc[e] * inv : inv;
    return some ? x.top + lg2(x.sum) : -INFINITY;
}

}  // namespace hq
