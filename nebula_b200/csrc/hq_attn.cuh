// hq_attn.cuh -- device helpers that the attention and cache kernels share.
#pragma once

#include "hq_attn.h"
#include "hq_attn_index.h"
#include "hq_common.cuh"

namespace hq {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// Whether one of the eight 16-bit values of v is Inf or NaN: one step more in the
// exponent's last place then reaches the sign's.
template <bool kBF16>
__device__ __forceinline__ bool not_finite(uint4 v) {
    constexpr uint32_t kStep = kBF16 ? 0x00800080u : 0x04000400u, kAbs = 0x7FFF7FFFu;
    return (((v.x & kAbs) + kStep) | ((v.y & kAbs) + kStep) | ((v.z & kAbs) + kStep) | ((v.w & kAbs) + kStep)) & 0x80008000u;
}

__device__ __forceinline__ float ld_dsmem_f1(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// 16-byte asynchronous copy into shared memory; zeros where there is nothing to copy.
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool have) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}

// Whether the phase is over, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_u32(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
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

}  // namespace hq
