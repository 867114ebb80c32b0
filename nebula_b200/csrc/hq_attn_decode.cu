// hq_attn_decode.cu -- attention of few rows over the paged cache: a decode step's
// single tokens (the rows of a sequence and key/value head, tokens x G, are at
// most 16), bound by reading the cache once.
//
// An item is one (sequence, key/value head); W warps work on it (8, a CTA; fewer
// where there are more items than CTAs and they are short), in units of 16 W keys.  A
// warp takes 16 keys of each unit, which lie in one page, through a ring of its own
// in shared memory (a TMA box of 16 keys each of K and V, two units of 8 KB ahead;
// nothing but its own copies to wait for): 128 KB in flight per SM, several times
// bandwidth x latency.
//   S^T = K Q^T    mma.sync m16n8k16: 16 keys x 8 rows (or 2 x 8)
//   P^T = 2^(c S - m), a running maximum m and sum per warp and row; m is moved, with O
//                  and the sum, only when a score is above it by more than 2^8, which
//                  a vote tells: lanes need not agree on each unit's maximum
//   O^T += V^T P^T mma.sync, V^T by transposing loads, P^T by an 8 x 8 transpose of the
//                  registers
// The tensor rate is no bound here, but with two warps a scheduler the instructions of
// a unit are: with the few rows as the MMA's N side there are half as many as with the
// rows as its M side, padded to 16.
// At an item's end the warps' sums are joined in shared memory.  Who takes which
// units (DecodeMode; decode_plan chooses):
//   kCluster  few items: a cluster of CTAs each, which join through distributed
//             shared memory
//   kWhole    each group of W warps every so manieth item
//   kFlat     each CTA an equal share of the line of all units, whatever the lengths:
//             items that CTAs share leave normalised fp32 partials (at most two a
//             CTA), joined by attn_join_kernel
// The CTAs work their share out from the lengths on the device, so no plan is made
// beforehand and a captured call follows them.  With a shared prefix its partials
// (tile kernel) are joined with the item's own before it is written.
// A short call is bound by fetching this code: it is kept in loops, each step in one
// place.
#include "hq_attn.cuh"
#include "hq_tmap.h"

#include <algorithm>
#include <cstring>
#include <type_traits>

namespace hq {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlice = 16;                 // keys of a warp in a unit
constexpr int kUnit = kSlice * kWarps;     // keys of a unit of a whole CTA
constexpr int kMaxRows = kDecodeRows;      // 16

template <int DP>
struct DecodeLayout {
    static constexpr int kStages = 384 / DP;            // 3 (DP 128) or 6: 24 KB a warp
    static constexpr int kBlk = DP / 64;                // 64-dim blocks of 128-byte rows
    static constexpr int kHalf = kBlk * kSlice * 128;   // K or V of a stage
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kJoin = kWarps * 8 * DP * 4;   // 8 rows of every warp
};

struct alignas(64) DecodeParams {
    CUtensorMap k_map, v_map;  // {64 dims, token, 64-dim block, head, page}: see kv_maps
    const void* q;
    long long q_st, q_sh;
    void* o;
    long long o_st, o_sh;
    float* lse;
    const int* cu_q;
    const int* table;
    long long table_stride;
    const int* kv_lens;
    int T, B, Hq, Hk, G, D;
    int page_size, page_shift, num_pages, max_pages;
    float scale_log2, inv_scale_log2;
    int whole_box;  // the maps have all dims in a box
    int only;  // no other kernel takes the sequences of more rows
    int mode, cluster;
    int group;  // W: warps of an item
    int max_rows;  // rows (tokens x G) that this kernel takes of a sequence
    // partials of items that CTAs share: two slots of 16 rows a CTA; with a prefix the
    // other items' by row in own_o, own_l [T * Hq] (kFlat)
    float *slot_o, *slot_l, *own_o, *own_l;
    const float *pre_o, *pre_l;  // the prefix's [prefix_splits][T * Hq]
    int prefix_splits, prefix_len;
    int overlap;  // launched while the kernel before it runs
    unsigned* err;
};

struct Seq {
    int first, n, len, tiles;  // rows, keys, units per head
};

// Sequence s, tiles 0 if it is not this kernel's.
__device__ __forceinline__ Seq seq_of(const int* cu_q, const int* kv_lens, int T, int G, int max_rows, int max_pages,
                                      int page_size, int unit, int s, unsigned* err) {
    Seq q{};
    if (!seq_rows(cu_q, s, T, q.first, q.n)) {
        bad_index(err);
        return q;
    }
    if (q.n <= 0 || (long long)q.n * G > max_rows) return q;
    q.len = kv_lens[s];
    if (!len_ok(q.len, max_pages, page_size)) {
        bad_index(err);
        return q;
    }
    q.tiles = max(1, (int)(((unsigned)q.len + (unsigned)unit - 1u) / (unsigned)unit));
    return q;
}

// A unit of an item.
struct Place {
    int s, h, tile;
    Seq seq;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// 8 x 8 16-bit values, a row in four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Sum of x over the block; `scratch`: kWarps values.  Two barriers.
__device__ __forceinline__ long long block_sum(long long x, long long* scratch) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
    __syncthreads();
    if (lane == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += scratch[w];
    return x;
}

template <int DP>
struct DecodeShared {
    uint64_t full[kWarps][DecodeLayout<DP>::kStages];
    Place place[kWarps][DecodeLayout<DP>::kStages];  // the unit in a stage
    float m[kWarps][kMaxRows], l[kWarps][kMaxRows];
    unsigned bad[2][DP];  // keys (bit j: key len - 16 + j) whose value in that dim is NaN | +Inf << 16, -Inf
    int any_bad, gave_up;
};

template <bool kBF16, int DP, int NT>  // NT: groups of 8 rows
__global__ void __launch_bounds__(kThreads, 1) attn_decode_kernel(const __grid_constant__ DecodeParams p) {
    using L = DecodeLayout<DP>;
    using T16 = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
    constexpr float kShift = kBF16 ? 0.f : 6.f;  // fp16: P scaled by 2^6, as is the sum
    constexpr int NS = L::kStages;

    extern __shared__ __align__(1024) uint8_t smem[];
    DecodeShared<DP>& sh = *reinterpret_cast<DecodeShared<DP>*>(smem + L::kRing + L::kJoin);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const int W = p.group, gw = warp & (W - 1), w0 = warp - gw;  // this warp in its group, the group's first
    const int unit = kSlice * W;
    const size_t rows = (size_t)p.T * p.Hq;
    pdl_launch_dependents();

    if (lane == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(&sh.full[warp][i], 1);
        fence_mbarrier_init();
        fence_async_smem();
    }
    if (tid < 2 * DP) (&sh.bad[0][0])[tid] = 0;
    if (tid == 0) sh.any_bad = sh.gave_up = 0;
    __syncthreads();

    auto seq_at = [&](int s) {
        const Seq q = seq_of(p.cu_q, p.kv_lens, p.T, p.G, p.max_rows, p.max_pages, p.page_size, unit, s, p.err);
        if (p.only && q.n > 0 && q.tiles == 0) bad_index(p.err);  // more rows than the caller's bound, or a bad length
        return q;
    };
    auto group_sync = [&] {
        if (W == 1) __syncwarp();
        else named_bar_sync(1 + w0 / W, 32 * W);
    };

    // `next` runs through the units of this warp's share; it begins before the first.
    Place next{};
    int units = 0x7fffffff;                          // in the share
    const int slots = gridDim.x * (kWarps / W);      // kWhole: groups, and the next item of this one
    int item = blockIdx.x * (kWarps / W) + w0 / W;
    if (p.mode == kCluster) {
        const int it = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
        next.s = it / p.Hk;
        next.h = it - next.s * p.Hk;
        next.seq = seq_at(next.s);
        const int a = (int)((unsigned)(next.seq.tiles * rank) / (unsigned)p.cluster);  // tiles <= 2^24, a cluster 8
        units = (int)((unsigned)(next.seq.tiles * (rank + 1)) / (unsigned)p.cluster) - a;
        next.tile = a - 1;
        if (next.seq.tiles == 0) {  // in all CTAs of the cluster
            if (p.overlap) pdl_wait();
            return;
        }
    } else if (p.mode == kFlat) {
        // ----------------------------------- this CTA's share of the line
        long long* scan = reinterpret_cast<long long*>(smem + L::kRing);
        Place* start = reinterpret_cast<Place*>(scan + kWarps);
        Seq mine{};
        long long count = 0;
#pragma unroll 1
        for (int s = tid; s < p.B; s += kThreads) {
            mine = seq_at(s);
            count += (long long)mine.tiles * p.Hk;
        }
        const long long total = block_sum(count, scan);
        const long long ctas = min((long long)gridDim.x, total);  // that have work, one unit at least
        if (blockIdx.x >= ctas) {
            if (p.overlap) pdl_wait();
            return;
        }
        const long long u0 = total * blockIdx.x / ctas;
        units = (int)(total * (blockIdx.x + 1) / ctas - u0);
        long long before = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < p.B && before <= u0; s0 += kThreads) {
            const int s = s0 + tid;
            if (p.B > kThreads) mine = s < p.B ? seq_at(s) : Seq{};
            const long long n = (long long)mine.tiles * p.Hk;
            long long incl = n;
#pragma unroll 1
            for (int d = 1; d < 32; d <<= 1) {
                const long long x = __shfl_up_sync(~0u, incl, d);
                if (lane >= d) incl += x;
            }
            __syncthreads();
            if (lane == 31) scan[warp] = incl;
            __syncthreads();
            long long lo = before + incl - n;
#pragma unroll 1
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) lo += scan[w];
                before += scan[w];
            }
            if (n > 0 && u0 >= lo && u0 < lo + n)
                *start = Place{s, (int)((u0 - lo) / mine.tiles), (int)((u0 - lo) % mine.tiles) - 1, mine};
        }
        __syncthreads();
        next = *start;
        __syncthreads();
    } else {
        item -= slots;
    }

    const uint32_t ring = smem_u32(smem) + warp * NS * L::kStage;
    float* join = reinterpret_cast<float*>(smem + L::kRing);
    // A cluster CTA's joined rows for the others: [16][DP] sums, [16] maxima and sums,
    // where the ring was (every warp is past its last unit by then).
    float* part = reinterpret_cast<float*>(smem);
    const int d = 4 * lane;  // the dims that this lane joins and writes

    // This lane's part of Q^T (row g of each group), of O^T (dims 16 i + g, + 8; rows
    // 2 t4, + 1), and rows 2 t4, + 1's maximum, sum, limit of keys, and the score above
    // which the maximum is moved.
    uint32_t qf[NT][DP / 16][2];
    float o[NT][DP / 16][4];
    float m[NT][2], l[NT][2], high[NT][2];
    int lim[NT][2], lim_min = 0, tile0 = 0;
    const int* pages = nullptr;  // of `next`
    // 16-byte chunk c of key r of a 64-dim block lies at chunk c ^ (r & 7): this lane's
    // addresses within K and V of a stage for the matrices of dims 0 .. 15
    const int kr = (lane >> 3 & 1) * 8 + (lane & 7), vr = (lane >> 4) * 8 + (lane & 7);
    const uint32_t ka = ring + kr * 128 + (((lane >> 4) ^ (kr & 7)) << 4);
    const uint32_t va = ring + L::kHalf + vr * 128 + (((lane >> 3 & 1) ^ (vr & 7)) << 4);
    bool first_seg = true, fresh = true, waited = !p.overlap, have = false, starts = false;
    Place at{};
    int page = 0, loaded = 0, load_st = 0, work_st = 0;
    uint32_t phase = 0;
    // Step u works on the warp's unit u, requests unit u + NS - 1 and finds the one after
    // it.  A CTA of a cluster may have no unit; it takes one empty step.
#pragma unroll 1
    for (int u = -NS;; ++u) {
        if (have) {
            // This warp's 16 keys of `next`: whole, their page has them.
            const int key = next.tile * unit + gw * kSlice;
            if (lane == 0) {
                if (starts) sh.place[warp][load_st] = next;
                if (key < next.seq.len) {
                    if (!page_ok(page, p.num_pages)) {
                        bad_index(p.err);
                        page = p.num_pages;  // out of range: the boxes read zeros
                    }
                    uint64_t* bar = &sh.full[warp][load_st];
                    uint8_t* dst = smem + (warp * NS + load_st) * L::kStage;
                    const int slot = key & (p.page_size - 1);
                    mbar_arrive_expect_tx(bar, L::kStage);
                    if (p.whole_box) {
                        tma_load_5d(dst, &p.k_map, 0, slot, 0, next.h, page, bar);
                        tma_load_5d(dst + L::kHalf, &p.v_map, 0, slot, 0, next.h, page, bar);
                    } else {
#pragma unroll 1
                        for (int b = 0; b < L::kBlk; ++b) {
                            tma_load_4d(dst + b * kSlice * 128, &p.k_map, 64 * b, slot, next.h, page, bar);
                            tma_load_4d(dst + L::kHalf + b * kSlice * 128, &p.v_map, 64 * b, slot, next.h, page, bar);
                        }
                    }
                }
            }
            load_st = load_st + 1 == NS ? 0 : load_st + 1;
            ++loaded;
        }
        have = false;
        if (loaded < units && next.s < p.B) {
            bool found = ++next.tile < next.seq.tiles;
            if (!found) {
                next.tile = 0;
#pragma unroll 1
                while (true) {  // the next item with work
                    if (p.mode == kWhole) {
                        item += slots;
                        next.s = item / p.Hk;
                        next.h = item - next.s * p.Hk;
                    } else if (++next.h == p.Hk) {
                        next.h = 0;
                        ++next.s;
                    }
                    if (next.s >= p.B) break;
                    if (p.mode == kWhole || next.h == 0) next.seq = seq_at(next.s);
                    if (next.seq.tiles > 0) {
                        found = true;
                        break;
                    }
                    next.h = p.Hk - 1;  // none of this sequence's
                }
            }
            have = found;
            starts = next.tile == 0 || loaded == 0;
            const int key = next.tile * unit + gw * kSlice;
            if (starts) pages = p.table + next.s * p.table_stride;
            if (found && key < next.seq.len) page = __ldg(pages + (key >> p.page_shift));
        }
        if (u < 0) continue;
        const bool work = u < loaded;
        if (!work && (p.mode != kCluster || u > 0)) break;
        if (!fresh) {
            ++at.tile;
        } else if (work) {
            __syncwarp();
            at = sh.place[warp][work_st];
        } else {
            at = next;
        }
        const int R = at.seq.n * p.G;
        if (fresh) {  // a new item: its rows of Q
            fresh = false;
            tile0 = at.tile;
            lim_min = keys_seen(at.seq.len, at.seq.n, 0, 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = 8 * nt + g;
                const bool live = r < R;
                const int tok = live ? r / p.G : 0, hd = at.h * p.G + (live ? r - tok * p.G : 0);
                const T16* q = static_cast<const T16*>(p.q) + (size_t)(at.seq.first + tok) * p.q_st + (size_t)hd * p.q_sh;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int dim = 16 * k + 8 * x + 2 * t4;
                        qf[nt][k][x] = live && dim < p.D ? __ldg(reinterpret_cast<const uint32_t*>(q + dim)) : 0u;
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 8 * nt + 2 * t4 + e;
                    lim[nt][e] = keys_seen(at.seq.len, at.seq.n, min(row, R - 1) / p.G, 1);
                    m[nt][e] = high[nt][e] = -INFINITY;
                    l[nt][e] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
            }
        }
        const int key0 = at.tile * unit + gw * kSlice;
        if (work && key0 < at.seq.len) {
            wait_bar(&sh.full[warp][work_st], phase >> work_st & 1u, &sh.gave_up, p.err);
            phase ^= 1u << work_st;
            __syncwarp();
            const uint32_t st = work_st * L::kStage, vst = ring + st + L::kHalf;
            const bool masked = key0 + kSlice > lim_min;
            if (masked) {
                // Rows of V behind the last key are zeroed: 0 x NaN would reach the sum.
                // So would values that only some rows see: those are taken out, and put
                // back into the rows that see them at the end.  Only the last n <= 16
                // keys can be such.
                const int lo = max(0, lim_min - key0), hi = min(kSlice, at.seq.len - key0);
#pragma unroll 1
                for (int x = lo * (DP / 8) + lane; x < kSlice * (DP / 8); x += 32) {
                    const int r = x / (DP / 8), c = x % (DP / 8);
                    const uint32_t a = vst + (c >> 3) * kSlice * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    uint4 v4 = r < hi ? lds128(a) : make_uint4(0u, 0u, 0u, 0u);
                    if (r < hi && !not_finite<kBF16>(v4)) continue;
                    if (r < hi) {
                        uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
                        constexpr uint32_t kExp = kBF16 ? 0x7F80u : 0x7C00u;
#pragma unroll 1
                        for (int e = 0; e < 8; ++e) {
                            const int i = e >> 1, sft = 16 * (e & 1);
                            const uint32_t word = i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3], h = word >> sft & 0xFFFFu;
                            if ((h & kExp) != kExp) continue;
                            const unsigned bit = 1u << (key0 + r - (at.seq.len - 16));
                            const bool nan = (h & 0x7FFFu) != kExp, minus = h & 0x8000u;
                            atomicOr(&sh.bad[!nan && minus][c * 8 + e], !nan && !minus ? bit << 16 : bit);
                            const uint32_t keep = ~(0xFFFFu << sft);
                            w[0] &= i == 0 ? keep : ~0u;
                            w[1] &= i == 1 ? keep : ~0u;
                            w[2] &= i == 2 ? keep : ~0u;
                            w[3] &= i == 3 ? keep : ~0u;
                        }
                        v4 = make_uint4(w[0], w[1], w[2], w[3]);
                        sh.any_bad = 1;
                    }
                    sts128(a, v4);
                }
                fence_async_smem();  // before the next request fills the stage
                __syncwarp();
            }
            float s[NT][4] = {}, s2[NT][4] = {};  // even and odd steps: two chains
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t a[4];
                ldsm4(((ka + st) ^ ((2 * k & 7) << 4)) + (k >> 2) * kSlice * 128, a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816<kBF16>(k & 1 ? s2[nt] : s[nt], a, qf[nt][k][0], qf[nt][k][1]);
            }
            bool above = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nt][e] += s2[nt][e];
                    if (masked && key0 + g + 8 * (e >> 1) >= lim[nt][e & 1]) s[nt][e] = -INFINITY;
                    above = above || s[nt][e] > high[nt][e & 1];
                }
            if (__any_sync(~0u, above)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(s[nt][e], s[nt][e + 2]);
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 16)) * p.scale_log2;
                        x = fmaxf(x, m[nt][e]);
                        const float f = ex2(m[nt][e] - (x == -INFINITY ? 0.f : x));
                        m[nt][e] = x;
                        high[nt][e] = (x + 8.f) * p.inv_scale_log2;
                        l[nt][e] *= f;
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i) {
                            o[nt][i][e] *= f;
                            o[nt][i][e + 2] *= f;
                        }
                    }
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float sub = m[nt][e & 1] == -INFINITY ? 0.f : kShift - m[nt][e & 1];
                    w[e] = ex2(fmaf(s[nt][e], p.scale_log2, sub));
                    l[nt][e & 1] += w[e];
                }
                // rounded to V's type for the MMA, as in the tile kernel; l has them in fp32
                pf[nt][0] = transpose8x8(pack2<kBF16>(w[0], w[1]));
                pf[nt][1] = transpose8x8(pack2<kBF16>(w[2], w[3]));
            }
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                uint32_t a[4];
                ldsm4_t(((va + st) ^ ((2 * i & 7) << 4)) + (i >> 2) * kSlice * 128, a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816<kBF16>(o[nt][i], a, pf[nt][0], pf[nt][1]);
            }
        }
        __syncwarp();  // the stage is read; the next request may fill it
        work_st = work_st + 1 == NS ? 0 : work_st + 1;
        if (at.tile + 1 < at.seq.tiles && u + 1 < units) continue;

        // ------------------------------------------------- the item's end
        const bool whole = p.mode != kFlat || (tile0 == 0 && at.tile + 1 == at.seq.tiles);
        if (p.prefix_splits && p.mode != kFlat && !waited) {  // the prefix's partials are complete
            pdl_wait();
            waited = true;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[nt][e];
                x += __shfl_xor_sync(~0u, x, 4);
                x += __shfl_xor_sync(~0u, x, 8);
                x += __shfl_xor_sync(~0u, x, 16);
                if (g == 0) {
                    sh.m[warp][8 * nt + 2 * t4 + e] = m[nt][e];
                    sh.l[warp][8 * nt + 2 * t4 + e] = x;
                }
            }
        // Rows 8 pass .. 8 pass + 7 of the group's warps are joined, one warp a row, four
        // dims a lane; in a cluster then the CTAs' joined rows.
        const int levels = p.mode == kCluster ? 2 : 1;
        int taken_out = 0;  // this item's any_bad
#pragma unroll 1
        for (int pass = 0; pass < (R > 8 ? 2 : 1) + levels - 1; ++pass) {
            const bool across = p.mode == kCluster && pass == (R > 8 ? 2 : 1);  // the CTAs of a cluster
            int r = 8 * pass + gw, step = W, end = min(R, 8 * pass + 8), sources = W;
            if (across) {
                cluster_sync();
                r = (int)cluster_ctarank() * kWarps + warp;
                step = p.cluster * kWarps;
                end = R;
                sources = p.cluster;
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 2 * t4 + e, flip = 8 * row & (DP - 1);  // dim d of row r at d ^ 8 r: the four rows of a store in two halves of the banks
                    float* to = join + (warp * 8 + row) * DP;
                    if (row + 8 * pass >= R) continue;
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        to[(16 * i + g) ^ flip] = NT > 1 && pass ? o[NT - 1][i][e] : o[0][i][e];
                        to[(16 * i + g + 8) ^ flip] = NT > 1 && pass ? o[NT - 1][i][e + 2] : o[0][i][e + 2];
                    }
                }
                group_sync();
            }
#pragma unroll 1
            for (; r < end; r += step) {
                const int tok = r / p.G, hd = at.h * p.G + r - tok * p.G;
                const int see = keys_seen(at.seq.len, at.seq.n, tok, 1);
                const size_t row = (size_t)(at.seq.first + tok) * p.Hq + hd;
                // source `lane`: its maximum and sum; all their maximum and sum
                Row x{};
                float mq = -INFINITY, lq = 0.f;
                if (lane < sources) {
                    if (across) {
                        const uint32_t ml = mapa_shared(smem_u32(part + kMaxRows * DP + r), lane);
                        mq = ld_dsmem_f1(ml);
                        lq = ld_dsmem_f1(ml + kMaxRows * 4);
                    } else {
                        mq = sh.m[w0 + lane][r];
                        lq = sh.l[w0 + lane][r];
                    }
                }
                x.top = warp_max(mq);
                const float f = ex2(mq - (x.top == -INFINITY ? 0.f : x.top));
                x.sum = warp_sum(f * lq);
#pragma unroll 2
                for (int q = 0; q < sources; ++q) {
                    const float fq = __shfl_sync(~0u, f, q);
                    if (d >= DP) continue;
                    const float4 y = across ? ld_dsmem_f4(mapa_shared(smem_u32(part + r * DP + d), q))
                                            : *reinterpret_cast<const float4*>(join + ((w0 + q) * 8 + (r & 7)) * DP +
                                                                               (d ^ (8 * (r & 7) & (DP - 1))));
                    x.acc[0] += fq * y.x;
                    x.acc[1] += fq * y.y;
                    x.acc[2] += fq * y.z;
                    x.acc[3] += fq * y.w;
                }
                if (!across && sh.any_bad && d < DP) {
                    const int vis = see - (at.seq.len - 16);  // of the last 16 keys, the first `vis` are seen
                    const unsigned mask = vis >= 16 ? 0xFFFFu : vis > 0 ? (1u << vis) - 1u : 0u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned b0 = sh.bad[0][d + e], b1 = sh.bad[1][d + e];
                        if ((b0 >> 16) & mask) x.acc[e] += INFINITY;
                        if (b1 & mask) x.acc[e] -= INFINITY;
                        if (b0 & mask) x.acc[e] = NAN;
                    }
                }
                if (p.mode == kCluster && !across) {
                    if (d < DP) *reinterpret_cast<float4*>(part + r * DP + d) = make_float4(x.acc[0], x.acc[1], x.acc[2], x.acc[3]);
                    if (lane == 0) {
                        part[kMaxRows * DP + r] = x.top;
                        part[kMaxRows * DP + kMaxRows + r] = x.sum;
                    }
                    continue;
                }
                const bool out = whole && !p.own_o;
                x.top -= kShift;
                if (out && p.prefix_splits)
                    join_parts(x, p.prefix_splits, p.pre_o, p.pre_l, p.D, d, [&](int i) { return i * rows + row; });
                // no key: zeros; scores that are all -inf: NaN, or left to the join
                const float l2 = finish_row(x, out && sees_any(see, p.prefix_len));
                if (out) {
                    if (d < p.D)
                        *reinterpret_cast<uint2*>(static_cast<T16*>(p.o) + (size_t)(at.seq.first + tok) * p.o_st +
                                                  (size_t)hd * p.o_sh + d) =
                            make_uint2(pack2<kBF16>(x.acc[0], x.acc[1]), pack2<kBF16>(x.acc[2], x.acc[3]));
                    if (lane == 0 && p.lse) p.lse[row] = l2 * 0.693147180559945309417f;
                } else {
                    const size_t slot = (size_t)(2 * blockIdx.x + (first_seg ? 0 : 1)) * kMaxRows + r;
                    float* dst = whole ? p.own_o + row * p.D : p.slot_o + slot * p.D;
                    if (d < p.D) *reinterpret_cast<float4*>(dst + d) = make_float4(x.acc[0], x.acc[1], x.acc[2], x.acc[3]);
                    if (lane == 0) (whole ? p.own_l[row] : p.slot_l[slot]) = l2;
                }
            }
            // All warps have set it before the first barrier of this item's, and the next item's
            // first cannot set it before all are past the last one: read between the two, it is
            // the same in all threads.
            taken_out = sh.any_bad;
            if (across) cluster_sync();  // the others' rows have been read
            else group_sync();
        }
        if (p.mode != kCluster && taken_out) {  // W = 8: groups of fewer warps take nothing out
            __syncthreads();
            if (tid < 2 * DP) (&sh.bad[0][0])[tid] = 0;
            if (tid == 0) sh.any_bad = 0;
            __syncthreads();
        }
        first_seg = false;
        fresh = true;
    }
    if (sh.gave_up) {  // copies still in flight land before the CTA exits
        for (int i = 0; i < NS; ++i) mbar_wait(&sh.full[warp][i], phase >> i & 1u, p.err);
    }
    if (!waited) pdl_wait();  // what waits for this kernel waits for the one before it, too
}

// kFlat: joins the partials of every item that more than one CTA worked on, and with
// a shared prefix of every one, with the prefix's.  One block an item, one warp a row.
struct JoinParams {
    const float *slot_o, *slot_l, *own_o, *own_l;
    const float *pre_o, *pre_l;  // [prefix_splits][T * Hq]
    void* o;
    long long o_st, o_sh;
    float* lse;
    const int* cu_q;
    const int* kv_lens;
    int T, B, Hq, Hk, G, D;
    int page_size, max_pages;
    int max_rows, ctas, prefix_splits, prefix_len;
};

template <bool kBF16>
__global__ void __launch_bounds__(kThreads) attn_join_kernel(const JoinParams p) {
    __shared__ long long scan[kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int s = blockIdx.x, hk = blockIdx.y;
    pdl_wait();
    auto seq_at = [&](int x) {
        return seq_of(p.cu_q, p.kv_lens, p.T, p.G, p.max_rows, p.max_pages, p.page_size, kUnit, x, nullptr);
    };
    const Seq me = seq_at(s);
    if (me.tiles == 0) return;
    long long before = 0, total = 0;
#pragma unroll 1
    for (int x = tid; x < p.B; x += kThreads) {
        const long long n = (long long)seq_at(x).tiles * p.Hk;
        total += n;
        if (x < s) before += n;
    }
    total = block_sum(total, scan);
    before = block_sum(before, scan);
    // CTA c has the units [total c / ctas, total (c + 1) / ctas)
    const long long ctas = min((long long)p.ctas, total);
    const long long ub = before + (long long)hk * me.tiles, ue = ub + me.tiles;
    const int c0 = (int)(((ub + 1) * ctas - 1) / total), c1 = (int)((ue * ctas - 1) / total);
    if (c0 == c1 && !p.prefix_splits) return;
    const int R = me.n * p.G, d = 4 * lane;
    const size_t rows = (size_t)p.T * p.Hq;
    const bool mid = ub != total * c0 / ctas;  // CTA c0 begins with another item
#pragma unroll 1
    for (int r = warp; r < R; r += kWarps) {
        const int tok = r / p.G, hd = hk * p.G + r - tok * p.G;
        const size_t row = (size_t)(me.first + tok) * p.Hq + hd;
        Row x{};
        x.top = -INFINITY;
#pragma unroll 1
        for (int k = 0; k < (p.prefix_splits ? 2 : 1); ++k) {
            const bool whole = c0 == c1;
            const float* po = k ? p.pre_o : whole ? p.own_o : p.slot_o;
            const float* pl = k ? p.pre_l : whole ? p.own_l : p.slot_l;
            join_parts(x, k ? p.prefix_splits : c1 - c0 + 1, po, pl, p.D, d, [&](int i) {
                return k ? i * rows + row : whole ? row : (size_t)(2 * (c0 + i) + (i == 0 && mid ? 1 : 0)) * kMaxRows + r;
            });
        }
        const float l2 = finish_row(x, sees_any(keys_seen(me.len, me.n, tok, 1), p.prefix_len));
        if (d < p.D)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + (size_t)(me.first + tok) * p.o_st + (size_t)hd * p.o_sh +
                                      d) = make_uint2(pack2<kBF16>(x.acc[0], x.acc[1]), pack2<kBF16>(x.acc[2], x.acc[3]));
        if (p.lse && lane == 0) p.lse[row] = l2 * 0.693147180559945309417f;
    }
}

template <bool kBF16, int DP, int NT>
cudaError_t launch_one(const DecodeParams& p, int ctas, int dev, cudaStream_t s) {
    constexpr int kSmem = DecodeLayout<DP>::kRing + DecodeLayout<DP>::kJoin + (int)sizeof(DecodeShared<DP>);
    auto fn = attn_decode_kernel<kBF16, DP, NT>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(fn), dev, kSmem);
    if (e != cudaSuccess) return e;
    static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (p.cluster > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)p.cluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    if (p.overlap) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, fn, p);
}

template <int NT>
cudaError_t launch_any(const AttnArgs& a, const DecodeParams& p, int ctas) {
    if (a.D <= 64)
        return a.dtype == DType::BF16 ? launch_one<true, 64, NT>(p, ctas, a.dev, a.stream)
                                      : launch_one<false, 64, NT>(p, ctas, a.dev, a.stream);
    return a.dtype == DType::BF16 ? launch_one<true, 128, NT>(p, ctas, a.dev, a.stream)
                                  : launch_one<false, 128, NT>(p, ctas, a.dev, a.stream);
}

}  // namespace

DecodePlan decode_plan(int B, int Hk, int max_q, int max_kv, int sms) {
    const long long items = (long long)B * Hk;
    const int last = std::max(1, max_kv) - 1;  // the last key; max_kv may be the largest int
    const int tiles = 1 + last / kUnit;
    DecodePlan pl{};
    pl.cluster = 1;
    pl.group = kWarps;
    // A cluster per item while they fill no more than the SMs and no CTA has more than
    // 16 units (2048 keys, 1 MB): beyond, a share of every SM is faster in spite of the
    // join's launch.  One stream over 8 key/value heads of 128, in clusters / as whole
    // items / in shares: 777 keys 8.9 / 12.0 / 10.6 us, 2000 keys 10.0 / 20.0 / 11.5, 16000
    // keys 24.1 / 128 / 24.6, 24000 keys 31.9 / 184 / 30.4.
    int cs = 1;
    while (cs < 8 && items * cs * 2 <= sms && cs < tiles) cs *= 2;
    if (cs > 1 && tiles <= 16 * cs) {
        pl.mode = kCluster;
        pl.cluster = cs;
        pl.ctas = (int)items * cs;
        return pl;
    }
    // Whole items, with so many warps each that one round takes all items if it can (64
    // streams of 100 keys: 11.3 us with 2 warps an item, 19.7 with 8), while no group has
    // more units than the shares' own costs and the join's launch are worth; smaller
    // groups, several a CTA, even out among themselves.  Streams of a tenth to all of the
    // longest, whole items / shares: 16 up to 3500 keys 36.9 / 41.5 us, up to 6000 keys 55.9 /
    // 51.7; 64 up to 1000 keys 39.4 / 56.7, up to 2000 keys 69.1 / 74.9.  (Groups of fewer than
    // 8 warps have no room for values that only some of a sequence's rows see: one row
    // each.)
    int W = kWarps;
    while (W > 1 && max_q == 1 && items * W > (long long)sms * kWarps) W /= 2;
    const long long slots = (long long)sms * (kWarps / W), rounds = (items + slots - 1) / slots;
    if (rounds * (1 + last / (kSlice * W)) <= (W == kWarps ? 40 : 64)) {
        pl.mode = kWhole;
        pl.group = W;
        pl.ctas = (int)std::min<long long>(sms, (items + kWarps / W - 1) / (kWarps / W));
        return pl;
    }
    pl.mode = kFlat;
    pl.ctas = (int)std::min<long long>(sms, items * tiles);
    return pl;
}

cudaError_t launch_attn_decode(const AttnArgs& a, const DecodeParts& parts) {
    DecodeParams p;
    memset(&p, 0, sizeof p);
    p.whole_box = a.D == 128;
    cudaError_t e = p.whole_box ? kv_maps_128(a, kSlice, &p.k_map, &p.v_map) : kv_maps(a, kSlice, &p.k_map, &p.v_map);
    if (e != cudaSuccess) return e;
    p.q = a.q;
    p.q_st = a.q_st;
    p.q_sh = a.q_sh;
    p.o = a.o;
    p.o_st = a.o_st;
    p.o_sh = a.o_sh;
    p.lse = a.lse;
    p.cu_q = a.cu_q;
    p.table = a.table;
    p.table_stride = a.table_stride;
    p.kv_lens = a.kv_lens;
    p.T = a.T;
    p.B = a.B;
    p.Hq = a.Hq;
    p.Hk = a.Hk;
    p.G = a.G;
    p.D = a.D;
    p.page_size = a.page_size;
    while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
    p.num_pages = a.num_pages;
    p.max_pages = a.max_pages;
    p.scale_log2 = a.scale * 1.44269504088896340736f;
    p.inv_scale_log2 = 1.f / p.scale_log2;
    p.only = parts.only;
    p.mode = parts.plan.mode;
    p.cluster = parts.plan.cluster;
    p.group = parts.plan.group;
    p.max_rows = parts.rows;
    p.slot_o = parts.slot_o;
    p.slot_l = parts.slot_l;
    p.own_o = parts.own_o;
    p.own_l = parts.own_l;
    p.pre_o = parts.pre_o;
    p.pre_l = parts.pre_l;
    p.prefix_splits = parts.prefix_splits;
    p.prefix_len = a.prefix_len;
    p.overlap = parts.overlap;
    p.err = a.err;
    return parts.rows > 8 ? launch_any<2>(a, p, parts.plan.ctas) : launch_any<1>(a, p, parts.plan.ctas);
}

cudaError_t launch_attn_join(const AttnArgs& a, const DecodeParts& parts) {
    JoinParams j{parts.slot_o, parts.slot_l, parts.own_o, parts.own_l, parts.pre_o, parts.pre_l, a.o, a.o_st, a.o_sh, a.lse,
                 a.cu_q, a.kv_lens, a.T, a.B, a.Hq, a.Hk, a.G, a.D, a.page_size, a.max_pages, parts.rows,
                 parts.plan.ctas, parts.prefix_splits, a.prefix_len};
    auto fn = a.dtype == DType::BF16 ? attn_join_kernel<true> : attn_join_kernel<false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.B, (unsigned)a.Hk);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = a.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, j);
}

}  // namespace hq
