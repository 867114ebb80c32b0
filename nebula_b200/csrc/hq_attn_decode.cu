// hq_attn_decode.cu -- attention of few rows over the paged cache: a decode step's
// single tokens (the rows of a sequence and key/value head, tokens x G, are at
// most 16), bound by reading the cache once.
//
// An item is one (sequence, key/value head); W warps work on it (8, a CTA; fewer
// where there are more items than CTAs and they are short), in units of 16 W keys.  A
// warp takes 16 keys of each unit, which lie in one page, through a ring of its own
// in shared memory (cp.async, three units of 8 KB ahead; nothing but its own copies
// to wait for): 128 KB in flight per SM, several times bandwidth x latency.
//   S = Q K^T  mma.sync m16n8k16, the 16 rows (padded) x 16 keys
//   P = 2^(c S - m), a running maximum m and sum per warp and row; m is moved, with O
//              and the sum, only when a score is above it by more than 2^8, which a
//              vote tells: lanes need not agree on each unit's maximum
//   O += P V   mma.sync, P straight from S's registers
// The tensor rate is no bound here: 16 rows x 128 dims x 2 products a key need a
// tenth of the rate that mma.sync has while 512 bytes of it arrive.
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
#include "hq_attn.cuh"

#include <algorithm>
#include <type_traits>

namespace hq {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlice = 16;                 // keys of a warp in a unit
constexpr int kUnit = kSlice * kWarps;     // keys of a unit of a whole CTA
constexpr int kMaxRows = kDecodeRows;      // 16: the MMA's M

template <int DP>
struct DecodeLayout {
    static constexpr int kStages = 384 / DP;            // 3 (DP 128) or 6: 24 KB a warp
    static constexpr int kStage = 2 * kSlice * DP * 2;  // K, then V
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kPitch = DP + 2;               // floats of a row in the join buffer
    static constexpr int kJoin = kWarps * 8 * kPitch * 4;
    static constexpr int kSmem = kRing + kJoin;
};

struct DecodeParams {
    const void* q;
    long long q_st, q_sh;
    void* o;
    long long o_st, o_sh;
    float* lse;
    const void *k, *v;
    long long k_sp, k_st, k_sh, v_sp, v_st, v_sh;
    const int* cu_q;
    const int* table;
    long long table_stride;
    const int* kv_lens;
    int T, B, Hq, Hk, G, D;
    int page_size, page_shift, num_pages, max_pages;
    float scale_log2;
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
    q.tiles = max(1, (int)((unsigned)(q.len + unit - 1) / (unsigned)unit));
    return q;
}

// A place in the line of units.
struct Place {
    int s, h, tile;
    Seq seq;
};

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

// One row's partial results on their way to the output: sums of 2^(x - top) v in
// acc (four dims d .. d + 3 of this lane) and of 2^(x - top) in sum.
struct Row {
    float acc[4], sum, top;
};

// Joins the prefix's partials of row `row` to it.
__device__ __forceinline__ void join_prefix(const float* pre_o, const float* pre_l, int splits, size_t rows, size_t row, int D,
                                            int d, Row& x) {
    const int lane = threadIdx.x & 31;
    const float l2 = lane < splits ? pre_l[lane * rows + row] : -INFINITY;  // splits <= 32
    float top = fmaxf(x.top, l2);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    const float f = ex2(x.top - base), w = ex2(l2 - base);
    x.sum *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) x.acc[e] *= f;
    // eight partials requested at a time
#pragma unroll 1
    for (int s0 = 0; s0 < splits; s0 += 8) {
        float4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = s0 + i < splits && d < D ? *reinterpret_cast<const float4*>(pre_o + ((s0 + i) * rows + row) * D + d)
                                            : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ws = __shfl_sync(~0u, w, (s0 + i) & 31);
            if (s0 + i >= splits) continue;
            x.sum += ws;
            x.acc[0] += ws * o[i].x;
            x.acc[1] += ws * o[i].y;
            x.acc[2] += ws * o[i].z;
            x.acc[3] += ws * o[i].w;
        }
    }
    x.top = top;
}

template <bool kBF16, int DP>
__global__ void __launch_bounds__(kThreads, 1) attn_decode_kernel(const __grid_constant__ DecodeParams p) {
    using L = DecodeLayout<DP>;
    using T16 = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
    constexpr float kShift = kBF16 ? 0.f : 6.f;  // fp16: P scaled by 2^6, as is the sum
    constexpr int NS = L::kStages, RB = 2 * DP;  // RB: bytes of a key's row
    constexpr int kChunks = DP / 8;

    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_scan[kWarps];
    __shared__ Place s_start;
    __shared__ float s_m[kWarps][kMaxRows], s_l[kWarps][kMaxRows];
    __shared__ unsigned s_bad[2][DP];  // keys (bit j: key len - 16 + j) whose value in that dim is NaN | +Inf << 16, -Inf
    __shared__ int s_any_bad;
    float* join = reinterpret_cast<float*>(smem + L::kRing);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const int W = p.group, gw = warp & (W - 1), w0 = warp - gw;  // this warp in its group, the group's first
    const int unit = kSlice * W;
    const size_t rows = (size_t)p.T * p.Hq;
    pdl_launch_dependents();

    auto seq_at = [&](int s) {
        const Seq q = seq_of(p.cu_q, p.kv_lens, p.T, p.G, p.max_rows, p.max_pages, p.page_size, unit, s, p.err);
        if (p.only && q.n > 0 && q.tiles == 0) bad_index(p.err);  // more rows than the caller's bound, or a bad length
        return q;
    };
    auto group_sync = [&] {
        if (W == 1) __syncwarp();
        else named_bar_sync(1 + w0 / W, 32 * W);
    };

    if (tid < 2 * DP) (&s_bad[0][0])[tid] = 0;
    if (tid == 0) s_any_bad = 0;

    Place at{};
    int units = 0x7fffffff;                                            // of this CTA's share
    const int slots = gridDim.x * (kWarps / W);                        // kWhole: groups
    int item = blockIdx.x * (kWarps / W) + w0 / W;
    // kWhole: the group's next item that has work; s = B: none
    auto next_item = [&](Place& x, int& i) {
        const int items = p.B * p.Hk;
        for (; i < items; i += slots) {
            x.s = i / p.Hk;
            x.h = i - x.s * p.Hk;
            x.tile = 0;
            x.seq = seq_at(x.s);
            if (x.seq.tiles) return;
        }
        x.s = p.B;
    };
    if (p.mode == kWhole) {
        next_item(at, item);
        __syncthreads();
    } else if (p.mode == kCluster) {
        const int it = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
        at.s = it / p.Hk;
        at.h = it - at.s * p.Hk;
        at.seq = seq_at(at.s);
        if (at.seq.tiles == 0) {  // in all CTAs of the cluster
            if (p.overlap) pdl_wait();
            return;
        }
        at.tile = (int)((long long)at.seq.tiles * rank / p.cluster);
        units = (int)((long long)at.seq.tiles * (rank + 1) / p.cluster) - at.tile;
        __syncthreads();
    } else {
        // ----------------------------------- this CTA's share of the line
        Seq mine{};
        long long count = 0;
#pragma unroll 1
        for (int s = tid; s < p.B; s += kThreads) {
            mine = seq_at(s);
            count += (long long)mine.tiles * p.Hk;
        }
        const long long total = block_sum(count, s_scan);
        const long long ctas = min((long long)gridDim.x, total);  // that have work, one unit at least
        if (blockIdx.x >= ctas) {
            if (p.overlap) pdl_wait();
            return;
        }
        const long long u0 = total * blockIdx.x / ctas;
        units = (int)(total * (blockIdx.x + 1) / ctas - u0);
        long long before = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < p.B; s0 += kThreads) {
            const int s = s0 + tid;
            if (p.B > kThreads) mine = s < p.B ? seq_at(s) : Seq{};
            const long long n = (long long)mine.tiles * p.Hk;
            long long incl = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const long long x = __shfl_up_sync(~0u, incl, d);
                if (lane >= d) incl += x;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = incl;
            __syncthreads();
            long long lo = before + incl - n, all = before;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) lo += s_scan[w];
                all += s_scan[w];
            }
            if (n > 0 && u0 >= lo && u0 < lo + n)
                s_start = Place{s, (int)((u0 - lo) / mine.tiles), (int)((u0 - lo) % mine.tiles), mine};
            before = all;
            if (before > u0) break;
        }
        __syncthreads();
        at = s_start;
    }
    // The unit after x (of this CTA's share, while there are any); s = B behind the last.
    auto next_unit = [&](Place& x, int& i) {
        if (++x.tile < x.seq.tiles) return;
        if (p.mode == kWhole) {
            i += slots;
            next_item(x, i);
            return;
        }
        x.tile = 0;
        if (++x.h < p.Hk) return;
        x.h = 0;
        do {
            if (++x.s >= p.B) return;
            x.seq = seq_at(x.s);
        } while (x.seq.tiles == 0);
    };

    Place ahead = at;  // `at`: the unit in work; `ahead`: the next one to load
    int ahead_item = item;
    const uint32_t ring = smem_u32(smem) + warp * NS * L::kStage;
    auto page_of = [&](const Place& x) {
        const int key = x.tile * unit + gw * kSlice;
        return x.s < p.B && key < x.seq.len ? __ldg(p.table + x.s * p.table_stride + (key >> p.page_shift)) : 0;
    };
    int page = units > 0 ? page_of(ahead) : 0;
    // This lane's 16-byte chunk of a step's rows r0, r0 + RS, ...: where it is read, and
    // where it goes (chunk c of row r at chunk c ^ (r & 7)).
    constexpr int RS = 32 / kChunks;
    const int chunk = lane % kChunks, r0 = lane / kChunks;
    const long long k_lane = r0 * p.k_st + chunk * 8, v_lane = r0 * p.v_st + chunk * 8;
    const uint32_t s_lane = r0 * RB + ((chunk ^ r0) << 4);

    uint32_t qf[DP / 16][4];
    float o[DP / 8][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int lim[2] = {0, 0}, lim_min = 0, tile0 = 0;
    bool first_seg = true, fresh = true, waited = !p.overlap;

    // Ends the item in work: joins the warps and writes it, or its partial.
    auto leave = [&](bool whole) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(~0u, l[e], 1);
            l[e] += __shfl_xor_sync(~0u, l[e], 2);
            if (t4 == 0) {
                s_m[warp][g + 8 * e] = m[e];
                s_l[warp][g + 8 * e] = l[e];
            }
        }
        const int R = at.seq.n * p.G;
        if (p.prefix_splits && p.mode != kFlat && !waited) {  // the prefix's partials are complete
            pdl_wait();
            waited = true;
        }
        // A cluster's partials: [16][DP] sums, [16] maxima and sums, where the ring was
        // (every warp is past its last unit at the barrier below).
        float* part = reinterpret_cast<float*>(smem);
        const int d = 4 * lane;
        // row r of the item from its joined sums
        auto write = [&](int r, Row& x) {
            const int tok = r / p.G, hd = at.h * p.G + r % p.G;
            const int see = keys_seen(at.seq.len, at.seq.n, tok, 1);
            const size_t row = (size_t)(at.seq.first + tok) * p.Hq + hd;
            const bool out = whole && !p.own_o;
            if (out && p.prefix_splits) {
                x.top -= kShift;
                join_prefix(p.pre_o, p.pre_l, p.prefix_splits, rows, row, p.D, d, x);
                x.top += kShift;
            }
            // no key: zeros; scores that are all -inf: NaN, or left to the join
            const float inv = x.sum != 0.f ? 1.f / x.sum : (out && see + p.prefix_len > 0 ? NAN : 0.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) x.acc[e] = x.sum != 0.f ? x.acc[e] * inv : inv;
            const float l2 = x.sum == 0.f ? -INFINITY : x.top - kShift + log2f(x.sum);
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
        };
#pragma unroll 1
        for (int half = 0; 8 * half < R; ++half) {
            if (g + 8 * half < R) {
#pragma unroll
                for (int i = 0; i < DP / 8; ++i)
                    *reinterpret_cast<float2*>(join + (warp * 8 + g) * L::kPitch + 8 * i + 2 * t4) =
                        half ? make_float2(o[i][2], o[i][3]) : make_float2(o[i][0], o[i][1]);
            }
            group_sync();
            // one warp a row, four dims a lane
#pragma unroll 1
            for (int r = 8 * half + gw; r < min(R, 8 * half + 8); r += W) {
                Row x{};
                x.top = -INFINITY;
#pragma unroll 4
                for (int w = 0; w < W; ++w) x.top = fmaxf(x.top, s_m[w0 + w][r]);
                const float base = x.top == -INFINITY ? 0.f : x.top;
#pragma unroll 4
                for (int w = 0; w < W; ++w) {
                    const float f = ex2(s_m[w0 + w][r] - base);
                    x.sum += f * s_l[w0 + w][r];
                    if (d < DP) {
                        const float2* src = reinterpret_cast<const float2*>(join + ((w0 + w) * 8 + (r & 7)) * L::kPitch + d);
                        const float2 a = src[0], b = src[1];
                        x.acc[0] += f * a.x;
                        x.acc[1] += f * a.y;
                        x.acc[2] += f * b.x;
                        x.acc[3] += f * b.y;
                    }
                }
                if (s_any_bad && d < DP) {
                    // of the last 16 keys, the first `vis` are seen
                    const int vis = keys_seen(at.seq.len, at.seq.n, r / p.G, 1) - (at.seq.len - 16);
                    const unsigned mask = vis >= 16 ? 0xFFFFu : vis > 0 ? (1u << vis) - 1u : 0u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned b0 = s_bad[0][d + e], b1 = s_bad[1][d + e];
                        if ((b0 >> 16) & mask) x.acc[e] += INFINITY;
                        if (b1 & mask) x.acc[e] -= INFINITY;
                        if (b0 & mask) x.acc[e] = NAN;
                    }
                }
                if (p.mode == kCluster) {
                    if (d < DP) *reinterpret_cast<float4*>(part + r * DP + d) = make_float4(x.acc[0], x.acc[1], x.acc[2], x.acc[3]);
                    if (lane == 0) {
                        part[kMaxRows * DP + r] = x.top;
                        part[kMaxRows * DP + kMaxRows + r] = x.sum;
                    }
                } else {
                    write(r, x);
                }
            }
            group_sync();
        }
        if (p.mode == kCluster) {
            cluster_sync();
            // the rows over all warps of the cluster
#pragma unroll 1
            for (int r = (int)cluster_ctarank() * kWarps + warp; r < R; r += p.cluster * kWarps) {
                Row x{};
                const uint32_t base = smem_u32(part);
                const bool have = lane < p.cluster;  // lane q: CTA q
                const uint32_t ml = mapa_shared(base + (kMaxRows * DP + r) * 4, have ? lane : 0);
                const float mq = have ? ld_dsmem_f1(ml) : -INFINITY, lq = have ? ld_dsmem_f1(ml + kMaxRows * 4) : 0.f;
                x.top = mq;
#pragma unroll
                for (int k = 16; k; k >>= 1) x.top = fmaxf(x.top, __shfl_xor_sync(~0u, x.top, k));
                const float f = ex2(mq - (x.top == -INFINITY ? 0.f : x.top));
                x.sum = f * lq;
#pragma unroll
                for (int k = 16; k; k >>= 1) x.sum += __shfl_xor_sync(~0u, x.sum, k);
#pragma unroll 4
                for (int q = 0; q < p.cluster; ++q) {
                    const float fq = __shfl_sync(~0u, f, q);
                    if (d >= DP) continue;
                    const float4 y = ld_dsmem_f4(mapa_shared(base + (r * DP + d) * 4, q));
                    x.acc[0] += fq * y.x;
                    x.acc[1] += fq * y.y;
                    x.acc[2] += fq * y.z;
                    x.acc[3] += fq * y.w;
                }
                write(r, x);
            }
            cluster_sync();  // the others' partials have been read
        } else if (s_any_bad) {  // W = 8: the same in all threads since the barriers above
            __syncthreads();
            if (tid < 2 * DP) (&s_bad[0][0])[tid] = 0;
            if (tid == 0) s_any_bad = 0;
            __syncthreads();
        }
        first_seg = false;
        fresh = true;
    };

    // The request of one unit runs NS - 1 units ahead of the work.  A CTA of a cluster
    // may have no unit; it takes one empty step.
    int loaded = 0, load_st = 0, work_st = 0;
#pragma unroll 1
    for (int u = 1 - NS;; ++u) {
        if (loaded < units && ahead.s < p.B) {
            // This warp's keys of unit `ahead`; rows behind the last key and dims behind D
            // are filled with zeros.
            const int key = ahead.tile * unit + gw * kSlice;
            if (key < ahead.seq.len) {
                const bool ok = page_ok(page, p.num_pages);
                if (!ok) bad_index(p.err);
                const long long pg = ok ? page : 0;
                const int slot = key & (p.page_size - 1), live = ok ? ahead.seq.len - key : 0;
                const T16* k = static_cast<const T16*>(p.k) + pg * p.k_sp + slot * p.k_st + ahead.h * p.k_sh;
                const T16* v = static_cast<const T16*>(p.v) + pg * p.v_sp + slot * p.v_st + ahead.h * p.v_sh;
                const uint32_t dst = ring + load_st * L::kStage + s_lane;
                const bool dims = chunk * 8 < p.D;
                const T16 *kl = k + k_lane, *vl = v + v_lane;
#pragma unroll
                for (int i = 0; i < kSlice / RS; ++i) {
                    const bool have = dims && r0 + i * RS < live;
                    const uint32_t to = (dst ^ ((i * RS & 7) << 4)) + i * RS * RB;
                    cp_async16_zfill(to, have ? kl : k, have);
                    cp_async16_zfill(to + kSlice * RB, have ? vl : v, have);
                    kl += RS * p.k_st;
                    vl += RS * p.v_st;
                }
            }
            load_st = load_st + 1 == NS ? 0 : load_st + 1;
            if (++loaded < units) {
                next_unit(ahead, ahead_item);
                page = page_of(ahead);
            }
        }
        cp_async_commit();
        if (u < 0) continue;
        const bool work = u < loaded;
        if (!work && (p.mode != kCluster || u > 0)) break;
        if (fresh) {  // a new item: its rows of Q, rows g and g + 8 in this lane
            fresh = false;
            const int R = at.seq.n * p.G;
            tile0 = at.tile;
            lim_min = keys_seen(at.seq.len, at.seq.n, 0, 1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = g + 8 * e;
                const bool live = r < R;
                const int tok = live ? r / p.G : 0, hd = at.h * p.G + (live ? r - tok * p.G : 0);
                lim[e] = live ? keys_seen(at.seq.len, at.seq.n, tok, 1) : at.seq.len;
                m[e] = -INFINITY;
                l[e] = 0.f;
                const T16* q = static_cast<const T16*>(p.q) + (size_t)(at.seq.first + tok) * p.q_st + (size_t)hd * p.q_sh;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int d = 16 * k + 8 * x + 2 * t4;
                        qf[k][e + 2 * x] = live && d < p.D ? __ldg(reinterpret_cast<const uint32_t*>(q + d)) : 0u;
                    }
            }
#pragma unroll
            for (int i = 0; i < DP / 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
        }
        cp_async_wait<NS - 1>();
        __syncwarp();
        const int key0 = at.tile * unit + gw * kSlice;
        if (work && key0 < at.seq.len) {
            const uint32_t kst = ring + work_st * L::kStage, vst = kst + kSlice * RB;
            const bool masked = key0 + kSlice > lim_min;
            if (masked && at.seq.n > 1) {
                // Values that only some rows see and that are not finite would reach the
                // others as 0 x NaN: taken out here, put back into the rows that see them
                // at the end.  Only the last n <= 16 keys can be such.
                const int lo = max(0, lim_min - key0), hi = min(kSlice, at.seq.len - key0);
#pragma unroll 1
                for (int x = lane; x < (hi - lo) * kChunks; x += 32) {
                    const int r = lo + x / kChunks, c = x % kChunks;
                    const uint32_t a = vst + r * RB + ((c ^ (r & 7)) << 4);
                    const uint4 v4 = lds128(a);
                    if (!not_finite<kBF16>(v4)) continue;
                    uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
                    constexpr uint32_t kExp = kBF16 ? 0x7F80u : 0x7C00u;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                        if ((h & kExp) != kExp) continue;
                        const unsigned bit = 1u << (key0 + r - (at.seq.len - 16));
                        if ((h & 0x7FFFu) != kExp) atomicOr(&s_bad[0][c * 8 + e], bit);
                        else if (h & 0x8000u) atomicOr(&s_bad[1][c * 8 + e], bit);
                        else atomicOr(&s_bad[0][c * 8 + e], bit << 16);
                        w[e >> 1] &= ~(0xFFFFu << (16 * (e & 1)));
                    }
                    sts128(a, make_uint4(w[0], w[1], w[2], w[3]));
                    s_any_bad = 1;
                }
                __syncwarp();
            }
            float s[2][4] = {}, s2[2][4] = {};  // even and odd steps: two chains an n-tile
            const int kr = ((lane >> 4) << 3) + (lane & 7), kc = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < DP / 16; k += 2) {
                uint32_t b[4];
                ldsm4(kst + kr * RB + (((2 * k + kc) ^ (kr & 7)) << 4), b);
                mma_16816<kBF16>(s[0], qf[k], b[0], b[1]);
                mma_16816<kBF16>(s[1], qf[k], b[2], b[3]);
                ldsm4(kst + kr * RB + (((2 * k + 2 + kc) ^ (kr & 7)) << 4), b);
                mma_16816<kBF16>(s2[0], qf[k + 1], b[0], b[1]);
                mma_16816<kBF16>(s2[1], qf[k + 1], b[2], b[3]);
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nt][e] = (s[nt][e] + s2[nt][e]) * p.scale_log2;
                    if (masked && key0 + 8 * nt + 2 * t4 + (e & 1) >= lim[e >> 1]) s[nt][e] = -INFINITY;
                }
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                x[e] = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
            if (__any_sync(~0u, x[0] > m[0] + 8.f || x[1] > m[1] + 8.f)) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[e] = fmaxf(x[e], __shfl_xor_sync(~0u, x[e], 1));
                    x[e] = fmaxf(x[e], __shfl_xor_sync(~0u, x[e], 2));
                    x[e] = fmaxf(x[e], m[e]);
                    f[e] = ex2(m[e] - (x[e] == -INFINITY ? 0.f : x[e]));
                    m[e] = x[e];
                    l[e] *= f[e];
                }
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    o[i][0] *= f[0];
                    o[i][1] *= f[0];
                    o[i][2] *= f[1];
                    o[i][3] *= f[1];
                }
            }
            uint32_t pf[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float sub = m[e] == -INFINITY ? 0.f : m[e] - kShift;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float a = ex2(s[nt][2 * e] - sub), b = ex2(s[nt][2 * e + 1] - sub);
                    l[e] += a + b;
                    pf[e + 2 * nt] = pack2<kBF16>(a, b);
                }
            }
            const int vr = (((lane >> 3) & 1) << 3) + (lane & 7), vc = lane >> 4;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                uint32_t b[4];
                ldsm4_t(vst + vr * RB + (((2 * i + vc) ^ (vr & 7)) << 4), b);
                mma_16816<kBF16>(o[2 * i], pf, b[0], b[1]);
                mma_16816<kBF16>(o[2 * i + 1], pf, b[2], b[3]);
            }
        }
        __syncwarp();  // the stage is read; the next request may fill it
        work_st = work_st + 1 == NS ? 0 : work_st + 1;
        if (at.tile + 1 == at.seq.tiles || u + 1 >= units) leave(p.mode != kFlat || (tile0 == 0 && at.tile + 1 == at.seq.tiles));
        if (u + 1 < units) next_unit(at, item);
    }
    cp_async_wait<0>();
    if (!waited) pdl_wait();  // what waits for this kernel waits for the one before it, too
}

// kFlat: joins the partials of every item that more than one CTA worked on, and with
// a shared prefix of every one, with the prefix's.  One block each; the
// partials' weights first, then warp w adds up every eighth partial.
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
    extern __shared__ __align__(16) float weights[];  // [partials][16]
    __shared__ float buf[kWarps][8][128];
    __shared__ long long scan[kWarps];
    __shared__ float s_sum[kMaxRows], s_top[kMaxRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int s = blockIdx.x, hk = blockIdx.y;
    pdl_wait();
    auto seq_at = [&](int x) {
        return seq_of(p.cu_q, p.kv_lens, p.T, p.G, p.max_rows, p.max_pages, p.page_size, kUnit, x, nullptr);
    };
    const Seq me = seq_at(s);
    if (me.tiles == 0) return;
    long long before = 0, total = 0;
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
    const bool whole = c0 == c1;
    if (whole && !p.prefix_splits) return;
    const int own = whole ? 1 : c1 - c0 + 1, parts = own + p.prefix_splits;
    const int R = me.n * p.G;
    const size_t rows = (size_t)p.T * p.Hq;
    const bool mid = ub != total * c0 / ctas;  // CTA c0 begins with another (sequence, head)
    auto row_of = [&](int r) { return (size_t)(me.first + r / p.G) * p.Hq + hk * p.G + r % p.G; };
    auto slot_of = [&](int i) { return (size_t)(2 * (c0 + i) + (i == 0 && mid ? 1 : 0)) * kMaxRows; };
    for (int x = tid; x < parts * kMaxRows; x += kThreads) {
        const int i = x / kMaxRows, r = x % kMaxRows;
        if (r < R)
            weights[x] = i >= own ? p.pre_l[(i - own) * rows + row_of(r)] : whole ? p.own_l[row_of(r)] : p.slot_l[slot_of(i) + r];
    }
    __syncthreads();
    for (int r = warp; r < R; r += kWarps) {
        float top = -INFINITY, sum = 0.f;
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, weights[i * kMaxRows + r]);
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const float base = top == -INFINITY ? 0.f : top;
        for (int i = lane; i < parts; i += 32) {
            const float w = ex2(weights[i * kMaxRows + r] - base);
            weights[i * kMaxRows + r] = w;
            sum += w;
        }
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if (lane == 0) {
            s_sum[r] = sum;
            s_top[r] = top;
        }
    }
    __syncthreads();
    const int d = 4 * lane;
    for (int r0 = 0; r0 < R; r0 += 8) {
        const int nr = min(8, R - r0);
        float acc[8][4] = {};
        if (d < p.D) {
            for (int i = warp; i < parts; i += kWarps) {
                const float* src = i >= own ? p.pre_o + (i - own) * rows * p.D
                                            : whole ? p.own_o : p.slot_o + slot_of(i) * p.D;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r >= nr) continue;
                    const size_t at = i >= own || whole ? row_of(r0 + r) : (size_t)(r0 + r);
                    const float4 x = *reinterpret_cast<const float4*>(src + at * p.D + d);
                    const float w = weights[i * kMaxRows + r0 + r];
                    acc[r][0] += w * x.x;
                    acc[r][1] += w * x.y;
                    acc[r][2] += w * x.z;
                    acc[r][3] += w * x.w;
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
            *reinterpret_cast<float4*>(&buf[warp][r][d]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
        __syncthreads();
        if (warp < nr) {
            const int r = r0 + warp;
            float x[4] = {};
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 y = *reinterpret_cast<const float4*>(&buf[w][warp][d]);
                x[0] += y.x;
                x[1] += y.y;
                x[2] += y.z;
                x[3] += y.w;
            }
            const int tok = r / p.G;
            const float sum = s_sum[r];
            const float inv =
                sum != 0.f ? 1.f / sum : (p.prefix_len + keys_seen(me.len, me.n, tok, 1) > 0 ? NAN : 0.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = sum != 0.f ? x[e] * inv : inv;
            if (d < p.D)
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + (size_t)(me.first + tok) * p.o_st +
                                          (size_t)(hk * p.G + r % p.G) * p.o_sh + d) =
                    make_uint2(pack2<kBF16>(x[0], x[1]), pack2<kBF16>(x[2], x[3]));
            if (p.lse && lane == 0)
                p.lse[row_of(r)] = sum == 0.f ? -INFINITY : (s_top[r] + log2f(sum)) * 0.693147180559945309417f;
        }
        __syncthreads();
    }
}

// Rows (tokens x G) of a sequence that the kernels take: alone, up to the caller's bound.
int max_rows(const AttnArgs& a, const DecodeParts& parts) {
    return parts.only ? std::min(kMaxRows, a.max_q * a.G) : kMaxRows;  // alone: max_q * G <= 16
}

template <bool kBF16, int DP>
cudaError_t launch_one(const DecodeParams& p, int ctas, int dev, cudaStream_t s) {
    auto fn = attn_decode_kernel<kBF16, DP>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(fn), dev, DecodeLayout<DP>::kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)DecodeLayout<DP>::kSmem;
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

}  // namespace

DecodePlan decode_plan(int B, int Hk, int max_q, int max_kv, int sms) {
    const long long items = (long long)B * Hk;
    const int tiles = std::max(1, (max_kv + kUnit - 1) / kUnit);
    DecodePlan pl{};
    pl.cluster = 1;
    pl.group = kWarps;
    // A cluster per item while they fill no more than the SMs and no CTA has more than
    // 8 units (1024 keys, 0.5 MB): beyond, a share of every SM is faster in spite of
    // the join's launch.
    int cs = 1;
    while (cs < 8 && items * cs * 2 <= sms && cs < tiles) cs *= 2;
    if (cs > 1 && tiles <= 8 * cs) {
        pl.mode = kCluster;
        pl.cluster = cs;
        pl.ctas = (int)items * cs;
        return pl;
    }
    // Whole items where no group has more than 24 units of work, with so many warps an
    // item that one round takes all items if it can.  (Groups of fewer than 8 warps
    // have no room for values that only some of a sequence's rows see: one row each.)
    int W = kWarps;
    while (W > 1 && max_q == 1 && items * W > (long long)sms * kWarps) W /= 2;
    const long long slots = (long long)sms * (kWarps / W), rounds = (items + slots - 1) / slots;
    if (rounds * std::max(1, (max_kv + kSlice * W - 1) / (kSlice * W)) <= 24) {
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
    DecodeParams p{};
    p.q = a.q;
    p.q_st = a.q_st;
    p.q_sh = a.q_sh;
    p.o = a.o;
    p.o_st = a.o_st;
    p.o_sh = a.o_sh;
    p.lse = a.lse;
    p.k = a.k;
    p.v = a.v;
    p.k_sp = a.k_sp;
    p.k_st = a.k_st;
    p.k_sh = a.k_sh;
    p.v_sp = a.v_sp;
    p.v_st = a.v_st;
    p.v_sh = a.v_sh;
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
    p.only = parts.only;
    p.mode = parts.plan.mode;
    p.cluster = parts.plan.cluster;
    p.group = parts.plan.group;
    p.max_rows = max_rows(a, parts);
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
    const int ctas = parts.plan.ctas;
    if (a.D <= 64)
        return a.dtype == DType::BF16 ? launch_one<true, 64>(p, ctas, a.dev, a.stream) : launch_one<false, 64>(p, ctas, a.dev, a.stream);
    return a.dtype == DType::BF16 ? launch_one<true, 128>(p, ctas, a.dev, a.stream) : launch_one<false, 128>(p, ctas, a.dev, a.stream);
}

cudaError_t launch_attn_join(const AttnArgs& a, const DecodeParts& parts) {
    JoinParams j{parts.slot_o, parts.slot_l, parts.own_o, parts.own_l, parts.pre_o, parts.pre_l, a.o, a.o_st, a.o_sh, a.lse,
                 a.cu_q, a.kv_lens, a.T, a.B, a.Hq, a.Hk, a.G, a.D, a.page_size, a.max_pages, max_rows(a, parts),
                 parts.plan.ctas, parts.prefix_splits, a.prefix_len};
    auto fn = a.dtype == DType::BF16 ? attn_join_kernel<true> : attn_join_kernel<false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.B, (unsigned)a.Hk);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)(parts.plan.ctas + parts.prefix_splits) * kMaxRows * 4;
    cfg.stream = a.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, j);
}

}  // namespace hq
