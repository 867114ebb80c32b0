// hq_attn_tile.cu -- attention of many rows on the tensor cores: whole prompts,
// prompt chunks over the paged cache, and a prefix that a batch shares.
//
// The rows of a key/value head are its sequence's tokens times the G query heads
// that share it, row r being head r % G of token r / G: a tile's rows read the
// same keys, so one pass over K and V serves all of them, and few rows of the
// causal triangle's edge are wasted.  One CTA takes 256 rows as two tiles of 128
// and walks the keys 128 at a time:
//   S = Q K^T        tcgen05.mma, both operands in shared memory, S (fp32) in
//                    tensor memory
//   P = 2^(c S - m)  one thread a row: running maximum m, running sum l (fp32);
//                    P rounded to the 16-bit type, over S in tensor memory
//   O += P V         tcgen05.mma, P from tensor memory, V from shared memory as
//                    it lies ([key][dim]: the MMA's N dimension is contiguous)
// While one tile's rows are in the softmax the tensor cores work on the other.
// m is moved, and O scaled, only when the maximum has grown by more than 2^8
// since it was last moved: until then the sums stay exact in fp32 and P, at most
// 2^8 (2^14 in fp16, see kShift), in range.
//
//   warp 0        loads: one TMA box per 64 dims and up to 128 keys of a page
//                 (page numbers from the table), K and V tiles alternate in a ring
//   warp 1        issues the MMAs (one thread); owns the tensor memory
//   warps 2, 3    V tiles that some row does not see in full: rows behind the
//                 last key are zeroed (0 x NaN would reach the sum), and values
//                 that are not finite are taken out and noted, to be put back into
//                 the rows that see them
//   warps 4-7, 8-11  softmax and output of tile 0, tile 1: thread = row = lane of
//                 tensor memory
// Bound: the tensor cores and the exponentials (16 a clock and SM) alike take
// 128 x 128 x 2 per 1024 cycles.
// Work is split over the keys when there are few rows: every split writes its
// normalised fp32 output and log2 of its sum, merged by attn_merge_kernel.
// Every wait is bounded (hq_common.cuh): after one that gave up the roles run on
// without waiting, so that all of them end.
#include "hq_attn.cuh"
#include "hq_tmap.h"

#include <algorithm>
#include <climits>
#include <cstring>
#include <type_traits>

namespace hq {

namespace {

constexpr int kRows = 128;  // rows of a tile (MMA M), keys of a tile
constexpr int kKeys = 128;
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;  // S / P of tile t at 128 t, O of tile t at 256 + DP t

template <int DP>
struct TileLayout {
    static constexpr int kBlk = DP / 64;             // 64-dim blocks of 128-byte rows
    static constexpr int kBlkBytes = 128 * 128;      // 128 rows of one block
    static constexpr int kTile = kBlk * kBlkBytes;   // 128 rows of Q, K or V
    static constexpr int kStages = DP == 128 ? 5 : 8;
    static constexpr int kSmem = 2 * kTile + kStages * kTile + 1024;  // Q, ring, alignment slack
};

struct alignas(64) TileParams {
    CUtensorMap k_map, v_map;  // {dim, token, head, page}
    const void* q;
    long long q_st, q_sh;
    void* o;
    long long o_st, o_sh;
    float* lse;
    float* part_o;  // [split][T * Hq][D] and [split][T * Hq]; null: out is written
    float* part_l;
    const int* cu_q;
    const int* table;
    long long table_stride;
    const int* kv_lens;
    int T, B, Hq, G, D;
    int causal;
    float scale_log2;
    int page_size, box_rows, num_pages, max_pages;  // page_size 0: packed rows
    int prefix_len;                                 // > 0: all T rows over the pages table[0..]
    int splits;
    int skip_rows;  // sequences of at most this many rows (tokens x G) are not this kernel's
    unsigned* err;
};

struct TileShared {
    uint64_t full[8], empty[8], q_full, s_full[2], p_full[2], o_full[2], v_req, v_clean;
    uint32_t tmem;
    int seq, block;              // this CTA's sequence and 256-row block; seq -1: none
    int any_bad;
    int bad[3][128];             // first key whose value in that dim is NaN, +Inf, -Inf
};

__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}

// Shared-memory matrix descriptor, N contiguous (V as the B operand): 128-byte
// swizzle, 64-element blocks kBlkBytes apart, groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t addr) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((128 * 128) >> 4) << 16;  // leading byte offset: the next 64 of N
    d |= (uint64_t)(1024 >> 4) << 32;         // stride byte offset: the next 8 of K
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// 32 columns of this warp's lanes; the wait is part of the statement, so nothing
// that uses the registers can be moved before it.
__device__ __forceinline__ void tmem_ld32_now(uint32_t taddr, float (&f)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// The sequence and 256-row block of this CTA: blocks are numbered through the
// sequences, and taken last first (the last block of a causal prompt has the
// most keys).  One warp; every lane returns the same.
__device__ void find_block(const TileParams& p, int want, int& seq, int& block, unsigned* err) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    seq = -1;
    block = 0;
    for (int s0 = 0; s0 < p.B; s0 += 32) {
        const int s = s0 + lane;
        int first = 0, n = 0, nb = 0;
        if (s < p.B) {
            bool ok = seq_rows(p.cu_q, s, p.T, first, n);
            if (ok && p.page_size) ok = len_ok(p.kv_lens[s], p.max_pages, p.page_size);
            if (!ok) bad_index(err);
            else if ((long long)n * p.G > p.skip_rows) nb = (int)(((long long)n * p.G + 2 * kRows - 1) / (2 * kRows));
        }
        int incl = nb;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(~0u, incl, d);
            if (lane >= d) incl += x;
        }
        const int lo = before + incl - nb;
        const unsigned hit = __ballot_sync(~0u, want >= lo && want < lo + nb);
        if (hit) {
            const int l = __ffs(hit) - 1;
            seq = s0 + l;
            block = want - __shfl_sync(~0u, lo, l);
            return;
        }
        before += __shfl_sync(~0u, incl, 31);
    }
}

template <bool kBF16, int DP>
__global__ void __launch_bounds__(kThreads, 1) attn_tile_kernel(const __grid_constant__ TileParams p) {
    using L = TileLayout<DP>;
    using T16 = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
    constexpr int S = L::kStages;
    // fp16 keeps 10 bits down to 2^-14 only: P is scaled by 2^6, which the sum l
    // carries too, so weights down to 2^-20 of the largest keep them.
    constexpr float kShift = kBF16 ? 0.f : 6.f;
    constexpr uint32_t kIdescS = umma_idesc_f16(kBF16, kRows, kKeys);
    constexpr uint32_t kIdescO = umma_idesc_f16(kBF16, kRows, DP) | (1u << 16);  // B: N contiguous

    extern __shared__ uint8_t smem_raw[];
    __shared__ TileShared sh;
    uint8_t* qs = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* ring = qs + 2 * L::kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0) {
        int seq = 0, block = (int)(gridDim.x - 1 - blockIdx.x);
        if (!p.prefix_len) find_block(p, block, seq, block, p.err);
        if (lane == 0) {
            sh.seq = seq;
            sh.block = block;
            sh.any_bad = 0;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            for (int i = 0; i < S; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1);
            }
            mbar_init(&sh.q_full, 256);
            for (int t = 0; t < 2; ++t) {
                mbar_init(&sh.s_full[t], 1);
                mbar_init(&sh.p_full[t], 128);
                mbar_init(&sh.o_full[t], 1);
            }
            mbar_init(&sh.v_req, 1);
            mbar_init(&sh.v_clean, 64);
            fence_mbarrier_init();
            fence_async_smem();
        }
        __syncwarp();
        tmem_alloc(&sh.tmem, kTmemCols);
        tmem_relinquish();
    } else if (warp >= 4) {
        for (int i = threadIdx.x - 128; i < 3 * 128; i += 256) (&sh.bad[0][0])[i] = INT_MAX;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int seq = sh.seq;

    // This CTA's rows and keys (the same numbers in every thread).
    int first = 0, n = 0, len = 0;
    if (seq >= 0) {
        if (p.prefix_len) {
            n = p.T;
            len = p.prefix_len;
        } else {
            seq_rows(p.cu_q, seq, p.T, first, n);
            len = p.page_size ? p.kv_lens[seq] : n;
        }
    }
    const int R = n * p.G;  // fits: n_tokens * n_heads does
    const int row0 = sh.block * 2 * kRows;
    const int hk = blockIdx.y, split = blockIdx.z;
    const int causal = p.causal && !p.prefix_len;
    auto seen_of = [&](int r) { return keys_seen(len, n, min(r, R - 1) / p.G, causal); };
    int ni[2] = {0, 0}, k_first = 0, m_first = 0;  // key tiles of each row tile; first key; first tile with a mask
    if (seq >= 0 && row0 < R) {
        const int end1 = (seen_of(row0 + 2 * kRows - 1) + kKeys - 1) / kKeys;
        const int end0 = (seen_of(row0 + kRows - 1) + kKeys - 1) / kKeys;
        const int a = (int)((long long)end1 * split / p.splits), b = (int)((long long)end1 * (split + 1) / p.splits);
        ni[0] = max(0, min(b, end0) - a);
        ni[1] = row0 + kRows < R ? b - a : 0;
        k_first = a * kKeys;
        m_first = max(0, seen_of(row0) / kKeys - a);
    }
    const int nt = max(ni[0], ni[1]);

    if (warp == 0) {
        // ---------------------------------------------------------- loads
        const int* table = p.prefix_len ? p.table : p.table + seq * p.table_stride;
        const int boxes = kKeys / p.box_rows;
        bool ok = true;
        int use = 0;
        for (int i = 0; i < nt; ++i) {
            const int k0 = k_first + i * kKeys;
            const int live = min(boxes, (len - k0 + p.box_rows - 1) / p.box_rows);
            for (int kv = 0; kv < 2; ++kv, ++use) {
                const int slot = use % S;
                if (ok) ok = mbar_wait(&sh.empty[slot], ((uint32_t)(use / S) & 1u) ^ 1u, p.err);
                uint8_t* dst = ring + slot * L::kTile;
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], (uint32_t)(live * L::kBlk * p.box_rows * 128));
                __syncwarp();
                for (int b = lane; b < live * L::kBlk; b += 32) {
                    const int box = b / L::kBlk, blk = b % L::kBlk;
                    const int key = k0 + box * p.box_rows;
                    int token = first + key, page = 0;
                    if (p.page_size) {
                        token = key & (p.page_size - 1);
                        page = table[key / p.page_size];
                        if (!page_ok(page, p.num_pages)) {
                            bad_index(p.err);
                            page = p.num_pages;  // out of range: the box reads zeros
                        }
                    }
                    tma_load_4d(dst + blk * L::kBlkBytes + box * p.box_rows * 128, kv ? &p.v_map : &p.k_map, blk * 64, token,
                                hk, page, &sh.full[slot]);
                }
            }
        }
        // Every stage filled here has been consumed (its commit has landed) before exit.
        for (int j = max(0, use - S); j < use; ++j) mbar_wait(&sh.empty[j % S], (uint32_t)(j / S) & 1u, p.err);
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        if (lane == 0 && nt > 0) {
            bool ok = mbar_wait(&sh.q_full, 0, p.err);
            auto wait_full = [&](int use) {
                if (ok) ok = mbar_wait(&sh.full[use % S], (uint32_t)(use / S) & 1u, p.err);
            };
            auto qk = [&](int t, int use) {
                const uint32_t qa = smem_u32(qs) + t * L::kTile, ka = smem_u32(ring) + (use % S) * L::kTile;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const uint32_t off = (k >> 2) * L::kBlkBytes + (k & 3) * 32;
                    umma_f16(tmem + 128u * t, sw128_kmajor_desc(qa + off), sw128_kmajor_desc(ka + off), kIdescS, k != 0);
                }
                umma_commit(&sh.s_full[t]);
            };
            wait_full(0);
            tc_fence_after();
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (ni[t] > 0) qk(t, 0);
            umma_commit(&sh.empty[0]);
            if (m_first == 0) mbar_arrive(&sh.v_req);
            for (int i = 0; i < nt; ++i) {
                wait_full(2 * i + 1);
                if (i + 1 < nt) wait_full(2 * i + 2);
                if (i >= m_first && ok) ok = mbar_wait(&sh.v_clean, (uint32_t)(i - m_first) & 1u, p.err);
                const uint32_t va = smem_u32(ring) + ((2 * i + 1) % S) * L::kTile;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (i >= ni[t]) continue;
                    if (ok) ok = mbar_wait(&sh.p_full[t], (uint32_t)i & 1u, p.err);
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma_ts_f16(tmem + kColO + (uint32_t)DP * t, tmem + 128u * t + 8u * k, sw128_mn_desc(va + k * 2048),
                                    kIdescO, (i | k) != 0);
                    umma_commit(&sh.o_full[t]);
                    if (i + 1 < ni[t]) qk(t, 2 * i + 2);
                }
                umma_commit(&sh.empty[(2 * i + 1) % S]);
                if (i + 1 < nt) {
                    umma_commit(&sh.empty[(2 * i + 2) % S]);
                    if (i + 1 >= m_first) mbar_arrive(&sh.v_req);
                }
            }
        }
        __syncwarp();
    } else if (warp < 4) {
        // ----------------------------------------- V tiles under a mask
        // v_req comes once the tile's K has been used, so V's stage is in this
        // use's phase or the one before it, and stays until v_clean.
        const int tid = threadIdx.x - 64;
        const int lim_min = nt > 0 ? seen_of(row0) : 0;
        bool ok = true;
        for (int i = m_first; i < nt; ++i) {
            const int use = 2 * i + 1;
            if (ok) ok = mbar_wait(&sh.v_req, (uint32_t)(i - m_first) & 1u, p.err);
            if (ok) ok = mbar_wait(&sh.full[use % S], (uint32_t)(use / S) & 1u, p.err);
            uint8_t* vt = ring + (use % S) * L::kTile;
            const int k0 = k_first + i * kKeys;
            const int valid = min(kKeys, len - k0), lo = min(valid, max(0, lim_min - k0));
            // 16-byte chunk c of row r of a block lies at chunk c ^ (r & 7)
            for (int x = tid; x < (kKeys - lo) * DP / 8; x += 64) {
                const int r = lo + x / (DP / 8), c = x % (DP / 8);
                uint4* at = reinterpret_cast<uint4*>(vt + (c >> 3) * L::kBlkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                if (r >= valid) {
                    *at = make_uint4(0u, 0u, 0u, 0u);
                    continue;
                }
                uint4 v = *at;
                constexpr uint32_t kExp = kBF16 ? 0x7F80u : 0x7C00u;
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
                bool hit = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                    if ((h & kExp) == kExp) {
                        const int kind = (h & 0x7FFFu) != kExp ? 0 : (h & 0x8000u) ? 2 : 1;
                        atomicMin(&sh.bad[kind][c * 8 + e], k0 + r);
                        w[e >> 1] &= ~(0xFFFFu << (16 * (e & 1)));
                        hit = true;
                    }
                }
                if (hit) {
                    *at = make_uint4(w[0], w[1], w[2], w[3]);
                    sh.any_bad = 1;
                }
            }
            fence_async_smem();
            mbar_arrive(&sh.v_clean);
        }
    } else {
        // ----------------------------------------------- softmax and output
        const int t = (warp - 4) >> 2, i0 = (threadIdx.x - 128) & 127;
        const int r = row0 + t * kRows + i0;
        const bool live = r < R;
        const int token = live ? r / p.G : 0, head = hk * p.G + (live ? r % p.G : 0);
        const int lim = live ? seen_of(r) : seen_of(R - 1);
        const int my = ni[t];
        if (nt > 0) {  // this row of Q, zeros behind the last row and dim
            const T16* q = static_cast<const T16*>(p.q) + (size_t)(first + token) * p.q_st + (size_t)head * p.q_sh;
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                const uint4 v = live && c * 8 < p.D ? ldg128_nc(q + c * 8) : make_uint4(0u, 0u, 0u, 0u);
                sts128(smem_u32(qs) + t * L::kTile + (c >> 3) * L::kBlkBytes + i0 * 128 + (((c & 7) ^ (i0 & 7)) << 4), v);
            }
            fence_async_smem();
            mbar_arrive(&sh.q_full);
        }
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + 128u * t, to = tmem + lanes + kColO + (uint32_t)DP * t;
        bool ok = true;
        float m = -INFINITY, l = 0.f;
        for (int i = 0; i < my; ++i) {
            if (ok) ok = mbar_wait(&sh.s_full[t], (uint32_t)i & 1u, p.err);
            __syncwarp();
            tc_fence_after();
            const int cut = i >= m_first ? lim - (k_first + i * kKeys) : kKeys;  // columns from `cut` on are not seen
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float s[32];
                tmem_ld32_now(ts + 32u * c, s);
                if (cut < kKeys) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[e] = 32 * c + e < cut ? s[e] : -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, s[e]);
            }
            mx *= p.scale_log2;
            const bool move = mx > m + 8.f;  // also from -inf; a first tile has no O yet
            if (__any_sync(~0u, move && l > 0.f)) {
                if (ok) ok = mbar_wait(&sh.o_full[t], (uint32_t)(i - 1) & 1u, p.err);
                __syncwarp();
                tc_fence_after();
                const float f = move ? ex2(m - mx) : 1.f;
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    float o[32];
                    uint32_t w[32];
                    tmem_ld32_now(to + 32u * c, o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[e] * f);
                    tmem_st32(to + 32u * c, w);
                }
                l *= f;
            }
            if (move) m = mx;
            const float sub = m == -INFINITY ? 0.f : m - kShift;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t w[32];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    float s[32];
                    tmem_ld32_now(ts + 64u * c + 32u * d, s);
                    if (cut < kKeys) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[e] = 64 * c + 32 * d + e < cut ? s[e] : -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float a = ex2(fmaf(s[e], p.scale_log2, -sub)), b = ex2(fmaf(s[e + 1], p.scale_log2, -sub));
                        sum += a + b;
                        w[16 * d + e / 2] = pack2<kBF16>(a, b);
                    }
                }
                tmem_st32(ts + 32u * c, w);
            }
            l += sum;
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&sh.p_full[t]);
        }
        if (my > 0) {
            if (ok) ok = mbar_wait(&sh.o_full[t], (uint32_t)(my - 1) & 1u, p.err);
            __syncwarp();
            tc_fence_after();
        }
        // l = 0: no key was seen (zeros), or every score was -inf (no softmax: NaN,
        // which a merge settles where other splits have a sum).
        const bool part = p.part_o != nullptr;
        const float inv = l != 0.f ? 1.f / l : (!part && lim > 0 ? NAN : 0.f);
        const size_t hrow = (size_t)(first + token) * p.Hq + head;
        const bool any_bad = sh.any_bad != 0;  // written before v_clean, which every PV waited for
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
            float o[32];
            __syncwarp();
            if (my > 0) {
                tmem_ld32_now(to + 32u * c, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = l != 0.f ? o[e] * inv : inv;
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = inv;
            }
            if (any_bad) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    if (sh.bad[1][32 * c + e] < lim) o[e] += INFINITY;
                    if (sh.bad[2][32 * c + e] < lim) o[e] -= INFINITY;
                    if (sh.bad[0][32 * c + e] < lim) o[e] = NAN;
                }
            }
            if (live && part) {
                float* dst = p.part_o + ((size_t)split * p.T * p.Hq + hrow) * p.D + 32 * c;
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    if (32 * c + e < p.D) *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else if (live) {
                T16* dst = static_cast<T16*>(p.o) + (size_t)(first + token) * p.o_st + (size_t)head * p.o_sh + 32 * c;
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    if (32 * c + e < p.D)
                        *reinterpret_cast<uint4*>(dst + e) =
                            make_uint4(pack2<kBF16>(o[e], o[e + 1]), pack2<kBF16>(o[e + 2], o[e + 3]),
                                       pack2<kBF16>(o[e + 4], o[e + 5]), pack2<kBF16>(o[e + 6], o[e + 7]));
            }
        }
        if (live) {
            const float l2 = l == 0.f ? -INFINITY : m - kShift + log2f(l);
            if (part) p.part_l[(size_t)split * p.T * p.Hq + hrow] = l2;
            else if (p.lse) p.lse[hrow] = l2 * 0.693147180559945309417f;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Merges the splits of every row: out = sum_s w_s o_s / sum_s w_s, w_s = 2^(l_s - max l)
// for split s's normalised output o_s and log2 of its sum l_s.  One warp a row and
// head, four dims a lane; reads each partial once.
struct MergeParams {
    const float *part_o, *part_l;
    void* o;
    long long o_st, o_sh;
    float* lse;
    const int* cu_q;
    const int* kv_lens;  // null: packed rows
    int T, B, Hq, D, causal, prefix_len, splits;
    int page_size, max_pages;
    int G, skip_rows;
};

template <bool kBF16>
__global__ void __launch_bounds__(256) attn_merge_kernel(const MergeParams p) {
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const size_t rows = (size_t)p.T * p.Hq;
    pdl_wait();
    if (row >= (long long)rows) return;
    const int t = (int)(row / p.Hq), h = (int)(row % p.Hq);
    // the row's sequence; rows of none, and those of the decode kernel, have no partials here
    int seen = -1;
    for (int s0 = 0; s0 < p.B && seen < 0; s0 += 32) {
        const int s = s0 + lane;
        int first = 0, n = 0, k = -1;
        if (s < p.B && seq_rows(p.cu_q, s, p.T, first, n) && t >= first && t < first + n &&
            (long long)n * p.G > p.skip_rows) {
            const int len = p.kv_lens ? p.kv_lens[s] : n;
            if (!p.kv_lens || len_ok(len, p.max_pages, p.page_size)) k = keys_seen(len, n, t - first, p.causal);
        }
        const unsigned hit = __ballot_sync(~0u, k >= 0);
        if (hit) seen = __shfl_sync(~0u, k, __ffs(hit) - 1);
    }
    if (seen < 0) return;
    float m = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_l[s * rows + row]);
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    const float base = m == -INFINITY ? 0.f : m;
    const bool have = 4 * lane < p.D;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float w = ex2(p.part_l[s * rows + row] - base);
        l += w;
        if (!have) continue;
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * p.D + 4 * lane);
        o.x += w * x.x;
        o.y += w * x.y;
        o.z += w * x.z;
        o.w += w * x.w;
    }
    const float inv = l != 0.f ? 1.f / l : (seen + p.prefix_len > 0 ? NAN : 0.f);
    if (l == 0.f) o = make_float4(1.f, 1.f, 1.f, 1.f);
    if (have) {
        uint16_t* dst = static_cast<uint16_t*>(p.o) + (size_t)t * p.o_st + (size_t)h * p.o_sh + 4 * lane;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<kBF16>(o.x * inv, o.y * inv), pack2<kBF16>(o.z * inv, o.w * inv));
    }
    if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309417f;
}

int ceil_div(long long a, int b) { return (int)((a + b - 1) / b); }

template <bool kBF16, int DP>
cudaError_t launch_tile(const TileParams& p, int blocks, int Hk, int dev, cudaStream_t s) {
    using L = TileLayout<DP>;
    auto fn = attn_tile_kernel<kBF16, DP>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(fn), dev, L::kSmem);
    if (e != cudaSuccess) return e;
    fn<<<dim3(blocks, Hk, p.splits), kThreads, L::kSmem, s>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_tile_any(const AttnArgs& a, const TileParams& p, int blocks) {
    if (a.D <= 64)
        return a.dtype == DType::BF16 ? launch_tile<true, 64>(p, blocks, a.Hk, a.dev, a.stream)
                                      : launch_tile<false, 64>(p, blocks, a.Hk, a.dev, a.stream);
    return a.dtype == DType::BF16 ? launch_tile<true, 128>(p, blocks, a.Hk, a.dev, a.stream)
                                  : launch_tile<false, 128>(p, blocks, a.Hk, a.dev, a.stream);
}

// Key splits of `blocks` x Hk CTAs over `keys` keys: enough to fill the SMs once,
// at least two key tiles each.
int key_splits(long long rows, int Hk, int keys, int sms) {
    const long long items = (long long)std::max(1, ceil_div(rows, 2 * kRows)) * Hk;
    const int by_keys = ceil_div(keys, kKeys) / 2;
    return (int)std::max(1LL, std::min({(long long)sms / items, (long long)by_keys, 32LL}));
}

cudaError_t kv_maps(const AttnArgs& a, TileParams& p) {
    // A dimension of one element takes any legal stride.
    const uint64_t any = 16;
    const uint64_t tokens = a.page_size ? a.page_size : a.T, pages = a.page_size ? a.num_pages : 1;
    const uint64_t dims[4] = {(uint64_t)a.D, tokens, (uint64_t)a.Hk, pages};
    auto one = [&](CUtensorMap* m, const void* base, long long st, long long sh, long long sp) {
        const uint64_t strides[3] = {tokens > 1 ? 2 * (uint64_t)st : any, a.Hk > 1 ? 2 * (uint64_t)sh : any,
                                     pages > 1 ? 2 * (uint64_t)sp : any};
        return make_tmap_4d(m, base, dims, strides, (uint32_t)p.box_rows);
    };
    cudaError_t e = one(&p.k_map, a.k, a.k_st, a.k_sh, a.k_sp);
    return e != cudaSuccess ? e : one(&p.v_map, a.v, a.v_st, a.v_sh, a.v_sp);
}

}  // namespace

AttnPlan attn_plan(int T, int B, int max_q, int Hq, int Hk, int D, bool paged, int max_kv, int prefix_len, int sms) {
    AttnPlan pl{};
    const int G = Hq / Hk;
    const long long rows = (long long)T * G;
    pl.tile = !paged || (long long)max_q * G > kDecodeRows;
    pl.decode = paged && G <= kDecodeRows && (!pl.tile || B > 1);
    pl.prefix = prefix_len > 0 ? key_splits(rows, Hk, prefix_len, sms) : 0;
    pl.own = pl.tile ? key_splits(rows, Hk, max_kv, sms) : 0;
    pl.planes = pl.prefix;
    if (pl.tile && pl.own + pl.prefix > 1) pl.planes += pl.own;
    size_t slots = 0;
    if (pl.decode) {
        pl.ctas = decode_ctas(B, Hk, max_kv, sms);
        // A join costs a launch: lengths that a CTA reads in less time are not split.
        pl.whole = max_kv <= 256;
        if (pl.prefix) ++pl.planes;
        if (!pl.whole) slots = (size_t)pl.ctas * 2 * kDecodeRows;
    }
    pl.bytes = ((pl.planes * T * Hq + slots) * (D + 1) * 4 + 255) & ~(size_t)255;
    return pl;
}

cudaError_t launch_attn(const AttnArgs& a) {
    const AttnPlan pl = attn_plan(a.T, a.B, a.max_q, a.Hq, a.Hk, a.D, a.page_size > 0, a.max_kv, a.prefix_len, a.sm_count);
    // workspace: outputs of the planes, of the decode slots, then the sums of both
    const size_t rows = (size_t)a.T * a.Hq, slots = pl.decode && !pl.whole ? (size_t)pl.ctas * 2 * kDecodeRows : 0;
    float* plane_o = reinterpret_cast<float*>(a.ws);
    float* slot_o = plane_o + pl.planes * rows * a.D;
    float* plane_l = slot_o + slots * a.D;
    float* slot_l = plane_l + pl.planes * rows;

    cudaError_t e = cudaSuccess;
    TileParams p;
    memset(&p, 0, sizeof p);
    if (pl.tile || pl.prefix) {
        p.q = a.q;
        p.q_st = a.q_st;
        p.q_sh = a.q_sh;
        p.o = a.o;
        p.o_st = a.o_st;
        p.o_sh = a.o_sh;
        p.lse = a.lse;
        p.cu_q = a.cu_q;
        p.kv_lens = a.kv_lens;
        p.T = a.T;
        p.B = a.B;
        p.Hq = a.Hq;
        p.G = a.G;
        p.D = a.D;
        p.causal = a.causal;
        p.scale_log2 = a.scale * 1.44269504088896340736f;
        p.page_size = a.page_size;
        p.box_rows = a.page_size ? std::min(a.page_size, kKeys) : kKeys;
        p.num_pages = a.num_pages;
        p.max_pages = a.max_pages;
        p.err = a.err;
        if ((e = kv_maps(a, p)) != cudaSuccess) return e;
    }
    const int row_blocks = ceil_div((long long)a.T * a.G, 2 * kRows);
    if (pl.prefix) {
        TileParams x = p;
        x.prefix_len = a.prefix_len;
        x.table = a.prefix_table;
        x.splits = pl.prefix;
        x.part_o = plane_o;
        x.part_l = plane_l;
        if ((e = launch_tile_any(a, x, row_blocks)) != cudaSuccess) return e;
    }
    if (pl.tile) {
        const bool part = pl.own + pl.prefix > 1;
        p.table = a.table;
        p.table_stride = a.table_stride;
        p.splits = pl.own;
        p.skip_rows = pl.decode ? kDecodeRows : 0;
        p.part_o = part ? plane_o + pl.prefix * rows * a.D : nullptr;
        p.part_l = part ? plane_l + pl.prefix * rows : nullptr;
        // every sequence may end inside a block
        const int blocks = (int)std::min((long long)row_blocks + a.B, (long long)0x7fffffff);
        if ((e = launch_tile_any(a, p, blocks)) != cudaSuccess) return e;
        if (part) {
            MergeParams m{plane_o, plane_l, a.o, a.o_st, a.o_sh, a.lse, a.cu_q, a.kv_lens, a.T, a.B, a.Hq, a.D, a.causal,
                          a.prefix_len, pl.own + pl.prefix, a.page_size, a.max_pages, a.G, p.skip_rows};
            const unsigned grid = (unsigned)((rows + 7) / 8);
            if (a.dtype == DType::BF16) attn_merge_kernel<true><<<grid, 256, 0, a.stream>>>(m);
            else attn_merge_kernel<false><<<grid, 256, 0, a.stream>>>(m);
            if ((e = cudaGetLastError()) != cudaSuccess) return e;
        }
    }
    if (pl.decode) {
        DecodeParts d{};
        d.ctas = pl.ctas;
        d.whole = pl.whole;
        d.only = !pl.tile;
        d.slot_o = slot_o;
        d.slot_l = slot_l;
        if (pl.prefix) {
            d.own_o = plane_o + (pl.planes - 1) * rows * a.D;
            d.own_l = plane_l + (pl.planes - 1) * rows;
            d.pre_o = plane_o;
            d.pre_l = plane_l;
            d.prefix_splits = pl.prefix;
        }
        if ((e = launch_attn_decode(a, d)) != cudaSuccess) return e;
        if (!pl.whole || pl.prefix) e = launch_attn_join(a, d);
    }
    return e;
}

}  // namespace hq
