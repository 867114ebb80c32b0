// hq_attn_tile.cu -- attention of many rows on the tensor cores: whole prompts,
// prompt chunks over the paged cache, and a prefix that a batch shares.
//
// The rows of a key/value head are its sequence's tokens times the G query heads
// that share it, row r being head r % G of token r / G: a tile's rows read the
// same keys, so one pass over K and V serves all of them, and few rows of the
// causal triangle's edge are wasted.  A tile of 128 rows holds as many tokens as fit
// with all their G heads, so that it is one box of a tensor map (G = 5 leaves 3 rows
// idle); one CTA takes two tiles and walks the keys 128 at a time:
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
// CTAs stay on their SM: warp 0 takes the next block of the grid and works out its
// rows and keys while the others are on the current one; the next block's Q and first
// keys are loaded, and its first S computed, while this one's output is written.
// Where there are more blocks than SMs it asks the launch hardware for the next
// (cluster launch control), so that CTAs share them as they get done; else every CTA
// has its own, and blocks that the lengths leave without rows cost nothing.
//   warp 0        the blocks, and their loads: Q, and one TMA box per 64 dims and up to
//                 128 keys of a page (page numbers from the table), K and V tiles
//                 alternate in a ring
//   warp 1        issues the MMAs; owns the tensor memory
//   warps 2, 3    V tiles that some row does not see in full: rows behind the last
//                 key are zeroed (0 x NaN would reach the sum), and values that
//                 are not finite are taken out and noted, to be put back into the
//                 rows that see them
//   warps 4-7, 8-11  softmax and output of tile 0, tile 1: thread = row = lane
//                 of tensor memory
// Bound: the tensor cores and the exponentials (16 a clock and SM) alike take
// 1024 cycles for a tile's 128 rows x 128 keys x 128 dims.
// Work is split over the keys when there are few rows: every split writes its
// normalised fp32 output and log2 of its sum, merged by attn_merge_kernel.
// Every wait is bounded: after one that gave up all roles run to the end of their
// block without waiting, and take no other.
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
    static constexpr int kStages = DP == 128 ? 4 : 8;
    static constexpr int kOut = 2 * kTile + kStages * kTile;  // Q, the ring, then 4 KB of output a softmax warp
    static constexpr int kShared = kOut + 8 * 4096;           // and TileShared
};

struct alignas(64) TileParams {
    CUtensorMap q_map;         // {dim, head, token}: a box is the rows of a tile
    CUtensorMap k_map, v_map;  // {dim, token, head, page}
    void* o;
    long long o_st, o_sh;
    float* lse;
    float* part_o;  // [split][T * Hq][D] and [split][T * Hq]; null: out is written
    float* part_l;
    const int* cu_q;
    const int* table;
    long long table_stride;
    const int* kv_lens;
    int T, B, Hq, Hk, G, D;
    int tile_tokens;  // tokens of a tile: 128 / G
    int causal;
    float scale_log2;
    int page_size, box_rows, num_pages, max_pages;  // page_size 0: packed rows
    int page_shift, box_shift;                      // their base-2 logarithms
    int prefix_len;                                 // > 0: all T rows over the pages table[0..]
    int blocks, splits;  // the grid: row blocks x Hk x splits
    int ask;        // blocks are shared out by cluster launch control
    int ctas;       // else: at most
    int overlap;    // launched while the kernel before it runs
    int skip_rows;  // sequences of at most this many rows (tokens x G) are not this kernel's
    unsigned* err;
};

// A block of rows and its share of the keys.
struct Item {
    int first, n, len;       // the sequence: first row (token), tokens, keys
    const int* table;        // its pages
    int token0, hk, split;   // first token of the block
    int ni[2];               // key tiles of each row tile
    int k_first, m_first;    // first key; first tile in which a row does not see every key
    int stop;                // no more blocks
};

struct TileShared {
    uint64_t full[8], empty[8], q_full[2], q_read[2], s_full[2], p_full[2][2], o_full[2], v_req, v_clean;
    uint64_t item_full[2], item_empty[2], next;
    uint4 next_block;
    Item item[2];
    uint32_t tmem;
    // first key, counted from the block's first masked tile, whose value in a dim is
    // NaN, +Inf, -Inf; 0xFFFF: none (masked tiles span less than 512 keys)
    int any_bad[2];
    int gave_up;
    uint16_t bad[2][3][128];
};

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

// All 128 columns of this warp's lanes, in four loads; the wait is part of the last
// statement, which takes all registers, so nothing that uses them can be moved
// before it.
__device__ __forceinline__ void tmem_ld128_now(uint32_t taddr, float (&f)[128]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]), "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31])
                 : "r"(taddr + 0u) : "memory");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(f[32]), "=f"(f[33]), "=f"(f[34]), "=f"(f[35]), "=f"(f[36]), "=f"(f[37]), "=f"(f[38]), "=f"(f[39]), "=f"(f[40]), "=f"(f[41]), "=f"(f[42]), "=f"(f[43]), "=f"(f[44]), "=f"(f[45]), "=f"(f[46]), "=f"(f[47]), "=f"(f[48]), "=f"(f[49]), "=f"(f[50]), "=f"(f[51]), "=f"(f[52]), "=f"(f[53]), "=f"(f[54]), "=f"(f[55]), "=f"(f[56]), "=f"(f[57]), "=f"(f[58]), "=f"(f[59]), "=f"(f[60]), "=f"(f[61]), "=f"(f[62]), "=f"(f[63])
                 : "r"(taddr + 32u) : "memory");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(f[64]), "=f"(f[65]), "=f"(f[66]), "=f"(f[67]), "=f"(f[68]), "=f"(f[69]), "=f"(f[70]), "=f"(f[71]), "=f"(f[72]), "=f"(f[73]), "=f"(f[74]), "=f"(f[75]), "=f"(f[76]), "=f"(f[77]), "=f"(f[78]), "=f"(f[79]), "=f"(f[80]), "=f"(f[81]), "=f"(f[82]), "=f"(f[83]), "=f"(f[84]), "=f"(f[85]), "=f"(f[86]), "=f"(f[87]), "=f"(f[88]), "=f"(f[89]), "=f"(f[90]), "=f"(f[91]), "=f"(f[92]), "=f"(f[93]), "=f"(f[94]), "=f"(f[95])
                 : "r"(taddr + 64u) : "memory");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%128];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=f"(f[96]), "=f"(f[97]), "=f"(f[98]), "=f"(f[99]), "=f"(f[100]), "=f"(f[101]), "=f"(f[102]), "=f"(f[103]), "=f"(f[104]), "=f"(f[105]), "=f"(f[106]), "=f"(f[107]), "=f"(f[108]), "=f"(f[109]), "=f"(f[110]), "=f"(f[111]), "=f"(f[112]), "=f"(f[113]), "=f"(f[114]), "=f"(f[115]), "=f"(f[116]), "=f"(f[117]), "=f"(f[118]), "=f"(f[119]), "=f"(f[120]), "=f"(f[121]), "=f"(f[122]), "=f"(f[123]), "=f"(f[124]), "=f"(f[125]), "=f"(f[126]), "=f"(f[127]),
                   "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7]), "+f"(f[8]), "+f"(f[9]), "+f"(f[10]), "+f"(f[11]), "+f"(f[12]), "+f"(f[13]), "+f"(f[14]), "+f"(f[15]), "+f"(f[16]), "+f"(f[17]), "+f"(f[18]), "+f"(f[19]), "+f"(f[20]), "+f"(f[21]), "+f"(f[22]), "+f"(f[23]), "+f"(f[24]), "+f"(f[25]), "+f"(f[26]), "+f"(f[27]), "+f"(f[28]), "+f"(f[29]), "+f"(f[30]), "+f"(f[31]), "+f"(f[32]), "+f"(f[33]), "+f"(f[34]), "+f"(f[35]), "+f"(f[36]), "+f"(f[37]), "+f"(f[38]), "+f"(f[39]), "+f"(f[40]), "+f"(f[41]), "+f"(f[42]), "+f"(f[43]), "+f"(f[44]), "+f"(f[45]), "+f"(f[46]), "+f"(f[47]), "+f"(f[48]), "+f"(f[49]), "+f"(f[50]), "+f"(f[51]), "+f"(f[52]), "+f"(f[53]), "+f"(f[54]), "+f"(f[55]), "+f"(f[56]), "+f"(f[57]), "+f"(f[58]), "+f"(f[59]), "+f"(f[60]), "+f"(f[61]), "+f"(f[62]), "+f"(f[63]), "+f"(f[64]), "+f"(f[65]), "+f"(f[66]), "+f"(f[67]), "+f"(f[68]), "+f"(f[69]), "+f"(f[70]), "+f"(f[71]), "+f"(f[72]), "+f"(f[73]), "+f"(f[74]), "+f"(f[75]), "+f"(f[76]), "+f"(f[77]), "+f"(f[78]), "+f"(f[79]), "+f"(f[80]), "+f"(f[81]), "+f"(f[82]), "+f"(f[83]), "+f"(f[84]), "+f"(f[85]), "+f"(f[86]), "+f"(f[87]), "+f"(f[88]), "+f"(f[89]), "+f"(f[90]), "+f"(f[91]), "+f"(f[92]), "+f"(f[93]), "+f"(f[94]), "+f"(f[95])
                 : "r"(taddr + 96u) : "memory");
}

// 32 columns, likewise.
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

__device__ __forceinline__ void tmem_ld16_now(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// 16 columns from registers to this warp's lanes.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Asks for the next block of the grid that no CTA has begun (16 bytes into `to`,
// counted on `bar`); its index, or -1 if there is none.
__device__ __forceinline__ void next_block_request(void* to, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(to)),
                 "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ int next_block_answer(const void* at) {
    const uint4 v = lds128(smem_u32(at));
    uint32_t got, x;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t.reg .b64 lo, hi;\n\t.reg .b32 y, z, w;\n\t"
        "mov.b64 lo, {%2, %3};\n\tmov.b64 hi, {%4, %5};\n\tmov.b128 h, {lo, hi};\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, h;\n\t}"
        : "=r"(got), "=r"(x)
        : "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
    return got ? (int)x : -1;
}

// The sequence and 256-row block with the number `want`: the blocks of all sequences
// by their place in their sequence, the last places first (under a causal mask they
// have the most keys, and the CTAs end together when the longest work comes first;
// 12 prompts of 172 to 1500 tokens took a fifth longer in the order of the sequences).
// -1: there are fewer blocks.  One warp; every lane returns the same.  It walks all
// sequences for each step of the search, behind the other block's work as long as there
// are few: prompts of 4 rows each, 40 heads on 8 of 128, take 33 us for 64 of them, 132
// for 256, 1450 for 1024 and 22500 for 4096.
__device__ __forceinline__ int find_block(const TileParams& p, int want, int& block) {
    const int lane = threadIdx.x & 31;
    auto blocks_of = [&](int s) {  // n * G fits: n_tokens * n_heads does
        int first = 0, n = 0;
        if (s >= p.B) return 0;
        bool ok = seq_rows(p.cu_q, s, p.T, first, n);
        if (ok && p.page_size) ok = len_ok(p.kv_lens[s], p.max_pages, p.page_size);
        if (!ok) bad_index(p.err);
        return ok && n * p.G > p.skip_rows ? (int)((unsigned)(n + 2 * p.tile_tokens - 1) / (unsigned)(2 * p.tile_tokens)) : 0;
    };
    const int mine = blocks_of(lane);  // the first 32 sequences'
    // blocks with a place below b
    auto below = [&](int b) {
        int sum = min(mine, b);
#pragma unroll 1
        for (int s = lane + 32; s < p.B; s += 32) sum += min(blocks_of(s), b);
        return __reduce_add_sync(~0u, sum);
    };
    int most = mine;
#pragma unroll 1
    for (int s = lane + 32; s < p.B; s += 32) most = max(most, blocks_of(s));
    most = __reduce_max_sync(~0u, most);
    int rank = below(most) - 1 - want;
    if (rank < 0) return -1;
    int lo = 0, hi = most;  // below(lo) <= rank < below(hi)
#pragma unroll 1
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (below(mid) <= rank) lo = mid;
        else hi = mid;
    }
    block = lo;
    if (lo > 0) rank -= below(lo);
    // the sequence with that rank among those that have such a block
#pragma unroll 1
    for (int s0 = 0; s0 < p.B; s0 += 32) {
        const bool has = (s0 ? blocks_of(s0 + lane) : mine) > lo;
        const unsigned all = __ballot_sync(~0u, has);
        const unsigned hit = __ballot_sync(~0u, has && __popc(all & ((1u << lane) - 1u)) == rank);
        if (hit) return s0 + __ffs(hit) - 1;
        rank -= __popc(all);
    }
    return -1;
}

// Block `index` of the grid: row blocks as find_block numbers them, then key/value
// heads, then key splits.
__device__ __forceinline__ bool make_item(const TileParams& p, int index, Item& it) {
    const int split = index % p.splits, rest = index / p.splits;
    it.hk = rest % p.Hk;
    it.split = split;
    int block = rest / p.Hk, seq = 0;
    if (p.prefix_len) {
        it.first = 0;
        it.n = p.T;
        it.len = p.prefix_len;
        it.table = p.table;
    } else {
        seq = find_block(p, block, block);
        if (seq < 0) return false;
        seq_rows(p.cu_q, seq, p.T, it.first, it.n);
        it.len = p.page_size ? p.kv_lens[seq] : it.n;
        it.table = p.table + seq * p.table_stride;
    }
    const int causal = p.causal && !p.prefix_len, tile = p.tile_tokens;
    it.token0 = block * 2 * tile;
    auto seen = [&](int token) { return keys_seen(it.len, it.n, min(token, it.n - 1), causal); };
    const int end1 = key_tiles(seen(it.token0 + 2 * tile - 1), kKeys), end0 = key_tiles(seen(it.token0 + tile - 1), kKeys);
    const int a = end1 * split / p.splits, b = end1 * (split + 1) / p.splits;  // end1 <= 2^24, splits <= 32
    it.ni[0] = max(0, min(b, end0) - a);
    it.ni[1] = it.token0 + tile < it.n ? b - a : 0;
    it.k_first = a * kKeys;
    it.m_first = max(0, seen(it.token0) / kKeys - a);
    it.stop = 0;
    return true;
}

// D (tensor memory) [+]= A x B: A from shared memory, A from tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}

// One lane of the warp (all lanes call it together).
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e)::"memory");
    return e != 0;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {  // (x, y) = (x, y) a + b
    asm("{\n\t.reg .b64 v, p, q;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 p, {%2, %2};\n\tmov.b64 q, {%3, %3};\n\t"
        "fma.rn.f32x2 v, v, p, q;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {  // (x, y) += (a, b)
    asm("{\n\t.reg .b64 v, p;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 p, {%2, %3};\n\tadd.rn.f32x2 v, v, p;\n\t"
        "mov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}

// A warpgroup's share of the registers that the block was launched with (168 a
// thread): 72 + 2 x 216 = 3 x 168.
constexpr int kRegsLoad = 72, kRegsSoftmax = 216;
template <int N>
__device__ __forceinline__ void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Takes the values of v (dims d .. d + 7 of key `key`) that are not finite out and
// notes them.
template <bool kBF16>
__device__ __noinline__ void take_out(uint16_t (*bad)[128], int d, int key, uint4& v) {
    constexpr uint32_t kExp = kBF16 ? 0x7F80u : 0x7C00u;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    for (int e = 0; e < 8; ++e) {
        const int sh = 16 * (e & 1);
        const uint32_t h = w[e >> 1] >> sh & 0xFFFFu;
        if ((h & kExp) != kExp) continue;
        const int kind = (h & 0x7FFFu) != kExp ? 0 : (h & 0x8000u) ? 2 : 1;
        unsigned* word = reinterpret_cast<unsigned*>(&bad[kind][d + (e & ~1)]);
        unsigned old = *word;
        while ((int)(old >> sh & 0xFFFFu) > key) {
            const unsigned seen = atomicCAS(word, old, (old & ~(0xFFFFu << sh)) | (unsigned)key << sh);
            if (seen == old) break;
            old = seen;
        }
        w[e >> 1] &= ~(0xFFFFu << sh);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
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

    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* qs = smem;
    uint8_t* ring = qs + 2 * L::kTile;
    TileShared& sh = *reinterpret_cast<TileShared*>(smem + L::kShared);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_launch_dependents();
    if (warp == 0) {
        if (lane < 3) tmap_prefetch(lane == 0 ? &p.q_map : lane == 1 ? &p.k_map : &p.v_map);
    } else if (warp == 1) {
        if (lane == 0) {
            for (int i = 0; i < S; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1);
            }
            for (int t = 0; t < 2; ++t) {
                mbar_init(&sh.q_full[t], 1);
                mbar_init(&sh.q_read[t], 1);
                mbar_init(&sh.s_full[t], 1);
                mbar_init(&sh.p_full[t][0], 128);
                mbar_init(&sh.p_full[t][1], 128);
                mbar_init(&sh.o_full[t], 1);
                mbar_init(&sh.item_full[t], 1);
                mbar_init(&sh.item_empty[t], 11);  // all warps but warp 0
            }
            mbar_init(&sh.v_req, 1);
            mbar_init(&sh.v_clean, 64);
            mbar_init(&sh.next, 1);
            fence_mbarrier_init();
            fence_async_smem();
        }
        __syncwarp();
        tmem_alloc(&sh.tmem, kTmemCols);
        tmem_relinquish();
    } else if (warp == 2) {
        for (int i = lane; i < 2 * 3 * 64; i += 32) reinterpret_cast<unsigned*>(&sh.bad[0][0][0])[i] = ~0u;
        if (lane < 2) sh.any_bad[lane] = 0;
        if (lane == 2) sh.gave_up = 0;
    }
    auto ready = [&] {
        fence_async_smem();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    };
    if (warp != 0) {  // warp 0 works its first block out before it comes to this barrier
        // rows of a tile behind its last token's
        for (int i = p.tile_tokens * p.G * 8 + (int)threadIdx.x - 32; i < kRows * 8; i += kThreads - 32)
#pragma unroll
            for (int b = 0; b < 2 * L::kBlk; ++b) sts128(smem_u32(qs) + b * L::kBlkBytes + i * 16, make_uint4(0u, 0u, 0u, 0u));
        ready();
    }
    const uint32_t tmem = warp != 0 ? sh.tmem : 0u;
    auto wait = [&](uint64_t* bar, uint32_t parity) { wait_bar(bar, parity & 1u, &sh.gave_up, p.err); };
    auto gave_up = [&] { return *reinterpret_cast<volatile int*>(&sh.gave_up) != 0; };
    // Item k of this CTA is in slot k & 1; false: there is none.
    auto item_wait = [&](int k) {
        wait(&sh.item_full[k & 1], (uint32_t)(k >> 1));
        return !gave_up() && !sh.item[k & 1].stop;
    };

    if (warp == 0) {
        // ----------------------------------------------- blocks and loads
        regs_down<kRegsLoad>();
        const int boxes = kKeys / p.box_rows;
        int index = (int)blockIdx.x, use = 0;
        uint32_t loads[2] = {0, 0};
        int none = INT_MAX;  // blocks from this number on have no rows
        for (int k = 0, asked = 0;; ++asked) {
            Item it;
            const bool found = index < none && make_item(p, index, it);
            if (!found) none = min(none, index);
            if (asked == 0) ready();
            if (p.ask && lane == 0) next_block_request(&sh.next_block, &sh.next);
            __syncwarp();
            if (found) {
                if (k >= 2) wait(&sh.item_empty[k & 1], (uint32_t)((k - 2) >> 1));
                __syncwarp();
                if (sh.any_bad[k & 1]) {
                    for (int i = lane; i < 3 * 64; i += 32) reinterpret_cast<unsigned*>(&sh.bad[k & 1][0][0])[i] = ~0u;
                    __syncwarp();
                }
                if (lane == 0) {
                    sh.any_bad[k & 1] = 0;
                    sh.item[k & 1] = it;
                    mbar_arrive(&sh.item_full[k & 1]);
                }
                __syncwarp();
                ++k;
                const int nt = max(it.ni[0], it.ni[1]);
                // Lane b looks up the page of a tile's box b, a tile ahead; one lane requests all
                // boxes.  (With a box a lane a tile over pages of 16 took 2000 cycles: a
                // request's operands come from uniform registers, so it is lane after lane.)
                const int box = lane;
                auto live_at = [&](int k0) { return min(boxes, ((it.len - k0 - 1) >> p.box_shift) + 1); };
                auto page_at = [&](int k0) {
                    return p.page_size && box < live_at(k0) ? __ldg(it.table + ((k0 + (box << p.box_shift)) >> p.page_shift)) : 0;
                };
                int page = 0, next_page = nt > 0 ? page_at(it.k_first) : 0;
#pragma unroll 1
                for (int i = 0; i < 2 * nt; ++i, ++use) {  // K, V of tile 0, of tile 1, ...
                    if (i == 1) {  // Q, once the block before has read its own; its first K may come before
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (it.ni[t] <= 0) continue;
                            if (loads[t] > 0) wait(&sh.q_read[t], loads[t] - 1);
                            ++loads[t];
                            if (lane == 0) mbar_arrive_expect_tx(&sh.q_full[t], (uint32_t)(L::kBlk * p.tile_tokens * p.G * 128));
                            __syncwarp();
                            if (lane < L::kBlk)
                                tma_load_3d(qs + t * L::kTile + lane * L::kBlkBytes, &p.q_map, lane * 64, it.hk * p.G,
                                            it.first + it.token0 + t * p.tile_tokens, &sh.q_full[t]);
                        }
                    }
                    const int k0 = it.k_first + (i >> 1) * kKeys, slot = use % S;
                    const int live = live_at(k0);
                    if (!(i & 1)) {
                        page = next_page;
                        if (p.page_size && box < live && !page_ok(page, p.num_pages)) {
                            bad_index(p.err);
                            page = p.num_pages;  // out of range: the box reads zeros
                        }
                        if (i + 2 < 2 * nt) next_page = page_at(k0 + kKeys);
                    }
                    wait(&sh.empty[slot], ((uint32_t)(use / S) & 1u) ^ 1u);
                    uint8_t* dst = ring + slot * L::kTile;
                    if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], (uint32_t)(live * L::kBlk * p.box_rows * 128));
                    __syncwarp();
#pragma unroll 1
                    for (int b = 0; b < live; ++b) {
                        const int at = b << p.box_shift, pg = __shfl_sync(~0u, page, b);
                        const int token = p.page_size ? (k0 + at) & (p.page_size - 1) : it.first + k0 + at;
                        if (elect_one()) {
#pragma unroll
                            for (int blk = 0; blk < L::kBlk; ++blk)
                                tma_load_4d(dst + blk * L::kBlkBytes + at * 128, i & 1 ? &p.v_map : &p.k_map, blk * 64, token,
                                            it.hk, pg, &sh.full[slot]);
                        }
                        __syncwarp();
                    }
                }
            }
            if (p.ask) {
                wait(&sh.next, (uint32_t)asked);
                __syncwarp();
                index = gave_up() ? -1 : next_block_answer(&sh.next_block);
            } else {
                const bool last = index >= p.blocks * p.Hk * p.splits - (int)gridDim.x;
                index = last || !found || gave_up() ? -1 : index + (int)gridDim.x;
            }
            if (index < 0) {
                if (k >= 2) wait(&sh.item_empty[k & 1], (uint32_t)((k - 2) >> 1));
                __syncwarp();
                if (lane == 0) {
                    sh.item[k & 1].stop = 1;
                    mbar_arrive(&sh.item_full[k & 1]);
                }
                break;
            }
            if (lane == 0) fence_async_smem();  // the answer is read before the next one is written
        }
        __syncwarp();
        // Every stage filled here has been consumed (its commits have landed) before exit.
#pragma unroll 1
        for (int j = max(0, use - S); j < use; ++j) mbar_wait(&sh.empty[j % S], (uint32_t)(j / S) & 1u, p.err);
        for (int t = 0; t < 2; ++t)
            if (loads[t] > 0) mbar_wait(&sh.q_read[t], (loads[t] - 1) & 1u, p.err);
    } else if (warp == 1) {
        // ----------------------------------------------------------- MMAs
        // The whole warp walks the loops, on values that the compiler can see to be
        // the same in all lanes, and one lane issues: operands then stay in uniform
        // registers.  (One thread in a branch of its own took 60 to 90 cycles an MMA,
        // more than the MMA.)
        regs_down<kRegsLoad>();
        auto same = [](int x) { return __shfl_sync(~0u, x, 0); };
        const uint32_t tm = (uint32_t)same((int)tmem), ring_a = smem_u32(ring), q_a = smem_u32(qs);
        uint32_t use = 0, cleaned = 0, loaded[2] = {0, 0}, done[2] = {0, 0};
        for (int k = 0; item_wait(k); ++k) {
            const int n0 = same(sh.item[k & 1].ni[0]), n1 = same(sh.item[k & 1].ni[1]), m_first = same(sh.item[k & 1].m_first);
            const int nt = max(n0, n1);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[k & 1]);
            // Step i: O += P V of key tile i, S = Q K^T of tile i + 1, for both row tiles.
#pragma unroll 1
            for (int i = -1; i < nt; ++i) {
                const uint32_t vu = use + 2 * i + 1, ku = vu + 1;
                const uint32_t va = ring_a + (vu % S) * L::kTile, ka = ring_a + (ku % S) * L::kTile;
                if (i >= 0) {
                    wait(&sh.full[vu % S], vu / S);
                    if (i >= m_first) wait(&sh.v_clean, cleaned++);
                }
                if (i + 1 < nt) wait(&sh.full[ku % S], ku / S);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int my = t ? n1 : n0;
                    const uint32_t sp = tm + 128u * t, op = tm + kColO + (uint32_t)DP * t;
                    if (i >= 0 && i < my) {
                        // P comes in halves of 64 keys
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            wait(&sh.p_full[t][h], done[t]);
                            __syncwarp();
                            tc_fence_after();
                            if (elect_one()) {
                                const uint64_t vd = sw128_mn_desc(va);
#pragma unroll
                                for (int j = 4 * h; j < 4 * h + 4; ++j)
                                    mma_ts(op, sp + 8u * j, vd + j * (2048 >> 4), kIdescO, (i | j) != 0);
                                if (h) umma_commit(&sh.o_full[t]);
                            }
                            __syncwarp();
                        }
                        ++done[t];
                    }
                    if (i + 1 < my) {
                        if (i < 0) {
                            wait(&sh.q_full[t], loaded[t]++);
                            __syncwarp();
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t qd = sw128_kmajor_desc(q_a + t * L::kTile), kd = sw128_kmajor_desc(ka);
#pragma unroll
                            for (int j = 0; j < DP / 16; ++j) {
                                const uint32_t off = ((j >> 2) * L::kBlkBytes + (j & 3) * 32) >> 4;
                                mma_ss(sp, qd + off, kd + off, kIdescS, j != 0);
                            }
                            umma_commit(&sh.s_full[t]);
                            if (i + 2 == my) umma_commit(&sh.q_read[t]);
                        }
                        __syncwarp();
                    }
                }
                if (elect_one()) {
                    if (i >= 0) umma_commit(&sh.empty[vu % S]);
                    if (i + 1 < nt) {
                        umma_commit(&sh.empty[ku % S]);
                        if (i + 1 >= m_first) mbar_arrive(&sh.v_req);
                    }
                }
                __syncwarp();
            }
            use += 2 * nt;
        }
    } else if (warp < 4) {
        // ----------------------------------------- V tiles under a mask
        // v_req comes once the tile's K has been used, so V's stage is in this use's
        // phase or the one before it, and stays until v_clean.
        regs_down<kRegsLoad>();
        uint32_t use = 0, asked = 0;
        constexpr int C = DP / 8, RS = 64 / C;  // 16-byte chunks of a row, rows of a step
        const int x = threadIdx.x - 64, c = x % C;
        for (int k = 0; item_wait(k); ++k) {
            const Item it = sh.item[k & 1];
            const int nt = max(it.ni[0], it.ni[1]);
            const int causal = p.causal && !p.prefix_len;
            const int lim_min = keys_seen(it.len, it.n, it.token0, causal);
            const int lim_max = keys_seen(it.len, it.n, min(it.token0 + 2 * p.tile_tokens, it.n) - 1, causal);
            const int base = it.k_first + it.m_first * kKeys;
#pragma unroll 1
            for (int i = it.m_first; i < nt; ++i) {
                const uint32_t vu = use + 2 * i + 1;
                wait(&sh.v_req, asked++);
                wait(&sh.full[vu % S], (vu / S));
                __syncwarp();
                const uint32_t vt = smem_u32(ring) + (vu % S) * L::kTile;
                const int k0 = it.k_first + i * kKeys;
                // keys [lo, hi) are seen by some rows only, those behind by none
                const int hi = min(kKeys, lim_max - k0), lo = min(hi, max(0, lim_min - k0));
                // chunk c of row r of a block lies at chunk c ^ (r & 7)
                const uint32_t col = vt + (c >> 3) * L::kBlkBytes;
                auto at = [&](int r) { return col + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
                // Eight rows at a time: a look at each by itself took 5000 cycles a tile, more
                // than its softmax.  (A row behind hi is zeroed below, whatever it holds.)
#pragma unroll 1
                for (int r0 = (lo & ~7) + x / C; r0 < hi; r0 += 8 * RS) {
                    uint32_t any = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) any |= not_finite<kBF16>(lds128(at(min(r0 + j * RS, kKeys - 1))));
                    if (!any) continue;
#pragma unroll 1
                    for (int r = r0; r < min(hi, r0 + 8 * RS); r += RS) {
                        uint4 v = lds128(at(r));
                        if (r < lo || !not_finite<kBF16>(v)) continue;
                        take_out<kBF16>(sh.bad[k & 1], c * 8, k0 + r - base, v);
                        sts128(at(r), v);
                        sh.any_bad[k & 1] = 1;
                    }
                }
#pragma unroll 1
                for (int r = hi + x / C; r < kKeys; r += RS) sts128(at(r), make_uint4(0u, 0u, 0u, 0u));
                fence_async_smem();
                mbar_arrive(&sh.v_clean);
            }
            use += 2 * nt;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[k & 1]);
        }
    } else {
        // --------------------------------------------- softmax and output
        regs_up<kRegsSoftmax>();
        const int t = (warp - 4) >> 2, i0 = (threadIdx.x - 128) & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + 128u * t, to = tmem + lanes + kColO + (uint32_t)DP * t;
        const int causal = p.causal && !p.prefix_len;
        const int tok = i0 / p.G, head0 = i0 - tok * p.G;  // this row's place in a tile
        uint32_t steps = 0;                                // key tiles of this row tile so far
        for (int k = 0; item_wait(k); ++k) {
            float m = -INFINITY, l = 0.f;
            const Item& it = sh.item[k & 1];  // stays until this warp has arrived on item_empty
            const int my = it.ni[t], k_first = it.k_first, m_first = it.m_first;
            // rows behind the last see what it sees
            const int place = min(it.token0 + t * p.tile_tokens + tok, it.n - 1);
            const int lim = keys_seen(it.len, it.n, place, causal);
#pragma unroll 1
            for (int i = 0; i < my; ++i) {
                wait(&sh.s_full[t], steps + i);
                __syncwarp();
                tc_fence_after();
                const int cut = i >= m_first ? lim - (k_first + i * kKeys) : kKeys;  // columns from here on are not seen
                float s[128];
                tmem_ld128_now(ts, s);
                if (i >= m_first) {
#pragma unroll
                    for (int c = 0; c < 128; c += 32)
                        if (cut < c + 32) {
#pragma unroll
                            for (int e = c; e < c + 32; ++e) s[e] = e < cut ? s[e] : -INFINITY;
                        }
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int e = 4; e < 128; ++e) top[e & 3] = fmaxf(top[e & 3], s[e]);
                float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                mx *= p.scale_log2;
                const bool move = mx > m + 8.f;  // also from -inf; a first tile has no O yet
                if (__any_sync(~0u, move && l > 0.f)) {
                    wait(&sh.o_full[t], (steps + i - 1));
                    __syncwarp();
                    tc_fence_after();
                    const float f = move ? ex2(m - mx) : 1.f;
#pragma unroll 1
                    for (int c = 0; c < DP / 16; ++c) {
                        uint32_t w[16];
                        tmem_ld16_now(to + 16u * c, w);
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
                        tmem_st16(to + 16u * c, w);
                    }
                    l *= f;
                }
                if (move) m = mx;
                const float sub = m == -INFINITY ? 0.f : m - kShift;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                auto exponentials = [&](int c) {  // of 32 columns
#pragma unroll
                    for (int e = 32 * c; e < 32 * c + 32; e += 2) {
                        fma2(s[e], s[e + 1], p.scale_log2, -sub);
                        s[e] = ex2(s[e]);
                        s[e + 1] = ex2(s[e + 1]);
                    }
                };
                // P is rounded to V's type, which the MMA asks of both operands: half a step of each
                // weight, 2^-8 (bf16) or 2^-11 (fp16); the sum l keeps the weights as they were. A
                // second MMA with what the rounding left would keep them too, at twice the P V
                // work: the error against 64 bits is 1.15 to 1.4 times that of weights in fp32, as the
                // output's own rounding to the same type is the larger part.
                auto put = [&](int c) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        add2(sum[e & 2], sum[(e & 2) + 1], s[32 * c + e], s[32 * c + e + 1]);
                        w[e / 2] = pack2<kBF16>(s[32 * c + e], s[32 * c + e + 1]);
                    }
                    tmem_st16(ts + 16u * c, w);
                };
                auto hand_over = [&](int half) {
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(&sh.p_full[t][half]);
                };
                // the function unit has the next columns' exponentials while these are stored
                exponentials(0);
                exponentials(1);
                put(0);
                exponentials(2);
                put(1);
                hand_over(0);
                exponentials(3);
                put(2);
                put(3);
                hand_over(1);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            steps += my;
            const int token = it.first + place, head = it.hk * p.G + head0;
            const bool live = tok < p.tile_tokens && it.token0 + t * p.tile_tokens + tok < it.n;
            const size_t hrow = (size_t)token * p.Hq + head;
            const size_t prow = (size_t)it.split * p.T * p.Hq + hrow;
            const int bad_lim = lim - (k_first + m_first * kKeys);
            if (my > 0) {
                wait(&sh.o_full[t], steps - 1);
                __syncwarp();
                tc_fence_after();
            }
            const bool any_bad = sh.any_bad[k & 1] != 0;  // written before v_clean, which every PV waited for
            // l = 0: no key was seen (zeros), or every score was -inf (no softmax: NaN,
            // which a merge settles where other splits have a sum).
            const bool part = p.part_o != nullptr;
            const float inv = l != 0.f ? 1.f / l : (!part && lim > 0 ? NAN : 0.f);
            // 128 bytes of each row at a time go through shared memory, so that a store takes
            // whole lines: a thread's own row in 16-byte stores took 3 us of a block of 8 steps
            // that took 21.
            const uint32_t stage = smem_u32(smem + L::kOut) + (warp - 4) * 4096;
            uint8_t* const to_out = part ? reinterpret_cast<uint8_t*>(p.part_o) : static_cast<uint8_t*>(p.o);
            const long long mine = !live ? -1 : part ? (long long)prow * p.D * 4 : 2 * (token * p.o_st + head * p.o_sh);
            const uint32_t own = stage + lane * 128;  // chunk c of row r lies at chunk c ^ (r & 7)
            // The staged 128 bytes of every row, the dims from `dim` on, `per` in 16 bytes.
            auto flush = [&](int dim, int per) {
                __syncwarp();
                dim += per * (lane & 7);
                uint4 v[8];
                long long off[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = 4 * i + (lane >> 3);
                    v[i] = lds128(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                    off[i] = __shfl_sync(~0u, mine, r);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (off[i] >= 0 && dim < p.D) *reinterpret_cast<uint4*>(to_out + off[i] + dim * (16 / per)) = v[i];
            };
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                float o[32];
                if (my > 0) tmem_ld32_now(to + c, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = my > 0 && l != 0.f ? o[e] * inv : inv;
                if (any_bad) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        if ((int)sh.bad[k & 1][1][c + e] < bad_lim) o[e] += INFINITY;
                        if ((int)sh.bad[k & 1][2][c + e] < bad_lim) o[e] -= INFINITY;
                        if ((int)sh.bad[k & 1][0][c + e] < bad_lim) o[e] = NAN;
                    }
                }
                if (part) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        sts128(own + ((e / 4 ^ (lane & 7)) << 4),
                               make_uint4(__float_as_uint(o[e]), __float_as_uint(o[e + 1]), __float_as_uint(o[e + 2]),
                                          __float_as_uint(o[e + 3])));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        sts128(own + (((c & 32 ? 4 : 0) + e / 8 ^ (lane & 7)) << 4),
                               make_uint4(pack2<kBF16>(o[e], o[e + 1]), pack2<kBF16>(o[e + 2], o[e + 3]),
                                          pack2<kBF16>(o[e + 4], o[e + 5]), pack2<kBF16>(o[e + 6], o[e + 7])));
                }
                if (part) flush(c, 4);
                else if (c & 32) flush(c - 32, 8);
            }
            if (live) {
                const float l2 = l == 0.f ? -INFINITY : m - kShift + log2f(l);
                if (part) p.part_l[prow] = l2;
                else if (p.lse) p.lse[hrow] = l2 * 0.693147180559945309417f;
            }
            __syncwarp();
            tc_fence_before();  // O is read before the next block's first PV, which p_full lets go
            if (lane == 0) mbar_arrive(&sh.item_empty[k & 1]);
        }
    }

    if (p.overlap) pdl_wait();  // what waits for this kernel waits for the one before it, too
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Merges the splits of every row: out = sum_s w_s o_s / sum_s w_s, w_s = 2^(l_s - max l)
// for split s's normalised output o_s and log2 of its sum l_s.  One warp a row and head.
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
    const unsigned row = blockIdx.x * 8 + (threadIdx.x >> 5);
    const size_t rows = (size_t)p.T * p.Hq;  // below 2^31
    const int t = (int)(row / (unsigned)p.Hq), h = (int)(row - (unsigned)t * p.Hq);
    // the row's sequence (while the kernels before this one run: they write none of what
    // this reads); rows of none, and those of the decode kernel, have no partials here
    int seen = -1;
    for (int s0 = 0; s0 < p.B && seen < 0 && row < rows; s0 += 32) {
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
    pdl_wait();
    if (seen < 0) return;
    Row x{};
    x.top = -INFINITY;
    const int d = 4 * lane;
    join_parts(x, p.splits, p.part_o, p.part_l, p.D, d, [&](int s) { return s * rows + row; });
    const float l2 = finish_row(x, sees_any(seen, p.prefix_len));
    if (d < p.D) {
        uint16_t* dst = static_cast<uint16_t*>(p.o) + (size_t)t * p.o_st + (size_t)h * p.o_sh + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<kBF16>(x.acc[0], x.acc[1]), pack2<kBF16>(x.acc[2], x.acc[3]));
    }
    if (p.lse && lane == 0) p.lse[row] = l2 * 0.693147180559945309417f;
}

int ceil_div(long long a, int b) { return (int)((a + b - 1) / b); }

template <bool kBF16, int DP>
cudaError_t launch_tile(const TileParams& p, int dev, cudaStream_t s) {
    constexpr int kSmem = TileLayout<DP>::kShared + (int)sizeof(TileShared);
    static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
    auto fn = attn_tile_kernel<kBF16, DP>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(fn), dev, kSmem);
    if (e != cudaSuccess) return e;
    const long long all = (long long)p.blocks * p.Hk * p.splits;
    if (all > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    const long long grid = p.ask ? all : std::min<long long>(all, p.ctas);
    return launch_overlapped(fn, (unsigned)grid, kThreads, kSmem, s, p.overlap, p);
}

cudaError_t launch_tile_any(const AttnArgs& a, const TileParams& p) {
    if (a.D <= 64)
        return a.dtype == DType::BF16 ? launch_tile<true, 64>(p, a.dev, a.stream) : launch_tile<false, 64>(p, a.dev, a.stream);
    return a.dtype == DType::BF16 ? launch_tile<true, 128>(p, a.dev, a.stream) : launch_tile<false, 128>(p, a.dev, a.stream);
}

cudaError_t q_map(const AttnArgs& a, CUtensorMap* m) {
    const uint64_t any = 16;  // a dimension of one element takes any legal stride
    const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.Hq, (uint64_t)a.T};
    const uint64_t strides[2] = {a.Hq > 1 ? 2 * (uint64_t)a.q_sh : any, a.T > 1 ? 2 * (uint64_t)a.q_st : any};
    const uint32_t box[3] = {64, (uint32_t)a.G, (uint32_t)(kRows / a.G)};
    return make_tmap_16bit(m, a.q, 3, dims, strides, box);
}

// Key splits of `row_blocks` x Hk CTAs over `keys` keys: enough to fill the SMs once,
// at least two key tiles each.  One prompt of 1500 tokens, 5 heads on one: 22.9 us, 28.2
// without splits; 8 rows under a prefix of 1024 keys 14.7, 24.1 without.
int key_splits(int row_blocks, int Hk, int keys, int sms) {
    const long long items = (long long)row_blocks * Hk;
    const int by_keys = ceil_div(keys, kKeys) / 2;
    return (int)std::max(1LL, std::min({(long long)sms / items, (long long)by_keys, 32LL}));
}

}  // namespace

cudaError_t kv_maps(const AttnArgs& a, int box_rows, CUtensorMap* k_map, CUtensorMap* v_map) {
    // A dimension of one element takes any legal stride.
    const uint64_t any = 16;
    const uint64_t tokens = a.page_size ? a.page_size : a.T, pages = a.page_size ? a.num_pages : 1;
    const uint64_t dims[4] = {(uint64_t)a.D, tokens, (uint64_t)a.Hk, pages};
    const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
    auto one = [&](CUtensorMap* m, const void* base, long long st, long long sh, long long sp) {
        const uint64_t strides[3] = {tokens > 1 ? 2 * (uint64_t)st : any, a.Hk > 1 ? 2 * (uint64_t)sh : any,
                                     pages > 1 ? 2 * (uint64_t)sp : any};
        return make_tmap_16bit(m, base, 4, dims, strides, box);
    };
    cudaError_t e = one(k_map, a.k, a.k_st, a.k_sh, a.k_sp);
    return e != cudaSuccess ? e : one(v_map, a.v, a.v_st, a.v_sh, a.v_sp);
}

cudaError_t kv_maps_128(const AttnArgs& a, int box_rows, CUtensorMap* k_map, CUtensorMap* v_map) {
    const uint64_t any = 16;
    const uint64_t dims[5] = {64, (uint64_t)a.page_size, 2, (uint64_t)a.Hk, (uint64_t)a.num_pages};
    const uint32_t box[5] = {64, (uint32_t)box_rows, 2, 1, 1};
    auto one = [&](CUtensorMap* m, const void* base, long long st, long long sh, long long sp) {
        const uint64_t strides[4] = {2 * (uint64_t)st, 128, a.Hk > 1 ? 2 * (uint64_t)sh : any,
                                     a.num_pages > 1 ? 2 * (uint64_t)sp : any};
        return make_tmap_16bit(m, base, 5, dims, strides, box);
    };
    cudaError_t e = one(k_map, a.k, a.k_st, a.k_sh, a.k_sp);
    return e != cudaSuccess ? e : one(v_map, a.v, a.v_st, a.v_sh, a.v_sp);
}

// Blocks of two tiles of n tokens.
static int blocks_of(int n, int G) { return ceil_div(n, 2 * (kRows / G)); }

AttnPlan attn_plan(int T, int B, int max_q, int Hq, int Hk, int D, bool paged, int max_kv, int prefix_len, int sms) {
    AttnPlan pl{};
    max_q = std::max(1, max_q);  // a bound of 0 may be wrong, too: rows of one each still have their kernel
    const int G = Hq / Hk, row_blocks = blocks_of(T, G);
    pl.tile = !paged || (long long)max_q * G > kDecodeRows;
    pl.decode = paged && G <= kDecodeRows && (!pl.tile || B > 1);
    pl.prefix = prefix_len > 0 ? key_splits(row_blocks, Hk, prefix_len, sms) : 0;
    if (pl.decode) pl.dec_rows = !pl.tile ? max_q * G : G <= 8 ? 8 : kDecodeRows;
    // Beside the decode kernel the tiles leave it its share of the SMs (a block counted as
    // three sequences), so that the two run at the same time.  16 streams and a chunk of 64
    // rows over 1500 keys: 36.8 us with all SMs for the tiles first (9 splits), 32.2 with 2
    // splits on 32 SMs, 36.6 with 1 on 16.  Of the sequences at least `big` are the tiles',
    // by their rows.
    pl.tile_blocks = row_blocks;
    pl.tile_sms = sms;
    if (pl.tile && pl.decode) {
        const long long few = (long long)B * (pl.dec_rows / G);
        const int big = (int)std::min<long long>(B, T > few ? ceil_div(T - few, max_q) : 0);
        pl.tile_blocks = std::max(row_blocks, big * blocks_of(std::min(max_q, T), G));
        pl.tile_sms = (int)std::max(1LL, 3LL * pl.tile_blocks * sms / (3LL * pl.tile_blocks + B - big));
    }
    pl.own = pl.tile ? key_splits(pl.tile_blocks, Hk, max_kv, pl.tile_sms) : 0;
    pl.planes = pl.prefix;
    if (pl.tile && pl.own + pl.prefix > 1) pl.planes += pl.own;
    if (pl.decode) {
        pl.dec = decode_plan(B, Hk, max_q, max_kv, sms);
        pl.join = pl.dec.mode == kFlat;
        if (pl.join) pl.slots = (size_t)pl.dec.ctas * 2 * kDecodeRows;
        if (pl.join && pl.prefix) ++pl.planes;
    }
    pl.bytes = ((pl.planes * T * Hq + pl.slots) * (D + 1) * 4 + 255) & ~(size_t)255;
    return pl;
}

cudaError_t launch_attn(const AttnArgs& a) {
    const AttnPlan pl = attn_plan(a.T, a.B, a.max_q, a.Hq, a.Hk, a.D, a.page_size > 0, a.max_kv, a.prefix_len, a.sm_count);
    // workspace: outputs of the planes, of the decode slots, then the sums of both
    const size_t rows = (size_t)a.T * a.Hq;
    float* plane_o = reinterpret_cast<float*>(a.ws);
    float* slot_o = plane_o + pl.planes * rows * a.D;
    float* plane_l = slot_o + pl.slots * a.D;
    float* slot_l = plane_l + pl.planes * rows;

    cudaError_t e = cudaSuccess;
    TileParams p;
    memset(&p, 0, sizeof p);
    if (pl.tile || pl.prefix) {
        p.o = a.o;
        p.o_st = a.o_st;
        p.o_sh = a.o_sh;
        p.lse = a.lse;
        p.cu_q = a.cu_q;
        p.kv_lens = a.kv_lens;
        p.T = a.T;
        p.B = a.B;
        p.Hq = a.Hq;
        p.Hk = a.Hk;
        p.G = a.G;
        p.tile_tokens = kRows / a.G;
        p.D = a.D;
        p.causal = a.causal;
        p.scale_log2 = a.scale * 1.44269504088896340736f;
        p.page_size = a.page_size;
        p.box_rows = a.page_size ? std::min(a.page_size, kKeys) : kKeys;
        while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
        while ((1 << p.box_shift) < p.box_rows) ++p.box_shift;
        p.num_pages = a.num_pages;
        p.max_pages = a.max_pages;
        p.err = a.err;
        if ((e = kv_maps(a, p.box_rows, &p.k_map, &p.v_map)) != cudaSuccess || (e = q_map(a, &p.q_map)) != cudaSuccess) return e;
    }
    const int row_blocks = blocks_of(a.T, a.G);
    if (pl.prefix) {
        TileParams x = p;
        x.prefix_len = a.prefix_len;
        x.table = a.prefix_table;
        x.splits = pl.prefix;
        x.part_o = plane_o;
        x.part_l = plane_l;
        x.blocks = row_blocks;
        x.ask = (long long)row_blocks * a.Hk * x.splits > a.sm_count;
        x.ctas = a.sm_count;
        if ((e = launch_tile_any(a, x)) != cudaSuccess) return e;
    }
    if (pl.tile) {
        const bool part = pl.own + pl.prefix > 1;
        p.table = a.table;
        p.table_stride = a.table_stride;
        p.splits = pl.own;
        p.overlap = pl.prefix > 0;
        p.skip_rows = pl.decode ? pl.dec_rows : 0;
        p.part_o = part ? plane_o + pl.prefix * rows * a.D : nullptr;
        p.part_l = part ? plane_l + pl.prefix * rows : nullptr;
        // every sequence may end inside a block
        p.blocks = (int)std::min((long long)row_blocks + a.B, 0x7fffffffLL);
        const long long ctas = (long long)pl.tile_blocks * a.Hk * p.splits;
        p.ask = ctas > a.sm_count;  // 12 prompts of 172 to 1500 tokens: 46.3 us, 53.0 without
        p.ctas = (int)std::min<long long>(a.sm_count, std::max<long long>(pl.tile_sms, ctas));
        if ((e = launch_tile_any(a, p)) != cudaSuccess) return e;
    }
    if (pl.decode) {
        DecodeParts d{};
        d.plan = pl.dec;
        d.only = !pl.tile;
        d.rows = pl.dec_rows;
        d.overlap = pl.prefix || pl.tile;  // the kernel before it is this call's own
        d.slot_o = slot_o;
        d.slot_l = slot_l;
        if (pl.prefix) {
            if (pl.join) {
                d.own_o = plane_o + (pl.planes - 1) * rows * a.D;
                d.own_l = plane_l + (pl.planes - 1) * rows;
            }
            d.pre_o = plane_o;
            d.pre_l = plane_l;
            d.prefix_splits = pl.prefix;
        }
        if ((e = launch_attn_decode(a, d)) != cudaSuccess) return e;
        if (pl.join && (e = launch_attn_join(a, d)) != cudaSuccess) return e;
    }
    if (pl.tile && pl.own + pl.prefix > 1) {
        MergeParams m{plane_o, plane_l, a.o, a.o_st, a.o_sh, a.lse, a.cu_q, a.kv_lens, a.T, a.B, a.Hq, a.D, a.causal,
                      a.prefix_len, pl.own + pl.prefix, a.page_size, a.max_pages, a.G, p.skip_rows};
        auto fn = a.dtype == DType::BF16 ? attn_merge_kernel<true> : attn_merge_kernel<false>;
        e = launch_overlapped(fn, (unsigned)((rows + 7) / 8), 256, 0, a.stream, true, m);
    }
    return e;
}

}  // namespace hq
