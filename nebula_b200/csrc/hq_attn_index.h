// hq_attn_index.h -- which rows, keys and pages a sequence has.  The numbers come
// from the caller's device arrays, so each is checked before it is used as an
// index; plain functions of their arguments, so that the checks run on the host too.
#pragma once

#ifdef __CUDACC__
#define HQ_HD __host__ __device__ __forceinline__
#else
#define HQ_HD inline
#endif

namespace hq {

// Rows [first, first + n) of sequence s among T rows (cu_q null: row s alone).
HQ_HD bool seq_rows(const int* cu_q, int s, int T, int& first, int& n) {
    if (!cu_q) {
        first = s;
        n = 1;
        return s < T;
    }
    const int c0 = cu_q[s], c1 = cu_q[s + 1];
    first = c0;
    n = c1 - c0;
    return c0 >= 0 && c1 >= c0 && c1 <= T;
}

// A sequence's keys fit its row of the page table.
HQ_HD bool len_ok(int len, int max_pages, int page_size) {
    return len >= 0 && (long long)len <= (long long)max_pages * page_size;
}

HQ_HD bool page_ok(int page, int num_pages) { return page >= 0 && page < num_pages; }

// Keys that row i of n sees of len: all, or those up to its own place.
HQ_HD int keys_seen(int len, int n, int i, int causal) {
    if (!causal) return len;
    const int x = len - n + i + 1;
    return x < 0 ? 0 : x;
}

// Tiles of `unit` keys that hold `keys` of them, which may be the largest int.
HQ_HD int key_tiles(int keys, int unit) { return keys / unit + (keys % unit != 0); }

// A row that sees `own` keys of its sequence and all `prefix` before them sees one.
HQ_HD bool sees_any(int own, int prefix) { return own > 0 || prefix > 0; }

}  // namespace hq
