// yl_paged.h -- where a row stands and where a position lies in a paged cache:
// the index arithmetic of the paged kernels, free of device code so that it
// can be run (and its bounds checked) on the host as well.
//
// Lengths, row starts and page tables come from device memory and are not
// known to the host that launches; every value that becomes an address goes
// through these functions, which map anything out of range to "nothing there".
#pragma once

#include <stddef.h>
#include <stdint.h>

#if defined(__HIPCC__)
#define YL_HD __host__ __device__ __forceinline__
#else
#define YL_HD inline
#endif

namespace yl {

struct PagedArgs {
    void* keys; void* values;        // [n_pages][n_kv][page][hd]
    int n_pages, page_shift, n_kv, hd;
    int n_seqs, n_rows, max_pages;
    const int32_t* table;            // [n_seqs][max_pages]
    const uint32_t* kv_len;          // [n_seqs]
    const uint32_t* row_start;       // [n_seqs + 1] or null
    int prefix_len;
    const int32_t* prefix_pages;
    int n_heads;
};

// Rows [first, end) of sequence s (empty where the starts do not ascend).
YL_HD void paged_rows(const PagedArgs& a, int s, int* first, int* end) {
    if (!a.row_start) { *first = s; *end = s + 1; return; }
    const uint32_t n = (uint32_t)a.n_rows;
    const uint32_t f = a.row_start[s], e = a.row_start[s + 1];
    *first = (int)(f < n ? f : n);
    *end = (int)(e < n ? e : n);
    if (*end < *first) *end = *first;
}

// The sequence of a row, -1 for a row outside all of them.
YL_HD int paged_seq_of_row(const PagedArgs& a, int row) {
    if (!a.row_start) return row < a.n_seqs ? row : -1;
    int lo = 0, hi = a.n_seqs;       // row_start[lo] <= row once lo > 0, row_start[hi] > row while hi < n_seqs
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (a.row_start[mid + 1] <= (uint32_t)row) lo = mid + 1; else hi = mid;
    }
    if (lo >= a.n_seqs) return -1;
    return a.row_start[lo] <= (uint32_t)row ? lo : -1;
}

// Position of a row whose sequence ends (kv_len) with row end - 1; negative: none.
YL_HD int64_t paged_row_pos(uint32_t kv_len, int end, int row) { return (int64_t)kv_len - (int64_t)(end - row); }

// Positions that sequences can hold: the prefix and every table entry's page.
YL_HD int64_t paged_capacity(const PagedArgs& a) { return (int64_t)a.prefix_len + ((int64_t)a.max_pages << a.page_shift); }

// How many positions, from 0 on, a row at position pos may attend to.
YL_HD int paged_limit(const PagedArgs& a, int64_t pos) {
    const int64_t cap = paged_capacity(a);
    const int64_t n = pos + 1;
    return (int)(n <= 0 ? 0 : n < cap ? n : cap);
}

// The page entry `i` names, or -1.
YL_HD int paged_page(int32_t entry, int n_pages) { return (uint32_t)entry < (uint32_t)n_pages ? entry : -1; }

// Element offset of (page, kv head, slot): 64 bits, a pool may hold more than 2^31 elements.
YL_HD size_t paged_offset(const PagedArgs& a, int page, int kvh, int slot) {
    return (((((size_t)page * a.n_kv + kvh) << a.page_shift) + slot)) * (size_t)a.hd;
}

// The page and slot of position pos (0 <= pos < capacity) of sequence s; false where nothing is held.
YL_HD bool paged_place(const PagedArgs& a, int s, int64_t pos, int* page, int* slot) {
    const bool shared = pos < a.prefix_len;
    const int64_t i = shared ? pos : pos - a.prefix_len;
    const int64_t e = i >> a.page_shift;
    if (pos < 0 || (!shared && e >= a.max_pages)) return false;
    *slot = (int)(i & ((1 << a.page_shift) - 1));
    *page = paged_page(shared ? a.prefix_pages[e] : a.table[(size_t)s * a.max_pages + e], a.n_pages);
    return *page >= 0;
}

#if defined(YALLMA3_H)
// The kernels' arguments from a caller's descriptions; YL_OK, or the refusal.
yl_status paged_args(const yl_paged_cache* c, const yl_paged_batch* b, uint32_t n_heads, PagedArgs* a);
#endif

}  // namespace yl
