// Paged K/V caches: where a slot lives in the pool, and which rows and slots a sequence has.  Every
// index that comes from device memory (page tables, lengths, slot and position lists) passes through
// these functions, which answer with something inside the buffers, or with "none", whatever it holds.
#pragma once
#include <stdint.h>

#if defined(__HIP__)
#define ICUA_HD __host__ __device__ __forceinline__
#else
#define ICUA_HD inline
#endif

namespace icua {

constexpr int PAGED_TILE = 16;  // slots of a matrix-core tile; pages are whole tiles

struct PageMap {
    int n_pages, n_kv, page_slots;
};

// Rows of the pool's K (or V) matrix: [page][KV head][slot].  Both functions give the row of KV head
// 0 (head g: + g * page_slots), or -1.
ICUA_HD int32_t page_row(const PageMap& m, int32_t page, int32_t slot_in_page) {
    if (page < 0 || page >= m.n_pages) return -1;
    return page * (m.n_kv * m.page_slots) + slot_in_page;
}
// Pool slots are numbered page * page_slots + slot in the page.
ICUA_HD int32_t pool_slot_row(const PageMap& m, int32_t slot) {
    if (slot < 0) return -1;
    const int32_t page = (int32_t)((uint32_t)slot / (uint32_t)m.page_slots);
    return page_row(m, page, slot - page * m.page_slots);
}
// Slot `slot` (>= 0) of a sequence with this row of the page table.
ICUA_HD int32_t seq_slot_row(const PageMap& m, const int32_t* table, int table_width, int32_t slot) {
    const int32_t i = (int32_t)((uint32_t)slot / (uint32_t)m.page_slots);
    if (i >= table_width) return -1;
    return page_row(m, table[i], slot - i * m.page_slots);
}

// New tokens t0 .. t0 + n_q - 1 of a sequence, which has n_kv slots; token i sees slots up to
// n_kv - n_q + i (none where that is negative).
struct SeqSpan {
    int t0, n_q, n_kv;
};
ICUA_HD SeqSpan seq_span(const int32_t* q_start, const int32_t* kv_len, int s, int n_tokens, int max_kv) {
    int t0 = q_start[s], t1 = q_start[s + 1], n = kv_len[s];
    t0 = t0 < 0 ? 0 : t0 > n_tokens ? n_tokens : t0;
    t1 = t1 < t0 ? t0 : t1 > n_tokens ? n_tokens : t1;
    n = n < 0 ? 0 : n > max_kv ? max_kv : n;
    return {t0, t1 - t0, n};
}

}  // namespace icua
