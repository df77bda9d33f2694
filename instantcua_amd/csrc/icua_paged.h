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

// Forms of the attention: every slot up to a token's own; a window of the last ones and a few first ones; sequences of
// a group share their first slots.
enum PagedForm { PAGED_ALL = 0, PAGED_WINDOW = 1, PAGED_PREFIX = 2 };

// The slots that a kernel goes through, numbered without the gap of those that it skips: number v stands for slot v,
// from `from` on for v + skip.
struct SlotGap {
    int from, skip;
};
ICUA_HD int32_t gap_slot(const SlotGap& g, int32_t v) { return v < g.from ? v : v + g.skip; }

// Window: rows whose own slots are first_own or later see slots below `sinks` and, up to their own, `window` slots.
// What lies between is skipped in steps of `step` slots.  (window and sinks are at most 2^30 here, and positive.)
ICUA_HD SlotGap window_gap(int first_own, int n_kv, int window, int sinks, int step) {
    const int start = first_own - window + 1, from = ((sinks < n_kv ? sinks : n_kv) + step - 1) / step * step;
    const int to = start > 0 ? start / step * step : 0;
    return {from, to > from ? to - from : 0};
}
// And the most slots that are left of 2^30 at most, for 128 rows and steps of up to 128.
ICUA_HD int window_slots(int max_kv, int window, int sinks) {
    const long long n = (long long)window + (sinks + 127) / 128 * 128 + 254;
    return n < max_kv ? (int)n : max_kv;
}

// Prefix: sequences s0 .. s1 - 1 share their first n slots, whole steps of PREFIX_STEP (0: they share none).
constexpr int PREFIX_STEP = 128, PREFIX_GROUPS = 64;
struct PrefixGroup {
    int s0, s1, n;
};
ICUA_HD PrefixGroup prefix_group(const int32_t* group_start, const int32_t* prefix_len, int g, int n_seqs, int max_prefix) {
    int s0 = group_start[g], s1 = group_start[g + 1], n = prefix_len[g];
    s0 = s0 < 0 ? 0 : s0 > n_seqs ? n_seqs : s0;
    s1 = s1 < s0 ? s0 : s1 > n_seqs ? n_seqs : s1;
    n = n < 0 ? 0 : n > max_prefix ? max_prefix : n;
    return {s0, s1, s1 - s0 < 2 ? 0 : n / PREFIX_STEP * PREFIX_STEP};
}

}  // namespace icua
