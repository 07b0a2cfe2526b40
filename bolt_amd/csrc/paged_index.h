// Where the tokens of a batch live in a paged key / value cache. Every number that comes from device memory (lengths, row
// offsets, page numbers) is checked here before it becomes an address: what points outside the rows, the page table or the
// pool is skipped, never followed. Plain integer code that compiles for the host as well.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "layout.h"

namespace bg {

// A divisor known to the host: quotients of numbers below 2^31 by one product. With s = ceil(log2 d) and
// m = floor(2^(31+s) / d) + 1 = (2^(31+s) + e) / d, 0 < e <= d <= 2^s, n m / 2^(31+s) is n / d plus less than 1 / d.
struct PagedDivisor {
    uint32_t d = 1, m = 0x80000001u, shift = 31;
};

inline PagedDivisor paged_divisor(uint32_t d)
{
    PagedDivisor r;
    r.d = d;
    r.shift = 31;
    while (1u << (r.shift - 31) < d) {
        ++r.shift;
    }
    r.m = (uint32_t)(((uint64_t)1 << r.shift) / d + 1);
    return r;
}

BG_HD inline uint32_t paged_div(uint32_t n, const PagedDivisor &d)
{
    return (uint32_t)((uint64_t)n * d.m >> d.shift);
}

struct PagedBatch {
    const int32_t *table = nullptr;    // [batch][max_pages] page numbers
    const int32_t *lens = nullptr;     // [batch] keys of each sequence, its new tokens included
    const int32_t *offsets = nullptr;  // [batch + 1] first row of each sequence's new tokens; null: one token each, row b
    uint32_t max_pages = 0, batch = 0, rows = 0;
};

// New tokens of sequence b: rows first .. first + count - 1 of the packed rows, at positions pos .. pos + count - 1.
// Rows outside [0, rows) and positions below 0 are the caller's to skip.
struct PagedSeq {
    int64_t first, count, pos;
};

BG_HD inline PagedSeq paged_seq_from(int32_t first, int64_t next, int32_t len)
{
    PagedSeq s;
    s.first = first;
    s.count = next > s.first ? next - s.first : 0;
    s.pos = (len > 0 ? len : 0) - s.count;
    return s;
}

BG_HD inline PagedSeq paged_seq(const PagedBatch &a, uint32_t b)
{
    return a.offsets ? paged_seq_from(a.offsets[b], a.offsets[b + 1], a.lens[b]) : paged_seq_from((int32_t)b, (int64_t)b + 1, a.lens[b]);
}

// The sequence that owns a packed row: the last b with offsets[b] <= row (offsets ascend); the caller checks that the row
// lies below offsets[b + 1]. batch >= 1.
BG_HD inline uint32_t paged_owner(const PagedBatch &a, uint32_t row)
{
    if (!a.offsets) {
        return row < a.batch ? row : a.batch - 1;
    }
    uint32_t lo = 0, hi = a.batch;  // offsets[lo] <= row < offsets[hi], as far as the ends say
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((int64_t)a.offsets[mid] <= (int64_t)row) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// Keys [lo, hi) that a token at position pos sees: its own and those before it, the last `window` of them (0: all), as far
// as the table has pages.
struct PagedSpan {
    uint32_t lo, hi;
};

BG_HD inline PagedSpan paged_span(int64_t pos, uint32_t window, uint32_t capacity)
{
    PagedSpan r = {0, 0};
    if (pos >= 0) {
        const int64_t end = pos + 1;
        r.hi = end < (int64_t)capacity ? (uint32_t)end : capacity;
        r.lo = window && end > (int64_t)window ? (uint32_t)(end - window) : 0;
        r.lo = r.lo < r.hi ? r.lo : r.hi;
    }
    return r;
}

// The same for the newest token of a sequence of `len` keys, paged_span(len - 1, ..): 32 bits hold all of it
BG_HD inline PagedSpan paged_span_newest(int32_t len, uint32_t window, uint32_t capacity)
{
    const uint32_t keys = len > 0 ? (uint32_t)len : 0;
    PagedSpan r;
    r.hi = keys < capacity ? keys : capacity;
    r.lo = window && keys > window ? keys - window : 0;
    r.lo = r.lo < r.hi ? r.lo : r.hi;
    return r;
}

// Slot of a key in the pool, in units of head rows: ((page * kv_heads + head) * page_size + place), or -1 where the page
// number is none of the pool's. key < max_pages << shift.
BG_HD inline int64_t paged_slot(const int32_t *table_row, uint32_t key, uint32_t shift, uint32_t pages, uint32_t kv_heads, uint32_t head)
{
    const uint32_t page = (uint32_t)table_row[key >> shift];
    if (page >= pages) {
        return -1;
    }
    return ((((int64_t)page * kv_heads + head) << shift) | (key & ((1u << shift) - 1)));
}

}  // namespace bg
