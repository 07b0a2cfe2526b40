// The index arithmetic of the paged cache on the host, with lists that point outside everything: prints "ok", or the first
// contradiction. Built with address and undefined-behaviour checks by tests/test_paged_cpu.py.
#include <cstdio>
#include <vector>

#include "../bolt_amd/csrc/paged_index.h"

using namespace bg;

#define WANT(x)                                      \
    do {                                             \
        if (!(x)) {                                  \
            printf("line %d: %s\n", __LINE__, #x);   \
            return 1;                                \
        }                                            \
    } while (0)

int main()
{
    const int32_t low = -0x7fffffff - 1, high = 0x7fffffff;
    const std::vector<int32_t> table = {3, -1, 7, low, high, 0, 1, 2};  // [2][4], pool of 8 pages
    const std::vector<int32_t> lens = {13, low};
    PagedBatch a;
    a.table = table.data();
    a.lens = lens.data();
    a.max_pages = 4;
    a.batch = 2;
    a.rows = 2;
    // one row per sequence
    PagedSeq s = paged_seq(a, 0);
    WANT(s.first == 0 && s.count == 1 && s.pos == 12);
    s = paged_seq(a, 1);
    WANT(s.first == 1 && s.count == 1 && s.pos == -1);
    WANT(paged_owner(a, 0) == 0 && paged_owner(a, 1) == 1 && paged_owner(a, 99) == 1);
    // pages outside the pool are no slots
    WANT(paged_slot(table.data(), 0, 2, 8, 5, 4) == ((3 * 5 + 4) << 2));
    WANT(paged_slot(table.data(), 3, 2, 8, 5, 4) == (((3 * 5 + 4) << 2) | 3));
    WANT(paged_slot(table.data(), 4, 2, 8, 5, 0) == -1 && paged_slot(table.data(), 12, 2, 8, 5, 0) == -1);
    WANT(paged_slot(table.data() + 4, 3, 2, 8, 5, 0) == -1 && paged_slot(table.data(), 8, 2, 7, 5, 0) == -1);
    const int32_t far = 0x7ffffffe;
    WANT(paged_slot(&far, 5, 12, 0x7fffffffu, 1024, 1023) == ((((int64_t)far * 1024 + 1023) << 12) | 5));
    // spans stay inside the table's reach, whatever the position
    const int64_t positions[] = {low, -1, 0, 1, 15, 16, 17, high, (int64_t)high + 5};
    const uint32_t windows[] = {0, 1, 2, 16, 0x7fffffffu, 0xffffffffu};
    for (int64_t p : positions) {
        for (uint32_t w : windows) {
            const PagedSpan r = paged_span(p, w, 16);
            WANT(r.lo <= r.hi && r.hi <= 16);
            for (uint32_t k = 0; k < 16; ++k) {
                const bool sees = (int64_t)k <= p && (w == 0 || (int64_t)k > p - (int64_t)w);
                WANT(sees == (k >= r.lo && k < r.hi));
            }
        }
    }
    // quotients by a product
    for (uint32_t d = 1; d <= 16384; d = d < 300 ? d + 1 : d * 3 / 2 + 1) {
        const PagedDivisor by = paged_divisor(d);
        for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 2 * d - 1, 2 * d, 1000 * d - 1, 1000 * d, 0x7fffffffu / d * d - 1, 0x7fffffffu / d * d, 0x7ffffffeu, 0x7fffffffu}) {
            WANT(paged_div(n, by) == n / d);
        }
    }
    // the newest token's
    const int32_t lengths[] = {low, -1, 0, 1, 2, 15, 16, 17, 100, high};
    for (int32_t len : lengths) {
        for (uint32_t w : windows) {
            for (uint32_t capacity : {1u, 16u, 0x7fffffffu}) {
                const PagedSpan r = paged_span_newest(len, w, capacity), q = paged_span((int64_t)len - 1, w, capacity);
                WANT(r.lo == q.lo && r.hi == q.hi);
            }
        }
    }
    // ragged rows: owners by search, with empty sequences, gaps in front and lists that descend or overrun
    const std::vector<std::vector<int32_t>> lists = {{0, 3, 3, 5}, {2, 2, 4, 9}, {5, 1, 9, 0}, {low, low, high, high}, {0, 0, 0, 0}};
    const std::vector<int32_t> three = {10, 20, high};
    for (const auto &o : lists) {
        PagedBatch r;
        r.table = table.data();
        r.lens = three.data();
        r.offsets = o.data();
        r.batch = 3;
        r.rows = 9;
        r.max_pages = 1;
        for (uint32_t row = 0; row < 9; ++row) {
            const uint32_t b = paged_owner(r, row);
            WANT(b < 3);
            const PagedSeq q = paged_seq(r, b);
            WANT(q.count >= 0 && q.count <= 0xffffffffll);
            if (o[0] <= o[1] && o[1] <= o[2] && o[2] <= o[3]) {
                const bool owned = (int64_t)row >= o[0] && (int64_t)row < o[3];
                WANT(owned == ((int64_t)row >= q.first && (int64_t)row < q.first + q.count));
            }
        }
    }
    printf("ok\n");
    return 0;
}
