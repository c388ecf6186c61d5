// The index arithmetic of the paged attention kernels on the CPU: sequences, pages
// and ranges of batches with malformed entries.  Prints "ok", or what is wrong.
#include "../fuel_amd/csrc/paged.hpp"

#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

using namespace frq;

#define CHECK(x) \
    do { \
        if (!(x)) { \
            printf("line %d: %s\n", __LINE__, #x); \
            return 1; \
        } \
    } while (0)

int main() {
    std::mt19937 rng(5);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    const int odd[] = {0, -1, 1, 1 << 30, -(1 << 30), 0x7fffffff, (int)0x80000000};
    for (int round = 0; round < 3000; round++) {
        const int n = pick(1, 40), width = pick(1, 9), rows = pick(0, 90);
        PagedKv c{nullptr, nullptr, pick(1, 50), pick(4, 7), 1};
        std::vector<int> table(n * width), kv(n), start(n + 1);
        PagedRows b{table.data(), kv.data(), pick(0, 3) ? start.data() : nullptr, n, width, rows, pick(0, width << c.log_ps)};
        if (!b.row_start) b.rows = n;
        for (int& t : table) t = pick(0, 9) ? pick(0, c.n_pages - 1) : odd[pick(0, 6)];
        for (int& l : kv) l = pick(0, 9) ? pick(0, b.cap) : odd[pick(0, 6)];
        for (int& r : start) r = pick(0, 9) ? pick(0, rows) : odd[pick(0, 6)];
        for (int s = 0; s < n; s++) {
            const PgSeq q = pg_seq(b, s);
            CHECK(q.kv >= 0 && q.kv <= b.cap && q.bad == (kv[s] < 0 || kv[s] > b.cap));
            CHECK(q.n >= 0 && (q.n == 0 || (q.row0 >= 0 && (long)q.row0 + q.n <= b.rows)));
            for (int j = 0; j < q.kv + 1100; j += 16) {  // (groups of 16 keys up to the end of a step of 1024)
                if (j < q.kv) CHECK(j >> c.log_ps < width);
                bool none;
                const int page = pg_page(c, table.data() + s * width, j, q.kv, none);
                CHECK(page >= 0 && page < c.n_pages);
                if (j < q.kv) CHECK(none == (table[s * width + (j >> c.log_ps)] != page));
                else CHECK(!none && page == 0);
            }
        }
    }
    for (int round = 0; round < 20000; round++) {  // ranges: whole, in order, none empty, and whose a unit is
        const int wgs = pick(1, PG_WGS);
        const int total = round % 3 ? wgs + pick(0, 5000) : round % 2 ? 0x7fffffff - pick(0, 1000) : wgs;
        CHECK(pg_start(0, total, wgs) == 0 && pg_start(wgs, total, wgs) == total);
        for (int w = 0; w < wgs; w++) {
            const int from = pg_start(w, total, wgs), to = pg_start(w + 1, total, wgs);
            CHECK(from < to);
            CHECK(pg_owner(from, total, wgs) == w && pg_owner(to - 1, total, wgs) == w);
        }
    }
    puts("ok");
    return 0;
}
