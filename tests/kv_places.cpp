/* The cache's places and the kernels' work items (tlm_hip_kv.h) without a GPU: every function that turns a caller's
 * lengths, bounds and page numbers into addresses and items, over small cases in full. */
#include "../tierlm_amd/csrc/tlm_hip_kv.h"

#include <set>
#include <stdio.h>
#include <stdlib.h>
#include <vector>

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)

static KvView view(int B, int64_t rows, const int32_t *cu, const int32_t *lens, int pages, int n_pages, int heads, int sh,
                   int hd) {
    KvView v = {};
    v.lens = lens; v.cu = cu; v.rows = rows; v.B = B; v.table_pages = pages; v.n_pages = n_pages; v.heads = heads;
    v.sh = sh; v.hd = hd;
    return v;
}

int main() {
    /* every (page, head, position, value) has a place of its own inside the arrays */
    for (int hd = 32; hd <= 96; hd += 32)
        for (int sh = 0; sh < 3; sh++) {
            const KvView v = view(1, 1, nullptr, nullptr, 4, 3, 2, sh, hd);
            std::set<int64_t> k, w;
            const int64_t all = (int64_t)3 * 2 * (16 << sh) * hd;
            for (int page = 0; page < 3; page++)
                for (int h = 0; h < 2; h++)
                    for (int p = 0; p < (16 << sh); p++)
                        for (int e = 0; e < hd; e++) {
                            const int64_t at = kv_block(v, page, p / 16, h);
                            CHECK(at >= 0);
                            k.insert(at + kv_key_at(p % 16, e));
                            w.insert(at + kv_value_at(p % 16, e));
                        }
            CHECK((int64_t)k.size() == all && (int64_t)w.size() == all);
            CHECK(*k.rbegin() == all - 1 && *w.rbegin() == all - 1);
            CHECK(kv_block(v, 1, (4 << sh) + 1, 1) == kv_block(v, 1, 1 & ((1 << sh) - 1), 1));
            for (int64_t page : {-1ll, 3ll, 2147483647ll, -2147483648ll}) CHECK(kv_block(v, (int32_t)page, 0, 0) < 0);
        }
    /* offsets past 32 bits */
    CHECK(kv_block(view(1, 1, nullptr, nullptr, 1, 2000000, 8, 2, 128), 1999999, 3, 7) ==
          ((((int64_t)1999999 * 8 + 7) << 2) + 3) * 2048);

    /* rows stay in range whatever cu holds */
    for (int32_t a : {-2147483647, -1, 0, 3, 7, 8, 2147483647})
        for (int32_t b : {-2147483647, -1, 0, 3, 7, 8, 2147483647}) {
            const int32_t cu[2] = {a, b};
            const KvRows r = kv_rows(view(1, 7, cu, nullptr, 1, 1, 1, 0, 32), 0);
            CHECK(r.first >= 0 && r.n >= 0 && r.first + r.n <= 7);
        }
    const int32_t lens[3] = {-1, 2147483647, 5};
    CHECK(kv_len(view(3, 3, nullptr, lens, 1, 1, 1, 0, 32), 0) == 0);
    CHECK(kv_len(view(3, 3, nullptr, lens, 1, 1, 1, 0, 32), 1) == 2147483647);
    CHECK(kv_cap(view(3, 3, nullptr, lens, 1 << 18, 1, 1, 8, 32)) == (int64_t)1 << 30);

    /* append: the blocks of n rows that end before position len, each once, as many as the launch allows for */
    for (int64_t n = 0; n < 70; n++)
        for (int64_t len = 0; len < 90; len++) {
            std::set<int64_t> blocks;
            for (int64_t p = len - n; p < len; p++) blocks.insert(p >= 0 ? p / 16 : -1 - (-1 - p) / 16);
            CHECK(kv_append_items(n, len) == (int64_t)blocks.size());
            if (n) CHECK(kv_floor16(len - n) == *blocks.begin());
            CHECK(kv_append_items(n, len) <= kv_append_most(n, 1));
        }
    for (int a = 0; a < 40; a++)
        for (int b = 0; b < 40; b++)
            for (int len = 0; len < 33; len += 3) {
                const int64_t most = kv_append_most(a + b, 2);
                CHECK(kv_append_items(a, a + len) + kv_append_items(b, b + 15 - len % 16) <= most);
            }

    /* decode: the workers' shares cover the units in order, in parts that differ by one at most; a unit's worker is found,
     * and no worker needs more than the two places it has */
    CHECK(kv_units(0) == 1 && kv_units(1) == 1 && kv_units(128) == 1 && kv_units(129) == 2 && kv_units(1 << 30) == 1 << 23);
    for (int W = 1; W < 40; W++)
        for (int U = 1; U < 200; U++) {
            const KvShares s = kv_shares(U, W);
            CHECK(kv_share(s, 0) == 0 && kv_share(s, W) == U);
            for (int w = 0; w < W; w++) {
                const int n = kv_share(s, w + 1) - kv_share(s, w);
                CHECK(n == U / W || n == U / W + 1);
                for (int x = kv_share(s, w); x < kv_share(s, w + 1); x++) CHECK(kv_worker(s, x) == w);
            }
            for (int step = 1; step < 30; step += 4) {       /* sequences of step units */
                std::set<int> slots;
                for (int a = 0; a < U; a += step) {
                    const int b = a + step < U ? a + step : U, w0 = kv_worker(s, a), n = kv_worker(s, b - 1) - w0 + 1;
                    for (int i = 0; i < n && n > 1; i++) CHECK(slots.insert(kv_slot(w0 + i, i == 0)).second);
                }
                CHECK(slots.empty() || (*slots.begin() >= 0 && *slots.rbegin() < 2 * W));
            }
        }
    CHECK(kv_share(kv_shares((1 << 30) - 1, 512), 512) == (1 << 30) - 1 && kv_worker(kv_shares((1 << 30) - 1, 512), (1 << 30) - 2) == 511);

    /* prompt: as many tiles as the launch allows for */
    for (int a = 0; a < 60; a++)
        for (int b = 0; b < 60; b++)
            for (int g : {1, 3, 8, 16})
                if (a + b > 0)
                    CHECK(kv_prompt_items(a, g, 128) + kv_prompt_items(b, g, 128) <= kv_prompt_most(a + b, 2, g, 128));
    puts("ok");
    return 0;
}
