// The paged cache's index arithmetic (vx_paged.h) on the host, over small
// sequences in full: what the tile list covers, and that clamps hold.
#include <stdio.h>

#include <set>

#include "vx_paged.h"

static int bad(const char *what, int n, int T, int w, int s, int t0, int t1) {
    printf("FAIL %s len=%d T=%d window=%d sink=%d tokens %d..%d\n", what, n, T, w, s, t0, t1);
    return 1;
}

int main() {
    const int windows[] = {0, 1, 2, 31, 32, 33, 40, 64, 100, 1000, 2147483647}, sinks[] = {0, 1, 31, 32, 33, 70, 500, 2147483647};
    long checked = 0;
    for (int n = 0; n <= 200; n += (n < 70 ? 1 : 13))
        for (int T : {0, 1, 2, 7, 40, 65})
            for (int w : windows)
                for (int s : sinks) {
                    const vx_pseq q = {5, T, n, n - T};
                    for (int t0 = 0; t0 < (T ? T : 1); t0 += 6)
                        for (int t1 : {t0 - 1, t0, t0 + 3, T - 1}) {
                            if (t1 >= T) continue;
                            std::set<int> want;
                            for (int t = t0; t <= t1; t++) {
                                const long i = n - T + t;
                                const vx_sight v = vx_paged_sight(q, t, w, s);
                                for (int j = 0; j < n + 40; j++) {
                                    const bool see = i >= 0 && j <= i && (w == 0 || j > i - w || j < s);
                                    if (see != v.sees(j)) return bad("sight", n, T, w, s, t0, t1);
                                    if (see) want.insert(j / 32);
                                    if (((v.block(j / 32 * 32) >> (j % 32)) & 1) != (uint32_t)see) return bad("bits", n, T, w, s, t0, t1);
                                }
                            }
                            const vx_tiles tl = vx_paged_tiles(q, t0, t1, w, s);
                            std::set<int> got;
                            for (int k = 0; k < tl.nt; k++) got.insert(tl.at(k));
                            if ((int)got.size() != tl.nt) return bad("a tile twice", n, T, w, s, t0, t1);
                            for (int k : want)
                                if (!got.count(k)) return bad("a tile left out", n, T, w, s, t0, t1);
                            for (int k : got)
                                if (k < 0 || k * 32 >= n) return bad("a tile outside", n, T, w, s, t0, t1);
                            if (t0 == 0 && t1 == T - 1 && got != want) return bad("a tile too many", n, T, w, s, t0, t1);
                            checked++;
                        }
                }
    // clamps: lengths, token ranges and pages from anywhere
    int table[4] = {0, 3, -1, 9}, flag = 0;
    const int vals[] = {-2147483647 - 1, -5, -1, 0, 1, 2, 3, 9, 64, 127, 128, 129, 2147483647};
    for (int n : vals)
        for (int s0 : vals)
            for (int s1 : vals)
                for (int max_T : {1, 3, 9}) {
                    int len[1] = {n}, start[2] = {s0, s1};
                    vx_paged p = {1, 2, 32, 4, 4, 5, table, len, start, 9, max_T, &flag};
                    flag = 0;
                    const vx_pseq s = vx_paged_seq(p, 0);
                    const bool ok = n >= 0 && n <= 128 && s0 >= 0 && s0 <= s1 && s1 <= 9 && s1 - s0 <= max_T;
                    if (s.len < 0 || s.len > 128 || s.start < 0 || s.T < 0 || s.start + s.T > 9 || s.T > max_T || flag == (int)ok)
                        return bad("clamp", n, max_T, s0, s1, s.start, s.T);
                    if (ok && (s.len != n || s.start != s0 || s.T != s1 - s0)) return bad("changed", n, max_T, s0, s1, s.start, s.T);
                }
    int len[1] = {0};
    vx_paged p = {1, 2, 32, 4, 4, 5, table, len, nullptr, 1, 1, &flag};
    for (int r = 0; r < 128; r++) {
        flag = 0;
        const int pg = vx_paged_page(p, 0, r), e = table[r / 32];
        if (pg < 0 || pg >= 4 || flag != (e < 0 || e >= 4) || (!flag && pg != e)) return bad("page", r, pg, e, 0, 0, 0);
    }
    p.page_size = 96;
    p.log2_page = -1;
    for (int r = 0; r < 384; r++)
        if (vx_page_slot(p, r) != r / 96) return bad("slot", r, 0, 0, 0, 0, 0);
    printf("ok %ld\n", checked);
    return 0;
}
