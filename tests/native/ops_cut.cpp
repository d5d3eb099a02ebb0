// How z2h_paged_plan cuts a call (csrc/z2h_ops_rules.h), without a GPU. Reads blocks, key heads, query heads per key head, sequences, groups, then
// row_start, kv_len, group_start and prefix_len; prints for narrow and for wide tiles a line: tiles, strips, shift, share, head (0: whole
// shares), the longest piece in steps, shares that have pieces of several strips, tiles of fewer than 97 row-heads.
#include "../../zonos2.cpp_amd/csrc/z2h_ops_rules.h"
#include <algorithm>
#include <cstdio>
#include <vector>

int main() {
    int blocks, nkv, group, n_seq, n_group;
    if (std::scanf("%d %d %d %d %d", &blocks, &nkv, &group, &n_seq, &n_group) != 5) return 1;
    auto read = [](int n) { std::vector<int32_t> v(n); for (auto & x : v) if (std::scanf("%d", &x) != 1) std::exit(1); return v; };
    const auto rows = read(n_seq + 1), len = read(n_seq), gs = read(n_group ? n_group + 1 : 0), pre = read(n_group);
    struct Tile { int heads, key0, key1; };
    std::vector<Tile> tiles;
    const int tr = z2o::tile_rows(group);
    auto span = [&](int r0, int r1, int key0, int key1, bool own, int n) {
        for (int r = r0; r < r1; r += tr) {
            const int m = std::min(tr, r1 - r);
            tiles.push_back({m * group, key0, own ? std::max(key0, std::min(key1, n - (r1 - r0) + (r - r0) + m)) : key1});
        }
    };
    for (int g = 0; g < n_group; ++g)
        if (gs[g] < gs[g + 1] && std::min(pre[g], len[gs[g]]) > 0) span(rows[gs[g]], rows[gs[g + 1]], 0, std::min(pre[g], len[gs[g]]), false, 0);
    for (int s = 0; s < n_seq; ++s) {
        const int g = z2o::group_of(gs.data(), n_group, s);
        span(rows[s], rows[s + 1], g < 0 ? 0 : std::min(pre[g], len[gs[g]]), len[s], true, len[s]);
    }
    long long total = 0;
    for (auto & t : tiles) total += z2o::strip_units(t.key0, t.key1, z2o::is_wide(t.heads), 0) * nkv;
    int shift = 0;
    while (total >> shift >= 1ll << 28) ++shift;
    for (const bool wide : {false, true}) {
        const int most = wide ? blocks : 4 * blocks, head = z2o::piece_cost(wide);
        std::vector<int> units;
        int small = 0;
        for (auto & t : tiles)
            if (z2o::is_wide(t.heads) == wide) { units.push_back((int) z2o::strip_units(t.key0, t.key1, wide, shift)); small += t.heads <= 96; }
        long long cost = 0;
        for (int u : units) cost += z2o::strip_cost(u, head) * nkv;
        const int in_row = z2o::row_share((int) cost, most, head);
        int whole = 0;
        if (!units.empty() && (long long) units.size() * nkv <= most)
            for (int j = 0; j < z2o::WHOLE_SHARES && !whole && z2o::whole_share(j) <= in_row + head; ++j) {
                long long n = 0;
                for (int u : units) n += (u + z2o::whole_share(j) - 1) / z2o::whole_share(j) * nkv;
                if (n <= most) whole = z2o::whole_share(j);
            }
        const z2o::Cut cut = z2o::choose_cut(in_row, whole, head);
        long long begin = 0;
        int longest = 0, several = 0, last = -1;
        for (int u : units) {
            const long long pitch = z2o::strip_pitch(z2o::strip_cost(u, cut.head), cut);
            for (int g = 0; g < nkv; ++g, begin += pitch)
                for (long long b = begin / cut.share; b * cut.share < begin + pitch; ++b) {
                    const z2o::Piece p = z2o::strip_piece((int) begin, u, cut, (int) b);
                    if (p.u0 >= p.u1) continue;
                    longest = std::max(longest, p.u1 - p.u0);
                    several += last == (int) b;
                    last = (int) b;
                }
        }
        std::printf("%zu %zu %d %d %d %lld %d %d\n", units.size(), units.size() * nkv, shift, cut.share, cut.head, (long long) longest << shift, several, small);
    }
}
