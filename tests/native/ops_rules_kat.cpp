// The checks and index rules of the operators on device tensors (csrc/z2h_ops_rules.h), without a GPU: prints "ok" or the
// first thing that is wrong.
#include "../../zonos2.cpp_amd/csrc/z2h_ops_rules.h"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <vector>

#define EXPECT(cond) do { if (!(cond)) { std::printf("line %d: %s\n", __LINE__, #cond); std::exit(1); } } while (0)

static z2h_pages good_pages() {
    static const int32_t table[4] = {0, 1, 2, 3};
    z2h_pages p{};
    p.k = (void *) 256; p.v = (void *) 512; p.table = table;
    p.type = Z2H_F16; p.n_pages = 4; p.page_rows = 16; p.n_head_kv = 2; p.head_dim = 64; p.n_seq = 2; p.table_len = 2;
    p.page_stride = 2 * 16 * 64;
    return p;
}

static void pages() {
    const z2h_pages good = good_pages();
    EXPECT(!z2o::check_pages(&good));
    EXPECT(z2o::check_pages(nullptr));
    auto bad = [](auto change) { z2h_pages p = good_pages(); change(p); return z2o::check_pages(&p) != nullptr; };
    EXPECT(bad([](auto & p) { p.k = nullptr; }));
    EXPECT(bad([](auto & p) { p.v = (void *) 520; }));
    EXPECT(bad([](auto & p) { p.table = nullptr; }));
    EXPECT(bad([](auto & p) { p.type = Z2H_F32; }));
    EXPECT(bad([](auto & p) { p.type = Z2H_Q8_0; }));
    EXPECT(bad([](auto & p) { p.head_dim = 16; }));
    EXPECT(bad([](auto & p) { p.head_dim = 96; }));
    EXPECT(bad([](auto & p) { p.page_rows = 8; p.page_stride = 1 << 20; }));
    EXPECT(bad([](auto & p) { p.page_rows = 24; p.page_stride = 1 << 20; }));
    EXPECT(bad([](auto & p) { p.page_rows = 8192; p.page_stride = 1 << 28; }));
    EXPECT(bad([](auto & p) { p.page_stride -= 8; }));
    EXPECT(bad([](auto & p) { p.page_stride += 4; }));
    EXPECT(bad([](auto & p) { p.n_pages = 0; }));
    EXPECT(bad([](auto & p) { p.n_head_kv = 0; }));
    EXPECT(bad([](auto & p) { p.n_seq = 0; }));
    EXPECT(bad([](auto & p) { p.table_len = 0; }));
    EXPECT(bad([](auto & p) { p.table_len = std::numeric_limits<int32_t>::max(); }));
    EXPECT(!bad([](auto & p) { p.page_stride += 8; }));
    // look-ups: every entry out of range is -1, never an address
    const int32_t table[6] = {0, 3, -1, 4, 2, std::numeric_limits<int32_t>::min()};
    auto at = [&](int seq, int pos) { return z2o::page_of(table, 2, 3, 4, 4, seq, pos); };
    EXPECT(at(0, 0) == 0 && at(0, 15) == 0 && at(0, 16) == 3 && at(0, 31) == 3 && at(0, 32) == -1);
    EXPECT(at(1, 0) == -1 && at(1, 16) == 2 && at(1, 40) == -1);
    EXPECT(at(0, 48) == -1 && at(0, -1) == -1 && at(-1, 0) == -1 && at(2, 0) == -1 && at(0, std::numeric_limits<int>::max()) == -1);
    for (int s = 4; s <= 12; ++s) EXPECT(z2o::page_shift_of(1 << s) == s);
}

static void rope() {
    z2h_rope r{10000.0f, 64, 0, 1.0f, 0.0f, 0.0f, 0, 1.0f};
    EXPECT(!z2o::check_rope(&r, 64) && !z2o::check_rope(&r, 128) && z2o::check_rope(&r, 32) && z2o::check_rope(nullptr, 64));
    EXPECT(z2o::check_rope(&r, 256) && z2o::check_rope(&r, 0) && z2o::check_rope(&r, 65));
    auto bad = [&](auto change) { z2h_rope x = r; change(x); return z2o::check_rope(&x, 128) != nullptr; };
    const float nan = std::numeric_limits<float>::quiet_NaN(), inf = std::numeric_limits<float>::infinity();
    EXPECT(bad([](auto & x) { x.n_dims = 63; }) && bad([](auto & x) { x.n_dims = -2; }) && bad([](auto & x) { x.n_dims = 130; }));
    EXPECT(!bad([](auto & x) { x.n_dims = 0; }));
    for (float v : {0.0f, -1.0f, nan, inf}) {
        EXPECT(bad([&](auto & x) { x.base = v; }) && bad([&](auto & x) { x.factor = v; }) && bad([&](auto & x) { x.mscale = v; }));
    }
    EXPECT(bad([](auto & x) { x.orig_ctx = -1; }) && bad([](auto & x) { x.orig_ctx = 1; }));
    EXPECT(!bad([](auto & x) { x.orig_ctx = 1; x.high_turns = 1.0f; }) && bad([&](auto & x) { x.orig_ctx = 1; x.high_turns = nan; }));
    double t[64];
    const double two_pi = 6.283185307179586476925;
    z2o::rope_turns(r, t);
    EXPECT(std::fabs(t[0] - 1.0 / two_pi) < 1e-16 && std::fabs(t[16] * two_pi - 0.01) < 1e-17);
    r.factor = 4.0f;
    z2o::rope_turns(r, t);
    EXPECT(std::fabs(t[0] - 0.25 / two_pi) < 1e-16);
    r.orig_ctx = 4096; r.low_turns = 1.0f; r.high_turns = 32.0f;                       // fast pairs as they are, slow ones by 4
    z2o::rope_turns(r, t);
    EXPECT(std::fabs(t[0] - 1.0 / two_pi) < 1e-16);
    EXPECT(std::fabs(t[31] / (std::pow(10000.0, -62.0 / 64) / 4 / two_pi) - 1.0) < 1e-12);
    for (int i = 1; i < 32; ++i) EXPECT(t[i] < t[i - 1]);
}

static void rows() {
    EXPECT(!z2o::check_rows((void *) 64, 128, 2, 64, Z2H_F16) && z2o::check_rows((void *) 64, 127, 2, 64, Z2H_F16));
    EXPECT(z2o::check_rows(nullptr, 128, 2, 64, Z2H_F16) && z2o::check_rows((void *) 65, 128, 2, 64, Z2H_F16));
    EXPECT(z2o::check_rows((void *) 66, 128, 2, 64, Z2H_F32) && z2o::check_rows((void *) 64, 128, 2, 64, Z2H_Q8_0));
    EXPECT(z2o::check_rows((void *) 64, 0, 65536, 65536, Z2H_F16));
    z2h_pages p = good_pages();
    EXPECT(!z2o::check_attn(&p, 2, 0, 0) && !z2o::check_attn(&p, 128, 5, 2) && z2o::check_attn(&p, 130, 5, 2) && z2o::check_attn(&p, 3, 5, 2));
    EXPECT(z2o::check_attn(&p, 0, 5, 2) && z2o::check_attn(&p, 2, -1, 2) && z2o::check_attn(&p, 2, 5, 3) && z2o::check_attn(&p, 2, 5, -1));
    EXPECT(z2o::check_attn(&p, 128, 1 << 20, 0) && !z2o::check_attn(&p, 64, 1 << 20, 0));
    EXPECT(!z2o::check_attn_type(Z2H_F32, Z2H_F16) && !z2o::check_attn_type(Z2H_F16, Z2H_F16) && !z2o::check_attn_type(Z2H_BF16, Z2H_BF16));
    EXPECT(z2o::check_attn_type(Z2H_F32, Z2H_BF16) && z2o::check_attn_type(Z2H_BF16, Z2H_F16) && z2o::check_attn_type(Z2H_Q4_K, Z2H_F16));
    EXPECT(!z2o::check_verify(0, 0, 1, 1) && !z2o::check_verify(64, 7, 9, 1 << 20) && z2o::check_verify(1 << 20, 7, 9, 1025) && z2o::check_verify(1, 1, 1, (1 << 20) + 1));
    EXPECT(z2o::check_verify(-1, 1, 1, 5) && z2o::check_verify(1, -1, 1, 5) && z2o::check_verify(1, 1, 0, 5) && z2o::check_verify(1, 1, 1, 0));
    EXPECT(z2o::check_verify(1 << 20, 4096, 1024, 5));
}

// the work of random batches, cut as the plan cuts it, fits the workspace
static void workspace() {
    unsigned long long x = 12345;
    auto rnd = [&](int n) { x = x * 6364136223846793005ull + 1442695040888963407ull; return (int) ((x >> 33) % (unsigned) n); };
    for (int trial = 0; trial < 3000; ++trial) {
        z2h_pages p = good_pages();
        const int group = 1 + rnd(trial % 2 ? 8 : z2o::MAX_GROUP);
        p.n_head_kv = 1 + rnd(16); p.n_seq = 1 + rnd(trial % 7 ? 20 : 300);
        const int heads = group * p.n_head_kv, target = 1 + rnd(1000);
        std::vector<int> rows(p.n_seq), len(p.n_seq), gs{0}, pre;
        int n_rows = 0;
        for (int s = 0; s < p.n_seq; ++s) { rows[s] = rnd(3) ? rnd(3) : rnd(400); len[s] = rnd(2) ? rnd(200) : rnd(30000); n_rows += rows[s]; }
        while (gs.back() < p.n_seq) { gs.push_back(std::min(p.n_seq, gs.back() + 1 + rnd(40))); pre.push_back(rnd(2) ? 0 : rnd(20000)); }
        const z2o::AttnWs w = z2o::attn_ws(p, heads, n_rows, (int) pre.size(), target);
        struct Tile { int rows, key0, key1; };
        std::vector<Tile> tiles;
        const int tr = z2o::tile_rows(group);
        EXPECT(tr >= 1 && tr * group <= z2o::TILE_RH);
        auto span = [&](int r, int k0, int k1) { for (int i = 0; i < r; i += tr) tiles.push_back({std::min(tr, r - i), k0, k1}); };
        for (size_t g = 0; g < pre.size(); ++g) {
            int r = 0;
            for (int s = gs[g]; s < gs[g + 1]; ++s) { r += rows[s]; span(rows[s], std::min(pre[g], len[gs[g]]), len[s]); }
            if (pre[g] > 0) span(r, 0, std::min(pre[g], len[gs[g]]));
        }
        const int shift = trial % 5 == 0 ? 1 + rnd(3) : 0;                             // (of calls far larger than these)
        int64_t parts = 0;
        for (const bool wide : {false, true}) {
            const int most_shares = wide ? target : 4 * target, head = z2o::piece_cost(wide);
            int64_t in_row = 0;
            int whole = 0;
            auto mine = [&](const Tile & t) { return z2o::is_wide(t.rows * group) == wide; };
            auto units_of = [&](const Tile & t) { return mine(t) ? z2o::strip_units(t.key0, t.key1, wide, shift) : 0; };
            for (auto & t : tiles) in_row += z2o::strip_cost(units_of(t), head) * p.n_head_kv;
            for (int j = z2o::WHOLE_SHARES - 1; j >= 0; --j) {
                int64_t n = 0;
                const int share = z2o::whole_share(j);
                EXPECT(share >= 1 && (j == 0 || share > z2o::whole_share(j - 1)));
                for (auto & t : tiles) n += (units_of(t) + share - 1) / share * p.n_head_kv;
                if (n <= most_shares) whole = share;
            }
            z2o::Cut cut = z2o::choose_cut(z2o::row_share(in_row, most_shares, head), whole, head);
            if (trial % 3 == 0) cut = z2o::Cut{z2o::row_share(in_row, most_shares, head), head};
            const int share = cut.share;
            int64_t begin = 0, total = 0;
            for (auto & t : tiles) total += z2o::strip_pitch(z2o::strip_cost(units_of(t), cut.head), cut) * p.n_head_kv;
            const int64_t shares = (total + share - 1) / share;
            EXPECT(shares <= most_shares && total < (1ll << 31));
            for (auto & t : tiles) {
                if (!mine(t)) continue;
                const int units = (int) units_of(t), cost = (int) z2o::strip_cost(units, cut.head), most = z2o::max_pieces(cost, share);
                const int64_t pitch = z2o::strip_pitch(cost, cut);
                parts += (int64_t) most * p.n_head_kv * t.rows * group;
                for (int g = 0; g < p.n_head_kv; ++g, begin += pitch) {
                    // the pieces of the shares that touch the strip are its units, each once, and are numbered in order
                    int u = 0, at = 0, n = -1;
                    if (!units) { EXPECT(z2o::strip_piece((int) begin, units, cut, 0).n == 0); continue; }
                    EXPECT(cut.head || begin % share == 0);
                    for (int b = (int) (begin / share); (int64_t) b * share < begin + pitch; ++b) {
                        EXPECT(b < shares);
                        const z2o::Piece q = z2o::strip_piece((int) begin, units, cut, b);
                        EXPECT(n < 0 || q.n == n);
                        n = q.n;
                        if (q.u0 >= q.u1) continue;
                        EXPECT(q.u0 == u && q.at == at && q.at < q.n);
                        u = q.u1;
                        ++at;
                    }
                    EXPECT(u == units && at == n && n <= most);
                    EXPECT(z2o::strip_piece((int) begin, units, cut, 0).n == n);
                }
            }
        }
        EXPECT((int64_t) tiles.size() <= w.max_tiles || n_rows == 0);
        EXPECT(parts <= w.max_parts);
        EXPECT(w.rows % 256 == 0 && w.tiles % 256 == 0 && w.shares % 256 == 0 && w.strips % 256 == 0 && w.ml % 256 == 0 && w.o % 256 == 0);
        EXPECT(w.bytes >= w.o + w.max_parts * p.head_dim * 4 && w.o >= w.ml + w.max_parts * 8 && w.ml >= w.shares + 5 * target * 64ll);
    }
    // the largest call's counts stay below 2^31
    z2h_pages p = good_pages();
    p.n_seq = 1 << 20; p.n_head_kv = 1;
    const z2o::AttnWs w = z2o::attn_ws(p, 64, 1 << 20, 1 << 20, 4096);
    EXPECT(w.max_parts < (1ll << 31) && w.max_tiles < (1ll << 31));
    p.n_head_kv = 1024; p.page_stride = 1ll << 30;
    const z2o::AttnWs v = z2o::attn_ws(p, 1024, 1 << 16, 1 << 20, 4096);
    EXPECT(v.max_parts < (1ll << 31));
}

int main() {
    workspace();
    pages();
    rope();
    rows();
    std::puts("ok");
}
