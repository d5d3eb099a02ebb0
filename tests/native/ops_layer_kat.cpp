// The checks, sizes and index rules of the operators for whole prompts, experts and a cache's upkeep (csrc/z2h_ops_rules.h), without a GPU:
// prints "ok" or the first thing that is wrong.
#include "../../zonos2.cpp_amd/csrc/z2h_ops_rules.h"
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <vector>

#define EXPECT(cond) do { if (!(cond)) { std::printf("line %d: %s\n", __LINE__, #cond); std::exit(1); } } while (0)

static void prompts() {
    EXPECT(!z2o::check_prompt(1, 10, 16, 4, 128) && !z2o::check_prompt(0, 0, 1, 1, 32) && !z2o::check_prompt(1 << 20, 1 << 20, 64, 1, 64));
    EXPECT(z2o::check_prompt(1, 10, 16, 4, 96) && z2o::check_prompt(1, 10, 15, 4, 64) && z2o::check_prompt(1, 10, 65, 1, 64) && z2o::check_prompt(1, 10, 0, 4, 64));
    EXPECT(z2o::check_prompt(1, 10, 4, 0, 64) && z2o::check_prompt(1, -1, 4, 4, 64) && z2o::check_prompt(-1, 1, 4, 4, 64));
    EXPECT(z2o::check_prompt((1 << 20) + 1, 1, 4, 4, 64) && z2o::check_prompt(1, 1 << 26, 2, 1, 64) && z2o::check_prompt(1, 1, 2048, 2048, 64));
    // every tile of every sequence has a slot of its own, inside the slots that are launched, and the search by slots ends at its sequence
    unsigned long long x = 99;
    auto rnd = [&](int n) { x = x * 6364136223846793005ull + 1442695040888963407ull; return (int) ((x >> 33) % (unsigned) n); };
    for (int trial = 0; trial < 2000; ++trial) {
        const int rows = 1 << rnd(8), n_seq = 1 + rnd(40);
        std::vector<int> start{rnd(3) ? 0 : rnd(100)};
        for (int s = 0; s < n_seq; ++s) start.push_back(start.back() + (rnd(4) ? rnd(trial % 2 ? 10 : 1000) : 0));
        const int n_rows = start.back() + (rnd(2) ? rnd(500) : 0);
        int64_t last = -1;
        for (int s = 0; s < n_seq; ++s)
            for (int j = 0; j * rows < start[s + 1] - start[s]; ++j) {
                const int64_t slot = z2o::prompt_slot(start[s], s, rows) + j;
                EXPECT(slot > last && slot < z2o::prompt_slots(n_rows, n_seq, rows));
                EXPECT(s + 1 == n_seq || slot < z2o::prompt_slot(start[s + 1], s + 1, rows));
                last = slot;
            }
    }
}

// which way calls are cut: the sizes that tests/test_gpu_ops_prompt.py names, on a card of 256 compute units
static void cuts() {
    for (int hd : {32, 64, 128})
        for (bool fp32 : {false, true}) {
            EXPECT(z2o::prompt_cut(260, 3, 4, 2, hd, fp32, 256) == z2o::PROMPT_SMALL);
            EXPECT(z2o::prompt_cut(1331, 8, 60, 20, hd, fp32, 256) == (hd == 32 && fp32 ? z2o::PROMPT_SMALL : z2o::PROMPT_WIDE));
        }
    EXPECT(z2o::prompt_cut(1310, 1, 16, 4, 128, false, 256) == z2o::PROMPT_PAIR && z2o::prompt_cut(2100, 2, 16, 8, 128, true, 256) == z2o::PROMPT_PAIR);
    EXPECT(z2o::prompt_cut(2100, 2, 16, 8, 64, false, 256) == z2o::PROMPT_PAIR && z2o::prompt_cut(2100, 2, 16, 8, 32, false, 256) == z2o::PROMPT_SMALL);
    EXPECT(z2o::prompt_cut(1, 1, 17, 1, 128, false, 256) == z2o::PROMPT_WIDE && z2o::prompt_cut(1, 1, 64, 1, 32, true, 256) == z2o::PROMPT_WIDE);   // (groups of more than 16)
    EXPECT(z2o::prompt_cut(1 << 20, 1 << 20, 64, 1, 128, true, 256) == z2o::PROMPT_WIDE);
}

static void experts() {
    z2h_experts good{(void *) 256, (void *) 512, (void *) 768, Z2H_F16, 32, 1536, 2048};
    EXPECT(!z2o::check_experts(&good) && z2o::check_experts(nullptr));
    auto bad = [&](auto change) { z2h_experts x = good; change(x); return z2o::check_moe(&x, 16, 4) != nullptr && z2o::check_experts(&x) != nullptr; };
    EXPECT(bad([](auto & x) { x.gate = nullptr; }) && bad([](auto & x) { x.up = nullptr; }) && bad([](auto & x) { x.down = nullptr; }));
    EXPECT(bad([](auto & x) { x.gate = (void *) 264; }) && bad([](auto & x) { x.up = (void *) 520; }) && bad([](auto & x) { x.down = (void *) 769; }));
    EXPECT(bad([](auto & x) { x.type = Z2H_F32; }) && bad([](auto & x) { x.type = Z2H_Q8_0; }) && bad([](auto & x) { x.n_expert = 0; }));
    EXPECT(bad([](auto & x) { x.n_expert = 1025; }) && bad([](auto & x) { x.n_ff = 1532; }) && bad([](auto & x) { x.n_embd = 0; }));
    EXPECT(bad([](auto & x) { x.n_embd = -8; }) && bad([](auto & x) { x.n_ff = 65544; }));
    EXPECT(!z2o::check_moe(&good, 0, 1) && !z2o::check_moe(&good, 128, 16) && z2o::check_moe(&good, 129, 1) && z2o::check_moe(&good, -1, 1));
    EXPECT(z2o::check_moe(&good, 1, 0) && z2o::check_moe(&good, 1, 17));
    good.n_expert = 3;
    EXPECT(!z2o::check_moe(&good, 1, 3) && z2o::check_moe(&good, 1, 4));
    EXPECT(!z2o::check_moe_type(Z2H_F32, Z2H_F16) && !z2o::check_moe_type(Z2H_F16, Z2H_F16) && !z2o::check_moe_type(Z2H_BF16, Z2H_BF16));
    EXPECT(z2o::check_moe_type(Z2H_F32, Z2H_BF16) && z2o::check_moe_type(Z2H_BF16, Z2H_F16) && z2o::check_moe_type(Z2H_Q8_0, Z2H_F16));
    // a workspace's parts follow each other and hold what the kernels put there; shares of an output dim are as many as the join takes
    for (int n_expert : {1, 8, 60, 1024})
        for (int dim : {8, 40, 1032, 2048, 65536})
            for (int n : {0, 1, 8, 17, 128})
                for (int k : {1, 16}) {
                    if (k > n_expert) continue;
                    const z2h_experts x{(void *) 256, (void *) 256, (void *) 256, Z2H_F16, n_expert, dim, dim};
                    EXPECT(!z2o::check_moe(&x, n, k));
                    const z2o::MoeWs w = z2o::moe_ws(x, n, k);
                    const int64_t routes = (int64_t) n * k, touched = routes < n_expert ? routes : n_expert, shares = z2o::moe_shares(dim);
                    EXPECT(shares >= 1 && shares <= z2o::MOE_SHARES && z2o::moe_h_stride(dim) >= dim && z2o::moe_h_stride(dim) % 32 == 0);
                    EXPECT(w.touched >= 32 && w.w >= w.touched + 24 * touched && w.row_sel >= w.w + 4 * routes && w.row_w >= w.row_sel + 4 * routes);
                    EXPECT(w.tickets >= w.row_w + 4 * routes && w.parts >= w.tickets + 4 * ((dim + 15) / 16));
                    EXPECT(w.h >= w.parts + (shares > 1 ? 4 * shares * n * dim : 0) && w.bytes >= w.h + 4 * routes * z2o::moe_h_stride(dim));
                    for (int64_t at : {w.touched, w.w, w.row_sel, w.row_w, w.tickets, w.parts, w.h, w.bytes}) EXPECT(at % 256 == 0);
                }
}

static void pool() {
    static const int32_t table[4] = {0, 1, 2, 3};
    z2h_pages p{};
    p.k = (void *) 256; p.v = (void *) 512; p.table = table;
    p.type = Z2H_F16; p.n_pages = 4; p.page_rows = 16; p.n_head_kv = 2; p.head_dim = 64; p.n_seq = 2; p.table_len = 2;
    p.page_stride = 2 * 16 * 64;
    EXPECT(!z2o::check_pool(&p, 0) && !z2o::check_pool(&p, 4096) && z2o::check_pool(&p, 4097) && z2o::check_pool(&p, -1) && z2o::check_pool(nullptr, 1));
    EXPECT(!z2o::check_layers(&p, 1, 0) && !z2o::check_layers(&p, 24, 4 * 2048) && z2o::check_layers(&p, 24, 4 * 2048 - 8) && z2o::check_layers(&p, 2, 4 * 2048 + 4));
    EXPECT(z2o::check_layers(&p, 0, 1 << 20) && z2o::check_layers(&p, 65537, 1 << 20));
    z2h_pages large = p;
    large.n_head_kv = 1024; large.head_dim = 128; large.page_rows = 4096; large.page_stride = 1ll << 29;
    EXPECT(!z2o::check_layers(&large, 8, 1ll << 40) && z2o::check_layers(&large, 9, 1ll << 40));
    p.n_pages = (1 << 22) + 1;
    EXPECT(z2o::check_pool(&p, 1));
    // sizes of a fork: rows of what the source holds, the room of what the table has
    auto is = [](z2o::ForkSize f, int rows, int room, int whole, int pages) { return f.rows == rows && f.room == room && f.whole == whole && f.pages == pages; };
    const int big = std::numeric_limits<int>::max(), least = std::numeric_limits<int>::min();
    EXPECT(is(z2o::fork_size(0, 0, 0, 4, 4), 0, 0, 0, 0) && is(z2o::fork_size(17, 20, 2, 4, 4), 17, 20, 1, 2) && is(z2o::fork_size(32, 0, 2, 4, 4), 32, 32, 2, 2));
    EXPECT(is(z2o::fork_size(33, 33, 2, 4, 4), 32, 33, 2, 3) && is(z2o::fork_size(big, big, 4, 4, 4), 64, 64, 4, 4) && is(z2o::fork_size(least, least, 4, 4, 4), 0, 0, 0, 0));
    EXPECT(is(z2o::fork_size(big, least, 1 << 18, 1 << 18, 12), 1 << 30, 1 << 30, 1 << 18, 1 << 18));
    EXPECT(is(z2o::fork_size(5, big, 1, 1 << 18, 12), 5, 1 << 30, 0, 1 << 18));
    // the workspace's parts follow each other and hold what they are for
    for (int n_pages : {1, 63, 64, 1023, 1024, 1025, 1 << 22})
        for (int n : {0, 1, 4096}) {
            const z2o::PoolWs w = z2o::pool_ws(n_pages, n);
            EXPECT((int64_t) w.segs * z2o::POOL_SEG >= n_pages && w.segs <= z2o::MAX_POOL / z2o::POOL_SEG);
            EXPECT(w.counts >= (int64_t) w.segs * 128 && w.items >= w.counts + 4 * w.segs && w.map >= w.items + 32 * n && w.moves >= w.map + 4ll * n_pages);
            EXPECT(w.bytes >= w.moves + 256 + 8ll * (n_pages / 2) && w.counts % 64 == 0 && w.items % 32 == 0 && w.map % 256 == 0 && w.moves % 256 == 0);
        }
}

int main() {
    prompts();
    cuts();
    experts();
    pool();
    std::puts("ok");
}
