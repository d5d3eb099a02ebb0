"""z2h_pages_fork and z2h_pages_compact against their definitions, item by item: shares, copies of partly filled pages in all layers, room,
sequences cut off and ended, pools that run dry, bad items, random histories, compaction in place and apart, streams, replayed graphs,
refusals, and a server's run of these with the attention that reads the pages."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, TYPES, Attn, attention, check, context, ints
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


class Pool:
    """A cache of several layers on the device beside a restatement of it on the host."""

    def __init__(self, ctx, n_seq, table_len, n_pages, page=16, kvh=2, hd=32, layers=3, dtype=torch.float16, seed=0, gap=0):
        self.ctx, self.page, self.kvh, self.hd, self.layers, self.dtype = ctx, page, kvh, hd, layers, dtype
        g = torch.Generator().manual_seed(seed)
        size = kvh * page * hd
        self.stride, self.layer_stride = size + gap, n_pages * (size + gap) + 2 * gap
        total = layers * self.layer_stride
        self.host = [torch.randn(total, generator=g).to(dtype) for _ in range(2)]
        self.dev = [t.to(DEV) for t in self.host]
        self.table, self.refs = np.full((n_seq, table_len), -1, np.int32), np.zeros(n_pages, np.int32)
        self.d_table, self.d_refs = ints(self.table), ints(self.refs)
        self.pages = z2h.Pages(k=self.dev[0].data_ptr(), v=self.dev[1].data_ptr(), page_stride=self.stride,
                               type=z2h.BF16 if dtype == torch.bfloat16 else z2h.F16, n_pages=n_pages, page_rows=page, n_head_kv=kvh, head_dim=hd,
                               table=self.d_table.data_ptr(), n_seq=n_seq, table_len=table_len)
        self.ws = torch.full((ctx.pages_ws_bytes(self.pages, 4096),), 255, dtype=torch.uint8, device=DEV)

    def view(self, t):
        """[layers][n_pages][kvh][page][hd] of a flat buffer."""
        return t.as_strided((self.layers, len(self.refs), self.kvh, self.page, self.hd),
                            (self.layer_stride, self.stride, self.page * self.hd, self.hd, 1))

    def put_tables(self):
        self.d_table.copy_(ints(self.table)), self.d_refs.copy_(ints(self.refs))

    def fork(self, items, stream=None):
        """items: (src, dst, rows, room). Runs on both sides; returns d_held."""
        cols = [ints([i[c] for i in items]) for c in range(4)]
        held = torch.full((len(items),), -9, dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        self.ctx.pages_fork(self.pages, self.layers, self.layer_stride, self.d_refs.data_ptr(), len(items), *(c.data_ptr() for c in cols),
                            held.data_ptr(), self.ws.data_ptr(), self.ws.numel(), stream=stream)
        torch.cuda.synchronize()
        want = self.fork_host(items)
        assert held.cpu().tolist() == want, (items, held.cpu().tolist(), want)
        self.same()
        return want

    def pages_held(self, table, s):
        out = []
        for p in table[s]:
            if not 0 <= p < len(self.refs):
                break
            out.append(int(p))
        return out

    def fork_host(self, items):
        P, T, S = self.page, self.table.shape[1], len(self.table)
        dsts = [i[1] for i in items]
        old, jobs, held = self.table.copy(), [], []
        for i, (s, d, rows, room) in enumerate(items):
            ok = 0 <= s < S and 0 <= d < S and d not in dsts[:i] and not (s != d and s in dsts)
            if not ok:
                jobs.append(None)
                continue
            have = self.pages_held(old, s)
            rows = min(max(rows, 0), len(have) * P)
            room = min(max(room, rows), T * P)
            whole, part = rows // P, rows % P
            stay = whole + (part > 0) if s == d else 0
            for p in self.pages_held(old, d)[stay:]:
                self.refs[p] -= 1
            if s != d:
                for p in have[:whole]:
                    self.refs[p] += 1
            jobs.append((s, d, have, rows, room, whole, part))
        keeps = [j is not None and j[0] == j[1] and j[6] > 0 and self.refs[j[2][j[5]]] <= 1 for j in jobs]
        free = [p for p in range(len(self.refs)) if self.refs[p] <= 0]
        for j, keep in zip(jobs, keeps):
            if j is None:
                held.append(-1)
                continue
            s, d, have, rows, room, whole, part = j
            row = have[:whole + keep]
            copy = part > 0 and not keep
            if copy and s == d:
                self.refs[have[whole]] -= 1
            need = -(-room // P) - len(row)
            got, free = free[:need], free[need:]
            for p in got:
                self.refs[p] = 1
            if copy and got:
                for t in self.host:
                    w = self.view(t)
                    w[:, got[0], :, :part] = w[:, have[whole], :, :part]
            self.table[d] = row + got + [-1] * (T - len(row) - len(got))
            held.append(min(room, (len(row) + len(got)) * P))
        return held

    def compact(self, apart=False, stream=None):
        table = torch.full_like(self.d_table, -9) if apart else self.d_table
        refs = torch.full_like(self.d_refs, -9) if apart else self.d_refs
        n = torch.full((1,), -9, dtype=torch.int32, device=DEV)
        before = self.d_table.clone(), self.d_refs.clone()
        torch.cuda.synchronize()
        self.ctx.pages_compact(self.pages, self.layers, self.layer_stride, self.d_refs.data_ptr(), table.data_ptr(), refs.data_ptr(),
                               n.data_ptr(), self.ws.data_ptr(), self.ws.numel(), stream=stream)
        torch.cuda.synchronize()
        if apart:
            assert torch.equal(before[0], self.d_table) and torch.equal(before[1], self.d_refs)
            self.d_table.copy_(table), self.d_refs.copy_(refs)
        used = int((self.refs > 0).sum())
        behind, holes = [p for p in range(used, len(self.refs)) if self.refs[p] > 0], [p for p in range(used) if self.refs[p] <= 0]
        assert len(behind) == len(holes)
        new = {a: b for a, b in zip(behind, holes)}
        for a, b in new.items():
            for t in self.host:
                w = self.view(t)
                w[:, b] = w[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.refs[used:] = 0
        for s, row in enumerate(self.table):
            self.table[s] = [-1 if not 0 <= p < len(self.refs) else new.get(int(p), -1 if p >= used else p) for p in row]
        assert int(n) == used
        self.same()
        return used

    def same(self):
        assert np.array_equal(self.d_table.cpu().numpy(), self.table), "table"
        assert np.array_equal(self.d_refs.cpu().numpy(), self.refs), "counts"
        for d, h in zip(self.dev, self.host):
            assert torch.equal(d.cpu(), h), "pages"

    def counts_hold(self):
        n = np.zeros_like(self.refs)
        for s in range(len(self.table)):
            for p in self.pages_held(self.table, s):
                n[p] += 1
        assert np.array_equal(n, self.refs)


@pytest.mark.parametrize("page,kvh,hd,layers,dtype,gap", [(16, 2, 32, 3, torch.float16, 0), (64, 4, 128, 1, torch.bfloat16, 0), (32, 1, 64, 5, torch.float16, 24),
                                                         (4096, 1, 32, 1, torch.bfloat16, 8)])
def test_a_prompt_taken_over(ctx, page, kvh, hd, layers, dtype, gap):
    """Room for a prompt, forks of it at lengths around pages, then each grown, cut off and ended."""
    print(f"pages of {page}, {kvh} heads of {hd}, {layers} layers", flush=True)
    p = Pool(ctx, 9, 6, 40, page, kvh, hd, layers, dtype, gap=gap)
    n = 2 * page + 5
    assert p.fork([(0, 0, 0, n)]) == [n]
    p.fork([(0, 1, n, n + 1), (0, 2, 2 * page, 2 * page), (0, 3, page - 1, page), (0, 4, 1, 0), (0, 5, 0, page), (0, 6, n + 1000, 7),
            (0, 7, page, 3 * page + 1)])
    p.counts_hold()
    p.fork([(1, 1, n, 3 * page + 1), (2, 2, 2 * page, 2 * page + 1), (3, 3, page - 1, 2 * page), (0, 0, n, n)])
    p.fork([(1, 1, n - 7, 0), (2, 2, page + 3, 0), (6, 6, 2 * page, 0)])         # cut off: pages that are shared are not written
    p.counts_hold()
    p.fork([(s, s, 0, 0) for s in range(9)])
    p.counts_hold()
    assert p.refs.sum() == 0


@pytest.mark.parametrize("n_pages", [20, 9000])
def test_copy_on_write_between_sharers(ctx, n_pages):
    """Two sequences that name the same partly filled page (one cut off inside what the other shares) and both go on."""
    p = Pool(ctx, 4, 4, n_pages)
    p.fork([(0, 0, 0, 40)])
    p.fork([(0, 1, 32, 32), (0, 2, 32, 32)])                                     # two whole pages shared
    p.fork([(1, 1, 20, 20), (2, 2, 19, 40)])                                     # both now end inside page 1
    p.fork([(1, 1, 20, 50), (2, 2, 19, 50), (0, 0, 20, 20)])
    p.counts_hold()


def test_a_destination_gives_up_what_it_had(ctx):
    """Pages given up in a call are handed out in the same call, except those that are copied from."""
    p = Pool(ctx, 6, 4, 12)
    p.fork([(0, 0, 0, 30), (1, 1, 0, 60), (2, 2, 0, 50)])
    assert (p.refs > 0).sum() == 10
    assert p.fork([(0, 1, 30, 64), (0, 2, 17, 20), (0, 3, 30, 30)]) == [64, 20, 30]
    p.counts_hold()


@pytest.mark.parametrize("taken", [0, 8191])
def test_a_pool_runs_dry(ctx, taken):
    """(taken: pages in use that no sequence of the table names)"""
    p = Pool(ctx, 6, 8, 9 + taken, kvh=1)
    p.refs[:taken] = 1
    p.put_tables()
    if taken:
        p.counts_hold = lambda: None
    p.fork([(0, 0, 0, 70)])                                                      # 5 of 9 pages
    assert p.fork([(0, 1, 70, 80), (0, 2, 70, 128), (0, 3, 70, 100), (4, 4, 0, 16)]) == [80, 112, 64, 0]
    p.counts_hold()
    assert p.fork([(3, 3, 64, 65), (2, 2, 40, 40)]) == [65, 40]
    p.fork([(0, 0, 3, 0), (1, 1, 75, 128)])
    p.counts_hold()


@pytest.mark.parametrize("n", [32, 40])
def test_needs_beyond_32_bits(ctx, n):
    """Items that ask for 2^26 pages each of a pool of 100: their sum passes 2^31."""
    print(f"pages items {n}", flush=True)
    length, n_pages = 1 << 26, 100
    table, refs = torch.full((n, length), -1, dtype=torch.int32, device=DEV), torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    k, v = (torch.zeros(n_pages * 16 * 32, dtype=torch.float16, device=DEV) for _ in range(2))
    pages = z2h.Pages(k=k.data_ptr(), v=v.data_ptr(), page_stride=16 * 32, type=z2h.F16, n_pages=n_pages, page_rows=16, n_head_kv=1, head_dim=32,
                      table=table.data_ptr(), n_seq=n, table_len=length)
    ws = torch.full((ctx.pages_ws_bytes(pages, n),), 255, dtype=torch.uint8, device=DEV)
    held = torch.full((n,), -9, dtype=torch.int32, device=DEV)
    seqs, rows = ints(list(range(n - 1, -1, -1))), ints([0] * n)

    def fork(room):
        ctx.pages_fork(pages, 1, 0, refs.data_ptr(), n, seqs.data_ptr(), seqs.data_ptr(), rows.data_ptr(), room.data_ptr(), held.data_ptr(),
                       ws.data_ptr(), ws.numel())
        torch.cuda.synchronize()
    for _ in range(2):
        fork(ints([40] + [1 << 30] * (n - 1)))
        assert held.tolist() == [40, 97 * 16] + [0] * (n - 2)
        assert table[n - 1, :4].tolist() == [0, 1, 2, -1] and torch.equal(table[n - 2, :98], ints([*range(3, 100), -1]).view(-1))
        assert refs.tolist() == [1] * n_pages and int((table >= 0).sum()) == n_pages
    fork(ints([0] * n))
    assert refs.tolist() == [0] * n_pages and int((table >= 0).sum()) == 0


@pytest.mark.parametrize("n_pages", [30, 8193])
def test_bad_items_change_nothing(ctx, n_pages):
    p = Pool(ctx, 5, 4, n_pages)
    p.fork([(0, 0, 0, 40), (1, 1, 0, 20)])
    big = 2 ** 31 - 1
    got = p.fork([(0, 2, 40, 50), (0, 2, 33, 33), (5, 3, 1, 1), (0, -1, 1, 1), (0, 5, 1, 1), (-3, 3, 1, 1), (2, 4, 10, 10), (big, big, big, big),
                  (-big, 3, 0, 0)])
    assert got == [50] + [-1] * 8
    assert p.fork([(0, 0, big, big), (0, 0, 1, 1), (0, 3, 1, 1), (1, 3, -5, -7)]) == [64, -1, -1, -1]
    p.fork([(1, 3, -5, -7), (1, 4, big, -big)])
    p.counts_hold()
    # entries out of range end what a sequence holds
    p.table[0, 1] = n_pages
    p.refs[:] = 0
    for s in range(5):
        for q in p.pages_held(p.table, s):
            p.refs[q] += 1
    p.put_tables()
    p.fork([(0, 2, 64, 64)])


@pytest.mark.parametrize("n", [1, 63, 64, 65, 300, 4096])
def test_many_items(ctx, n):
    """As many forks of one prompt as a call may have, in any order."""
    print(f"{n} forks", flush=True)
    p = Pool(ctx, n + 2, 3, 2 * n + 20, layers=1, hd=32, kvh=1)
    p.fork([(0, 0, 0, 35)])
    order = np.random.default_rng(n).permutation(n) + 1
    items = [(0, int(d), 35 - int(d) % 5, 40) for d in order]
    p.fork(items)
    if n > 1:
        p.fork(items[::2])
    p.counts_hold()


@pytest.mark.parametrize("n_pages", [1, 63, 64, 65, 1023, 1024, 1025, 8191, 8192, 8193, 70000])
def test_pools_of_any_size(ctx, n_pages):
    """Free pages far up, in several segments of the pool, in whole words and at their ends."""
    print(f"{n_pages} pages", flush=True)
    p = Pool(ctx, 3, 64, n_pages, layers=1, kvh=1, hd=32, page=16)
    rng = np.random.default_rng(n_pages)
    p.refs[:] = 1
    free = rng.permutation(n_pages)[:min(n_pages, 50)]
    p.refs[free] = 0
    p.put_tables()
    p.fork([(0, 0, 0, 16 * 20 + 3)])
    p.fork([(0, 1, 16 * 20 + 3, 16 * 40), (2, 2, 0, 16)])
    p.compact(apart=True)


@pytest.mark.parametrize("n_pages,most", [(60, 8), (8300, 8), (400, 50)])
def test_random_histories(ctx, n_pages, most):
    """Pools and items that one block takes care of, and ones for which there are several."""
    print(f"histories: {n_pages} pages, {most} items", flush=True)
    for seed in range(6):
        rng = np.random.default_rng(seed)
        p = Pool(ctx, 12, 7, n_pages, page=16, layers=2, kvh=1, seed=seed)
        for step in range(25):
            items = []
            for _ in range(int(rng.integers(1, most))):
                s = int(rng.integers(0, 12))
                items.append((s, s if rng.random() < 0.5 else int(rng.integers(0, 12)), int(rng.integers(0, 112)), int(rng.integers(0, 120))))
            p.fork(items)
            p.counts_hold()
            if rng.random() < 0.3:
                used = p.compact(apart=bool(rng.integers(0, 2)))
                assert (p.refs[:used] > 0).all() and (p.refs[used:] == 0).all()
                p.counts_hold()


@pytest.mark.parametrize("items", [1, 20])
def test_pages_beyond_32_bits(ctx, items):
    """Pages 2^27 bytes apart: rows copied from, to and between pages that lie more than 2^32 bytes behind the first."""
    print(f"pages far apart, items {items}", flush=True)
    n_pages, stride, P, hd = 40, 1 << 26, 16, 32
    k, v = (torch.zeros(n_pages * stride, dtype=torch.float16, device=DEV) for _ in range(2))
    table, refs = np.full((items + 1, 4), -1, np.int32), np.zeros(n_pages, np.int32)
    refs[:36] = 1                                                # (held by nobody here: taken)
    table[0, :2], refs[34:36] = (35, 34), 1
    d_table, d_refs = ints(table), ints(refs)
    rows = [torch.randn((P, hd), generator=torch.Generator().manual_seed(i)).half() for i in range(4)]
    for t, (a, b) in zip((k, v), (rows[:2], rows[2:])):
        t[35 * stride:35 * stride + P * hd], t[34 * stride:34 * stride + P * hd] = a.reshape(-1).to(DEV), b.reshape(-1).to(DEV)
    pages = z2h.Pages(k=k.data_ptr(), v=v.data_ptr(), page_stride=stride, type=z2h.F16, n_pages=n_pages, page_rows=P, n_head_kv=1, head_dim=hd,
                      table=d_table.data_ptr(), n_seq=items + 1, table_len=4)
    ws = torch.full((ctx.pages_ws_bytes(pages, items),), 255, dtype=torch.uint8, device=DEV)
    src, dst, take, room = ints([0] * items), ints(list(range(1, items + 1))), ints([P + 5] * items), ints([P + 5] * items)
    ctx.pages_fork(pages, 1, 0, d_refs.data_ptr(), items, src.data_ptr(), dst.data_ptr(), take.data_ptr(), room.data_ptr(), 0, ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    got = d_table.cpu().numpy()
    at = lambda t, p: t[p * stride:p * stride + P * hd].view(P, hd).cpu()
    for i in range(min(items, 4)):
        assert got[i + 1].tolist() == [35, 36 + i, -1, -1]
        for t, r in ((k, rows[1]), (v, rows[3])):
            assert torch.equal(at(t, 36 + i)[:5], r[:5]) and not bool(at(t, 36 + i)[5:].any())
    # the first 33 pages end: 33 .. move to the front
    refs = d_refs.cpu().numpy()
    refs[:34] = 0
    d_refs.copy_(ints(refs))
    n = torch.zeros(1, dtype=torch.int32, device=DEV)
    ctx.pages_compact(pages, 1, 0, d_refs.data_ptr(), d_table.data_ptr(), d_refs.data_ptr(), n.data_ptr(), ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    assert int(n) == int((refs > 0).sum()) and d_table[0].tolist() == [1, 0, -1, -1]
    for t, (a, b) in zip((k, v), (rows[:2], rows[2:])):
        assert torch.equal(at(t, 1), a) and torch.equal(at(t, 0), b) and torch.equal(at(t, 2)[:5], b[:5])


def test_compact_edges(ctx):
    """Nothing in use, all in use, one page at the very end, entries that name nothing."""
    p = Pool(ctx, 2, 3, 1500, layers=2, kvh=1, hd=32)
    assert p.compact() == 0
    p.table[1, 0], p.refs[1499] = 1499, 1
    p.table[0] = [-5, 1500, 1400]                                                # (1400 has a count of 0)
    p.put_tables()
    assert p.compact(apart=True) == 1
    p.refs[:] = 1
    p.put_tables()
    assert p.compact() == 1500


def test_streams_and_graphs(ctx):
    """A captured fork and compaction replayed on new items: as the restatement has it."""
    p = Pool(ctx, 8, 6, 50)
    p.fork([(0, 0, 0, 70), (1, 1, 0, 20)])
    cols = [ints([0] * 3) for _ in range(4)]
    held = torch.zeros(3, dtype=torch.int32, device=DEV)
    n = torch.zeros(1, dtype=torch.int32, device=DEV)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        ctx.pages_fork(p.pages, p.layers, p.layer_stride, p.d_refs.data_ptr(), 3, *(c.data_ptr() for c in cols), held.data_ptr(), p.ws.data_ptr(),
                       p.ws.numel(), stream=side.cuda_stream)
        ctx.pages_compact(p.pages, p.layers, p.layer_stride, p.d_refs.data_ptr(), p.d_table.data_ptr(), p.d_refs.data_ptr(), n.data_ptr(),
                          p.ws.data_ptr(), p.ws.numel(), stream=side.cuda_stream)
    for items in ([(0, 2, 70, 80), (0, 3, 33, 33), (1, 4, 20, 40)], [(2, 2, 0, 0), (1, 1, 19, 19), (3, 5, 30, 60)], [(0, 0, 0, 0), (4, 2, 20, 96), (5, 5, 30, 31)]):
        for c, col in enumerate(cols):
            col.copy_(torch.tensor([i[c] for i in items]))
        graph.replay()
        torch.cuda.synchronize()
        assert held.cpu().tolist() == p.fork_host(items)
        graph_state = [t.clone() for t in (p.d_table, p.d_refs, *p.dev)]
        # the compaction on the host, from the restatement's fork
        q = Pool.compact
        p.d_table.copy_(ints(p.table)), p.d_refs.copy_(ints(p.refs))
        for d, h in zip(p.dev, p.host):
            d.copy_(h.to(DEV))
        q(p)
        for a, b in zip(graph_state, (p.d_table, p.d_refs, *p.dev)):
            assert torch.equal(a, b)
        torch.randn(1000, device=DEV).sum().item()
    st = torch.cuda.Stream()
    p.fork([(5, 6, 31, 40)], stream=st.cuda_stream)
    p.compact(stream=st.cuda_stream)


def test_a_server_run(ctx):
    """A prompt attended over its own rows and appended, taken over by three requests, each of which appends rows of its own behind it and
    attends over its pages; one ends, the pool is made compact, and the others go on: every output as the 64-bit history has it."""
    heads, kvh, hd, P, n = 8, 2, 64, 16, 37
    p = Pool(ctx, 4, 6, 40, P, kvh, hd, layers=1)
    g = torch.Generator().manual_seed(1)
    rope = z2h.Rope(base=10000.0, n_dims=0)
    w = (heads + 2 * kvh) * hd

    class View:                                                                  # what the attention's restatement reads
        pass
    view = View()
    view.kvh = kvh
    history = {0: [], 1: [], 2: [], 3: []}
    view.rows = lambda s, m: [torch.stack([h[i] for h in history[s]][:m]).double() for i in (0, 1)]

    def append(seqs, pos, x):
        d, at, rows = x.to(DEV), ints(seqs), ints(pos)
        ctx.paged_append(p.pages, rope, len(seqs), at.data_ptr(), rows.data_ptr(), z2h.F16, d.data_ptr() + 2 * heads * hd, w,
                         d.data_ptr() + 2 * (heads + kvh) * hd, w)
        torch.cuda.synchronize()
        for s, row in zip(seqs, x):
            history[s].append((row[heads * hd:(heads + kvh) * hd].view(kvh, hd), row[(heads + kvh) * hd:].view(kvh, hd)))
        return d

    def attend(seqs, rows, d):
        """The last `rows` rows of each sequence in `seqs`, this call's own."""
        row_start, lens = [0], []
        for s in range(4):
            row_start.append(row_start[-1] + (rows if s in seqs else 0))
            lens.append(len(history[s]))

        class Held:
            pages, kvh = p.pages, view.kvh
            rows = staticmethod(view.rows)
        a = Attn(ctx, Held, heads, row_start, lens, (), "f16")
        out = torch.zeros((row_start[-1], heads * hd), dtype=torch.float16, device=DEV)
        a.plan()
        a.run(d, out, hd ** -0.5)
        torch.cuda.synchronize()
        q = d[:, :heads * hd].cpu().double().view(-1, heads, hd)
        ref, tol = attention(Held, q, row_start, lens, hd ** -0.5, torch.float16)
        check(out.view(-1, heads, hd), ref, tol)
        return out

    def resync():
        torch.cuda.synchronize()
        for h, d in zip(p.host, p.dev):
            h.copy_(d.cpu())
    p.fork([(0, 0, 0, n)])
    x = torch.randn((n, w), generator=g).half()
    d = append([0] * n, list(range(n)), x)
    resync()
    start, out = ints([0, n]), torch.zeros((n, heads * hd), dtype=torch.float16, device=DEV)
    ptr = d.data_ptr()
    ctx.prompt_attn(1, start.data_ptr(), n, heads, kvh, hd, hd ** -0.5, z2h.F16, ptr, w, ptr + 2 * heads * hd, w, ptr + 2 * (heads + kvh) * hd, w,
                    out.data_ptr(), heads * hd)
    torch.cuda.synchronize()
    ref, tol = attention(view, x[:, :heads * hd].double().view(n, heads, hd), [0, n], [n], hd ** -0.5, torch.float16)
    check(out.view(n, heads, hd), ref, tol, "prompt")
    paged = attend([0], n, d)                                                    # the same over the pages
    check(paged.view(n, heads, hd), ref, tol, "prompt over pages")
    p.fork([(0, s, n, n + 20) for s in (1, 2, 3)])
    for s in (1, 2, 3):
        history[s] = list(history[0])
    for step in range(6):
        live = [1, 2, 3] if step < 3 else [1, 3]
        if step == 3:
            p.fork([(2, 2, 0, 0), (0, 0, 0, 0)])
            history[2], history[0] = [], []
            p.compact(apart=True)
        x = torch.randn((len(live), w), generator=g).half()
        d = append(live, [len(history[s]) for s in live], x)
        attend(live, 1, d)
        resync()
    p.counts_hold()


def test_refusals_and_nothing_to_do(ctx):
    p = Pool(ctx, 3, 4, 20)
    one = ints([0, 1, 2]).data_ptr()
    good = dict(pages=p.pages, layers=3, ls=p.layer_stride, refs=p.d_refs.data_ptr(), n=1, src=one, dst=one, rows=one, room=one, ws=p.ws.data_ptr(),
                nb=p.ws.numel(), t=p.d_table.data_ptr())
    fork = lambda a: ctx.pages_fork(a["pages"], a["layers"], a["ls"], a["refs"], a["n"], a["src"], a["dst"], a["rows"], a["room"], 0, a["ws"], a["nb"])
    compact = lambda a: ctx.pages_compact(a["pages"], a["layers"], a["ls"], a["refs"], a["t"], a["refs"], 0, a["ws"], a["nb"])
    shared = [dict(layers=0), dict(layers=-1), dict(ls=8), dict(ls=p.layer_stride + 4), dict(refs=0), dict(ws=0), dict(ws=p.ws.data_ptr() + 8), dict(nb=64),
              dict(layers=70000)]
    for bad in shared + [dict(n=-1), dict(n=4097), dict(src=0), dict(dst=0), dict(rows=0), dict(room=0)]:
        with pytest.raises(z2h.Z2HError):
            fork({**good, **bad})
    for bad in shared + [dict(t=0)]:
        with pytest.raises(z2h.Z2HError):
            compact({**good, **bad})
    for field, value in (("n_pages", (1 << 22) + 1), ("n_pages", 0), ("page_rows", 24), ("type", z2h.F32), ("table", 0), ("k", 0), ("n_seq", 0)):
        x = z2h.Pages.from_buffer_copy(p.pages)
        setattr(x, field, value)
        for call in (lambda: ctx.pages_ws_bytes(x, 1), lambda: fork({**good, "pages": x}), lambda: compact({**good, "pages": x})):
            with pytest.raises(z2h.Z2HError):
                call()
    fork({**good, "n": 0, "src": 0, "dst": 0, "ws": 0, "nb": 0})
    torch.cuda.synchronize()
    p.same()
