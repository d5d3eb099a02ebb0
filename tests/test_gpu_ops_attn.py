"""z2h_paged_plan / z2h_paged_attn against 64-bit attention: one token to long prompts, shared prefixes that end inside pages,
empty sequences and rows that see nothing, head groups, types, strides, garbage in every cache row that must not be read,
the same values with and without sharing, streams, replayed graphs, and a run of the operators together."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, TYPES, Attn, Cache, attention, check, context, ints, rotate, rotate_tol
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def _case(ctx, typ, lens, rows, heads, kvh, hd, page, groups=(), seed=0, qscale=1.0, **cache):
    """lens, rows: cache rows and query rows of every sequence."""
    dtype = TYPES[typ][1]
    c = Cache(lens, kvh, hd, page, torch.bfloat16 if typ == "bf16" else torch.float16, seed + 1, shared=groups, **cache)
    row_start = np.concatenate([[0], np.cumsum(rows)]).astype(int)
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn((int(row_start[-1]), heads, hd), generator=g) * qscale).to(dtype)
    return c, row_start, q, Attn(ctx, c, heads, row_start, lens, groups, typ)


def _check(ctx, typ, lens, rows, heads, kvh, hd, page, groups=(), seed=0, qscale=1.0, **cache):
    print(f"attn {typ} lens {lens[:8]} rows {rows[:8]} heads {heads}/{kvh} hd {hd} page {page} groups {groups[:4]}", flush=True)
    c, row_start, q, a = _case(ctx, typ, lens, rows, heads, kvh, hd, page, groups, seed, qscale, **cache)
    d = q.to(DEV)
    out = torch.full(d.shape, float("nan"), dtype=d.dtype, device=DEV)
    a.plan()
    a.run(d.view(len(d), -1), out.view(len(d), -1), hd ** -0.5)
    torch.cuda.synchronize()
    ref, tol = attention(c, q.double(), row_start, lens, hd ** -0.5, d.dtype)
    check(out, ref, tol, typ)
    return c, row_start, q, a, out


# lengths around pages, key tiles and chunks; query rows: single tokens
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd,page", [(16, 4, 128, 16), (8, 8, 64, 32), (4, 1, 32, 64), (14, 2, 128, 128), (64, 1, 64, 16)])
def test_single_tokens(ctx, typ, heads, kvh, hd, page):
    lens = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 300, 700]
    _check(ctx, typ, lens, [1] * len(lens), heads, kvh, hd, page)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 5, 4097])
def test_one_sequence(ctx, typ, n):
    _check(ctx, typ, [n], [1], 16, 4, 128, 16)


# drafts and prompt chunks: several rows per sequence, causal among them, some longer than their cache (rows that see nothing)
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd,page", [(16, 4, 128, 16), (8, 8, 64, 32), (6, 2, 32, 16), (32, 2, 128, 64)])
def test_several_rows(ctx, typ, heads, kvh, hd, page):
    _check(ctx, typ, [40, 5, 3, 0, 100, 33, 9, 257], [5, 5, 7, 2, 1, 33, 0, 70], heads, kvh, hd, page)


@pytest.mark.parametrize("typ,heads,kvh,hd", [("f32", 4, 2, 64), ("f16", 16, 4, 128), ("bf16", 2, 2, 32), ("f16", 3, 1, 128)])
def test_prompt_chunk(ctx, typ, heads, kvh, hd):
    _check(ctx, typ, [700, 260], [300, 260], heads, kvh, hd, 32)


# groups that share a prefix: whole pages, pages that the prefix ends in, sequences without rows of their own behind it
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd,page", [(16, 4, 128, 16), (8, 8, 64, 32), (4, 1, 32, 128)])
def test_shared_prefix(ctx, typ, heads, kvh, hd, page):
    lens = [300, 260, 511, 257] + [90, 64] + [77, 700, 701, 709, 700, 720, 1]
    _check(ctx, typ, lens, [1] * 4 + [2, 3] + [1, 1, 4, 1, 1, 9, 1], heads, kvh, hd, page,
           [(0, 4, 257), (4, 6, 64), (7, 12, 699)])


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_wide_group(ctx, typ):
    """More row-heads behind one prefix than a tile holds."""
    rng = np.random.default_rng(1)
    lens = [1000 + int(n) for n in rng.integers(0, 60, 45)]
    _check(ctx, typ, lens, [1] * 45, 8, 2, 128, 16, [(0, 45, 1000)])


def test_long_prefix(ctx):
    lens = [20000 + n for n in (1, 50, 200, 7)]
    _check(ctx, "f16", lens, [1, 1, 1, 2], 8, 2, 128, 64, [(0, 4, 20000)])


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_repeated_calls_agree_bit_for_bit(ctx, typ):
    """Long shared prefix, several wide tiles, two of them partly filled: keys and values pass through LDS in many steps, which
    waves that have nothing to multiply help to fill. No answer depends on who came first."""
    c, row_start, q, a, first = _check(ctx, typ, [4100 + 3 * s for s in range(18)], [1] * 18, 32, 2, 128, 64, groups=[(0, 18, 4096)])
    d = q.to(DEV)
    outs = [torch.empty_like(first) for _ in range(40)]
    for o in outs:
        a.run(d.view(len(d), -1), o.view(len(d), -1), 128 ** -0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_peaked_and_large_queries(ctx):
    """Scores far apart (softmax near one-hot), and queries that f16 could not hold as fp32 rows."""
    _check(ctx, "f32", [300, 40], [1, 3], 8, 2, 64, 16, qscale=30.0)
    _check(ctx, "f16", [300, 40], [1, 3], 8, 2, 64, 16, qscale=30.0)
    c, row_start, q, a = _case(ctx, "f32", [130, 20], [1, 2], 4, 2, 64, 16)
    scale = [1e-6, 1e6, 1e-30, 3e20]                        # per head; the call's scale takes the largest back to size
    for i, s in enumerate(scale):
        q[:, i] *= s
    d, out = q.to(DEV), torch.zeros_like(q, device=DEV)
    a.plan()
    for call_scale in (0.1, 1e-6, 1e-21):
        a.run(d.view(3, -1), out.view(3, -1), call_scale)
        torch.cuda.synchronize()
        ref, tol = attention(c, q.double(), row_start, [130, 20], float(np.float32(call_scale)), torch.float32)
        heads = [i for i, s in enumerate(scale) if s * call_scale <= 2]
        check(out[:, heads], ref[:, heads], tol[:, heads], f"scale {call_scale}")


def test_garbage_is_not_read(ctx):
    """NaN in every cache row behind a sequence's length, in unused pages, and (with the rows of the call in the cache) in
    rows that a query must not see: the same outputs as with finite values there."""
    for typ in ("f32", "f16", "bf16"):
        lens, rows = [40, 21, 300], [3, 5, 40]
        c, row_start, q, a = _case(ctx, typ, lens, rows, 8, 2, 64, 16, fill=float("nan"))
        ref, tol = attention(c, q.double(), row_start, lens, 0.125, q.dtype)
        # the last row of every sequence: only its last query row sees it
        for which, bad in ((0, float("nan")), (1, float("nan")), (1, float("inf"))):
            for s, n in enumerate(lens):
                c.cell(which, s, n - 1)[:] = bad
        c.upload()
        a = Attn(ctx, c, 8, row_start, lens, (), typ)
        d = q.to(DEV)
        out = torch.zeros_like(d)
        a.plan()
        a.run(d.view(len(d), -1), out.view(len(d), -1), 0.125)
        torch.cuda.synchronize()
        hidden = torch.ones(len(q), dtype=torch.bool)
        hidden[row_start[1:] - 1] = False
        check(out[hidden.to(DEV)], ref[hidden], tol[hidden], typ)


def test_infinite_values_reach_the_rows_that_see_them(ctx):
    """An infinite value in the cache gives infinity in the rows that see it and leaves the others alone."""
    for typ in ("f32", "f16"):
        c, row_start, q, _ = _case(ctx, typ, [70], [6], 4, 2, 64, 16)
        c.cell(1, 0, 67)[0, 5] = float("inf")
        c.cell(1, 0, 67)[1, 9] = float("-inf")
        c.upload()
        a = Attn(ctx, c, 4, row_start, [70], (), typ)
        d = q.to(DEV)
        out = torch.zeros_like(d)
        a.plan()
        a.run(d.view(6, -1), out.view(6, -1), 0.125)
        torch.cuda.synchronize()
        ref, tol = attention(c, q.double(), row_start, [70], 0.125, q.dtype)
        assert torch.isinf(ref).sum() == 3 * 4
        tol = torch.where(torch.isfinite(tol), tol, torch.ones_like(tol))
        check(out, ref, tol, typ)


def test_sharing_changes_nothing_but_rounding(ctx):
    """The same cache and queries with the prefix named as shared and not."""
    lens, groups = [530, 515, 900, 512], [(0, 4, 512)]
    c, row_start, q, a = _case(ctx, "f32", lens, [1, 2, 1, 1], 16, 4, 128, 16, groups)
    b = Attn(ctx, c, 16, row_start, lens, (), "f32")
    d = q.to(DEV)
    x, y = torch.zeros_like(d), torch.zeros_like(d)
    a.plan(), b.plan()
    a.run(d.view(5, -1), x.view(5, -1), 0.1), b.run(d.view(5, -1), y.view(5, -1), 0.1)
    torch.cuda.synchronize()
    ref, tol = attention(c, q.double(), row_start, lens, float(np.float32(0.1)), torch.float32)
    check(x, ref, tol), check(y, ref, tol)


def test_strides_alignment_and_in_place(ctx):
    """Queries as columns of a wider row at an odd offset, outputs likewise; then in place."""
    for typ in ("f32", "f16", "bf16"):
        c, row_start, q, a = _case(ctx, typ, [100, 37, 20], [2, 1, 40], 4, 2, 64, 16)
        ref, tol = attention(c, q.double(), row_start, [100, 37, 20], 0.125, q.dtype)
        wide = torch.zeros((43, 301), dtype=q.dtype, device=DEV)
        wide[:, 3:259] = q.view(43, 256).to(DEV)
        out = torch.full((43, 263), 4.0, dtype=q.dtype, device=DEV)
        a.plan()
        a.run(wide[:, 3:], out[:, 5:], 0.125)
        torch.cuda.synchronize()
        check(out[:, 5:261].reshape(43, 4, 64), ref, tol, typ)
        assert bool((out[:, :5] == 4).all()) and bool((out[:, 261:] == 4).all())
        a.run(wide[:, 3:], wide[:, 3:], 0.125)
        torch.cuda.synchronize()
        assert torch.equal(wide[:, 3:259], out[:, 5:261]) and bool((wide[:, :3] == 0).all()) and bool((wide[:, 259:] == 0).all())


def test_lengths_are_clamped_and_bad_pages_stay_inside(ctx):
    """Lengths past the table count as the table's; a page entry out of range reads page 0; a group whose prefix is longer than its
    first sequence shares what that one has."""
    c, row_start, q, _ = _case(ctx, "f16", [64, 48, 40], [1, 1, 1], 4, 2, 64, 16, fill=0.5)
    c.table_host[1, 1] = -7
    c.upload()
    a = Attn(ctx, c, 4, row_start, [10**6, 48, -3], (), "f16")
    d = q.to(DEV)
    out = torch.zeros_like(d)
    a.plan()
    a.run(d.view(3, -1), out.view(3, -1), 0.125)
    torch.cuda.synchronize()
    c.table_host[1, 1] = 0
    ref, tol = attention(c, q.double(), row_start, [64, 48, 0], 0.125, q.dtype)
    check(out, ref, tol)
    c, row_start, q, _ = _case(ctx, "f16", [64, 100], [1, 1], 4, 2, 64, 16, [(0, 2, 64)])
    a = Attn(ctx, c, 4, row_start, [64, 100], [(0, 2, 5000)], "f16")
    out = torch.zeros_like(q, device=DEV)
    d = q.to(DEV)
    a.plan()
    a.run(d.view(2, -1), out.view(2, -1), 0.125)
    torch.cuda.synchronize()
    check(out, *attention(c, q.double(), row_start, [64, 100], 0.125, q.dtype))


def test_rows_outside_the_sequences_give_zeros(ctx):
    """Rows behind the last sequence's see nothing."""
    c, row_start, q, _ = _case(ctx, "f16", [20, 30], [1, 3], 4, 2, 64, 16)
    a = Attn(ctx, c, 4, [0, 1, 4], [20, 30], (), "f16")
    a.row_start = ints([0, 1, 2])
    d = q.to(DEV)
    out = torch.full_like(d, 3.0)
    a.plan()
    a.run(d.view(4, -1), out.view(4, -1), 0.125)
    torch.cuda.synchronize()
    ref, tol = attention(c, q.double()[:2], [0, 1, 2], [20, 30], 0.125, q.dtype)
    check(out[:2], ref, tol)
    assert bool((out[2:] == 0).all())


def test_another_shape_than_the_plans_leaves_the_output(ctx):
    c, row_start, q, a = _case(ctx, "f16", [20, 30], [1, 1], 4, 2, 64, 16)
    d = q.to(DEV)
    out = torch.full_like(d, 3.0)
    a.ws.zero_()
    a.run(d.view(2, -1), out.view(2, -1), 0.125)            # no plan at all
    b = Attn(ctx, c, 4, [0, 1], [20], (), "f16")
    a.plan()
    ws = a.ws if a.ws.numel() >= b.ws.numel() else b.ws
    ctx.paged_attn(c.pages, 4, 1, 0, 0.125, z2h.F16, d.data_ptr(), 256, out.data_ptr(), 256, ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    assert bool((out == 3).all())


def test_side_stream_and_two_calls_at_once(ctx):
    """Two plans with a workspace each on two streams, their calls interleaved: as on the null stream."""
    cases = [_case(ctx, "f16", [700, 1200, 33], [1, 2, 1], 16, 4, 128, 16, seed=s) for s in (1, 2)]
    want = []
    for c, row_start, q, a in cases:
        d, out = q.to(DEV), torch.zeros_like(q, device=DEV)
        a.plan(), a.run(d.view(4, -1), out.view(4, -1), 0.1)
        torch.cuda.synchronize()
        want.append(out)
    streams = [torch.cuda.Stream() for _ in cases]
    ds, outs = [q.to(DEV) for _, _, q, _ in cases], [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, (c, row_start, q, a), d, out in zip(streams, cases, ds, outs):
            a.plan(stream=st.cuda_stream)
            a.run(d.view(4, -1), out.view(4, -1), 0.1, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w, o)


def test_decode_loop_in_a_replayed_graph(ctx):
    """One captured step (append with rotation, plan, attention) replayed while the sequences grow across pages: every step as the
    64-bit restatement of the whole history has it."""
    P, kvh, heads, hd, S = 16, 2, 8, 64, 3
    lens = [30, 47, 64]
    c = Cache(lens, kvh, hd, P, torch.float16, 5, shared=[(0, 3, 30)], room=20, fill=0.0)
    rope = z2h.Rope(base=10000.0, n_dims=64, halves=1)
    g = torch.Generator().manual_seed(1)
    w = (heads + 2 * kvh) * hd
    x = torch.zeros((S, w), device=DEV)
    q = torch.zeros((S, heads * hd), device=DEV)
    out = torch.zeros((S, heads * hd), device=DEV)
    seq, pos = ints(range(S)), ints([0] * S)
    a = Attn(ctx, c, heads, [0, 1, 2, 3], lens, [(0, 3, 30)], "f32")

    def step(stream):
        ctx.paged_append(c.pages, rope, S, seq.data_ptr(), pos.data_ptr(), z2h.F32, x.data_ptr() + 4 * heads * hd, w,
                         x.data_ptr() + 4 * (heads + kvh) * hd, w, heads, x.data_ptr(), w, q.data_ptr(), heads * hd, stream=stream)
        a.plan(stream=stream)
        a.run(q, out, hd ** -0.5, stream=stream)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for i in range(5):
        new = torch.randn((S, w), generator=g)
        x.copy_(new)
        pos.copy_(torch.tensor([n + i for n in lens]))
        a.kv_len.copy_(torch.tensor([n + i + 1 for n in lens]))
        graph.replay()
        torch.cuda.synchronize()
        tpos = torch.tensor([n + i for n in lens])
        qr = rotate(new[:, :heads * hd].reshape(S, heads, hd).double(), tpos, 10000.0, 64, True)
        kr = rotate(new[:, heads * hd:(heads + kvh) * hd].reshape(S, kvh, hd).double(), tpos, 10000.0, 64, True)
        check(q.view(S, heads, hd), qr, rotate_tol(new[:, :heads * hd].reshape(S, heads, hd).double(), qr, 64, True, 1.0, torch.float32))
        for s in range(S):                                  # the device's own rounding of the new rows goes on in the history
            at, r = c.table_host[s, (lens[s] + i) // P], (lens[s] + i) % P
            for t in range(2):
                c.buf[t][at].view(kvh, P, hd)[:, r] = c.dev[t][at].view(kvh, P, hd)[:, r].cpu()
            assert torch.allclose(c.cell(0, s, lens[s] + i).double(), kr[s], atol=4e-3)
            assert torch.equal(c.cell(1, s, lens[s] + i), new[s, (heads + kvh) * hd:].reshape(kvh, hd).half())
        ref, tol = attention(c, q.cpu().double().view(S, heads, hd), [0, 1, 2, 3], [n + i + 1 for n in lens], hd ** -0.5, torch.float32)
        check(out.view(S, heads, hd), ref, tol, f"step {i}")
        torch.randn(1000, device=DEV).sum().item()


def test_refusals(ctx):
    c, row_start, q, a = _case(ctx, "f16", [20, 30], [1, 1], 4, 2, 64, 16)
    d = q.to(DEV)
    p, i, ws, n = d.data_ptr(), a.kv_len.data_ptr(), a.ws.data_ptr(), a.ws.numel()
    for bad in (dict(heads=3), dict(heads=0), dict(rows=-1), dict(groups=3), dict(rs=0), dict(kl=0), dict(gs=0, groups=1), dict(ws=0),
                dict(ws=ws + 16), dict(n=16)):
        x = dict(heads=4, rows=2, groups=0, rs=i, kl=i, gs=i, ws=ws, n=n, **{})
        x.update(bad)
        with pytest.raises(z2h.Z2HError):
            ctx.paged_plan(c.pages, x["heads"], x["rows"], x["rs"], x["kl"], x["groups"], x["gs"], i, x["ws"], x["n"])
    for bad in (dict(heads=3), dict(rows=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(type=z2h.BF16), dict(type=8),
                dict(q=0), dict(out=0), dict(qs=255), dict(os=255), dict(ws=0), dict(n=16), dict(q=p + 1), dict(out=p, os=300)):
        x = dict(heads=4, rows=2, scale=0.1, type=z2h.F16, q=p, qs=256, out=p + 1024, os=256, ws=ws, n=n)
        x.update(bad)
        with pytest.raises(z2h.Z2HError):
            ctx.paged_attn(c.pages, x["heads"], x["rows"], 0, x["scale"], x["type"], x["q"], x["qs"], x["out"], x["os"], x["ws"], x["n"])
    for field, value in (("page_rows", 24), ("head_dim", 48), ("type", 0), ("n_seq", 0), ("k", 0), ("page_stride", 8)):
        bad = z2h.Pages.from_buffer_copy(c.pages)
        setattr(bad, field, value)
        with pytest.raises(z2h.Z2HError):
            ctx.paged_ws_bytes(bad, 4, 2, 0)
    b = Attn(ctx, c, 4, [0], [20, 30], (), "f16")           # no rows: nothing to do
    b.row_start = ints([0, 0, 0])
    b.plan()
    b.run(d.view(2, -1), d.view(2, -1), 0.1)
    torch.cuda.synchronize()
