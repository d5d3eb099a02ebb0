"""z2h_paged_plan / z2h_paged_attn where they are easily wrong: infinities in the cache, wherever they lie and whatever way their keys are
walked (a piece that stores its rows itself, pieces that are joined, tiles of one wave and of four); and how near the results come."""
import math

import numpy as np
import pytest
import torch

from ops_cut_cases import CASES
from ops_helpers import DEV, TYPES, Attn, Cache, check, context, half_step
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu
INF = float("inf")
UP = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step of a weight as it meets the values


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def reference(cache, q, row_start, kv_len, scale, dtype, up=None):
    """64-bit attention and the tolerance that ops_helpers.attention derives, by products over a sequence's rows at once. A key with a score
    of minus infinity has no weight; a value that is not finite reaches the rows that see it whatever its weight."""
    R, nh, hd = q.shape
    kvh, grp = cache.kvh, nh // cache.kvh
    up = UP[dtype] if up is None else up
    uq = 2.0 ** -21 if dtype == torch.float32 else 0.0
    ref, tol = torch.zeros_like(q), torch.zeros_like(q)
    for s in range(len(kv_len)):
        r0, m, n = int(row_start[s]), int(row_start[s + 1] - row_start[s]), int(kv_len[s])
        if m == 0 or n == 0:
            continue
        k, v = (t.transpose(0, 1).contiguous() for t in cache.rows(s, n))                 # [kvh][n][hd]
        x = q[r0:r0 + m].reshape(m, kvh, grp, hd).transpose(0, 1).reshape(kvh, m * grp, hd)
        see = (n - m + torch.arange(m) + 1).clamp(min=0).repeat_interleave(grp)            # cache rows that each row sees
        hidden = torch.arange(n)[None, :] >= see[:, None]
        sc = scale * torch.matmul(x, k.transpose(1, 2).contiguous())
        size = torch.matmul(x.abs(), torch.nan_to_num(k, 0.0, 0.0, 0.0).abs().transpose(1, 2).contiguous())
        sc = sc.masked_fill(hidden, -INF)
        p = torch.nan_to_num(torch.softmax(sc, -1), 0.0) if bool((see == 0).any()) else torch.softmax(sc, -1)
        v0 = torch.nan_to_num(v, 0.0, 0.0, 0.0)
        o = torch.matmul(p, v0)
        shown = (~hidden).double()
        for bad, sign in (((v == INF) | v.isnan(), INF), ((v == -INF) | v.isnan(), -INF)):
            if bool(bad.any()):
                o = torch.where(torch.matmul(shown, bad.double()) > 0, o + sign, o)
        ds = abs(scale) * size.masked_fill(hidden, 0.0).amax(-1) * (8 * 2.0 ** -24 * math.sqrt(hd) + uq)
        rel = 2 * ds + 94 * 2.0 ** -24 + up + 8 * torch.sqrt(see.double()) * 2.0 ** -24
        t = rel[..., None] * torch.matmul(torch.nan_to_num(p, 0.0), v0.abs())
        for dst, val in ((ref, o), (tol, t)):
            dst[r0:r0 + m] = val.reshape(kvh, m, grp, hd).transpose(0, 1).reshape(m, nh, hd)
    return ref, tol + half_step(torch.nan_to_num(ref, 0.0, 0.0, 0.0), dtype) * (1 + 2.0 ** -10)


def case(typ, lens, rows, heads, kvh, hd, page, groups=(), seed=0, qscale=1.0, **cache):
    dtype = TYPES[typ][1]
    c = Cache(lens, kvh, hd, page, torch.bfloat16 if typ == "bf16" else torch.float16, seed + 1, shared=groups, **cache)
    row_start = np.concatenate([[0], np.cumsum(rows)]).astype(int)
    g = torch.Generator().manual_seed(seed + 2)
    return c, row_start, (torch.randn((int(row_start[-1]), heads, hd), generator=g) * qscale).to(dtype)


def run(ctx, typ, c, row_start, q, lens, groups=(), scale=0.125, in_place=False):
    a = Attn(ctx, c, q.shape[1], row_start, lens, groups, typ)
    d = q.to(DEV)
    out = d if in_place else torch.full_like(d, 7.0)
    a.plan()
    a.run(d.view(len(d), -1), out.view(len(d), -1), scale)
    torch.cuda.synchronize()
    return out


# ---- infinities in the cache
SHAPES = {
    # one piece that stores its rows, two pieces, several
    "few": dict(lens=[40, 70, 300], rows=[2, 6, 1], heads=4, kvh=2, hd=64, page=16, groups=()),
    # a shared prefix for 160 row-heads of each key head: a tile of four waves, one of a wave, and the sequences' own keys
    "shared": dict(lens=[300 + s % 40 for s in range(1, 41)], rows=[1] * 40, heads=8, kvh=2, hd=128, page=16, groups=[(0, 40, 300)]),
    # whole prompts: tiles of four waves whose rows see more and more
    "prompt": dict(lens=[150], rows=[150], heads=4, kvh=2, hd=32, page=16, groups=()),
}


def _infinite(ctx, typ, shape, qscale, poison, change=None, in_place=False):
    print(f"infinite {typ} {shape} {qscale} {poison}", flush=True)
    p = SHAPES[shape]
    c, row_start, q = case(typ, **p, seed=11, qscale=qscale)
    if change is not None:
        change(q)
    for which, seq, key, head, dim, value in poison:
        c.cell(which, seq, key)[head, dim] = value
    c.upload()
    ref, tol = reference(c, q.double(), row_start, p["lens"], 0.125, q.dtype)
    check(run(ctx, typ, c, row_start, q, p["lens"], p["groups"], in_place=in_place), ref, tol, typ)
    return ref


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("qscale", [1.0, 30.0])             # (30: most weights are below what f16 holds)
def test_infinite_values_wherever_they_lie(ctx, typ, shape, qscale):
    ref = _infinite(ctx, typ, shape, qscale, [(1, 0, 0, 0, 1, INF), (1, 0, 3, 0, 5, INF), (1, 0, 20, 1, 9, -INF), (1, 0, 7, 1, 11, INF),
                                              (1, 0, 33, 1, 11, -INF), (1, 0, 39, 0, 2, INF), (1, 0, 12, 0, 30, float("nan"))])
    assert torch.isinf(ref).any() and torch.isnan(ref).any() and torch.isfinite(ref).any()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_infinite_values_in_place(ctx, typ, shape):
    _infinite(ctx, typ, shape, 3.0, [(1, 0, 2, 0, 5, INF), (1, 0, 30, 1, 9, -INF)], in_place=True)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_infinite_keys(ctx, typ, shape):
    """A row whose component there has the other sign gives the key no weight, one with the same sign (or 0) has no answer."""
    def change(q):
        q[0, 0, 7], q[0, 1, 7], q[1, :, 7] = 0.0, -1e-30 if q.dtype == torch.float32 else -1e-4, -0.5
    ref = _infinite(ctx, typ, shape, 1.0, [(0, 0, 3, 0, 7, INF), (0, 0, 25, 1, 6, -INF)], change)
    assert torch.isnan(ref).any() and torch.isfinite(ref).any()
    assert typ != "f32" or torch.isfinite(ref[0, 1]).all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_infinite_keys_and_values(ctx, typ):
    def change(q):
        q[..., 7] = -q[..., 7].abs() - 0.01
    ref = _infinite(ctx, typ, "shared", 1.0, [(0, 0, 3, 0, 7, INF), (0, 0, 150, 1, 7, INF), (1, 0, 200, 0, 4, INF), (1, 0, 64, 1, 4, -INF)], change)
    assert not torch.isnan(ref).any() and torch.isinf(ref).any()


@pytest.mark.parametrize("typ", ["f32", "f16"])
def test_infinities_with_large_queries_and_a_negative_scale(ctx, typ):
    """Scores formed once more keep to the range of the queries and to the scale's sign."""
    p = SHAPES["few"]
    c, row_start, q = case(typ, **p, seed=12)
    big = 1e30 if typ == "f32" else 1e3
    q *= big
    c.cell(1, 1, 5)[:, 3] = INF
    c.upload()
    scale = float(np.float32(-0.125 / big))
    ref, tol = reference(c, q.double(), row_start, p["lens"], scale, q.dtype)
    check(run(ctx, typ, c, row_start, q, p["lens"], scale=scale), ref, tol, typ)


# ---- how near 16-bit results come: the output's own rounding, and next to it what fp32 sums leave
# A weight is carried as two numbers of the cache's type: off by half a step of half a step, 2^-22 of it in f16 and 2^-16 in bf16. In f16 the second
# part is below the normal range where the weight is below 2^-3, and then off by 2^-25 at most; the largest weight is 2^6 or more, so n keys add
# n 2^-31 of the largest value.
TWO = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}


def below_normal(c, q, lens):
    return 0.0 if q.dtype == torch.bfloat16 else max(lens) * 2.0 ** -31 * float(torch.nan_to_num(c.buf[1], 0.0).abs().max())


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("shape", list(SHAPES) + ["long", "wide"])
@pytest.mark.parametrize("qscale", [0.01, 1.0, 5.0])        # (weights all alike, as they usually are, and peaked)
def test_16_bit_results_have_the_outputs_rounding_only(ctx, typ, shape, qscale):
    p = SHAPES.get(shape) or {"long": dict(lens=[4097, 1000], rows=[1, 3], heads=8, kvh=2, hd=128, page=64, groups=()),
                              "wide": dict(lens=[1500] * 33, rows=[1] * 33, heads=16, kvh=4, hd=64, page=32, groups=[(0, 33, 1480)])}[shape]
    print(f"rounding {typ} {shape} {qscale}", flush=True)
    c, row_start, q = case(typ, **p, seed=21, qscale=qscale)
    ref, tol = reference(c, q.double(), row_start, p["lens"], 0.125, q.dtype, up=TWO[q.dtype])
    tol += below_normal(c, q, p["lens"])
    out = run(ctx, typ, c, row_start, q, p["lens"], p["groups"])
    check(out, ref, tol, typ)
    mine, least = (float((x.double().cpu() - ref).square().mean().sqrt()) for x in (out, ref.to(q.dtype)))
    assert mine <= 1.01 * least                             # (some values on a border between two steps go to the other one)


# ---- no groups: both tables NULL
def test_no_groups_without_tables(ctx):
    lens, rows = [40, 300, 17], [1, 3, 0]
    c, row_start, q = case("f16", lens, rows, 8, 2, 64, 16, seed=31)
    a = Attn(ctx, c, 8, row_start, lens, (), "f16")
    d = q.to(DEV)
    out = torch.zeros_like(d)
    for _ in range(2):
        a.ctx.paged_plan(c.pages, 8, a.R, a.row_start.data_ptr(), a.kv_len.data_ptr(), 0, 0, 0, a.ws.data_ptr(), a.ws.numel())
        a.run(d.view(len(d), -1), out.view(len(d), -1), 0.125)
        torch.cuda.synchronize()
        check(out, *reference(c, q.double(), row_start, lens, 0.125, q.dtype), "no groups")


# ---- tables that go back would put a row into several spans: no plan, and the output stays as it was
def test_tables_that_are_not_ascending_make_no_plan(ctx):
    lens, rows = [40, 60, 17, 90], [2, 3, 1, 2]
    c, row_start, q = case("f16", lens, rows, 8, 2, 64, 16, seed=32)
    d = q.to(DEV)
    groups = [(0, 2, 32), (2, 4, 16)]
    for field, bad in (("row_start", [0, 5, 2, 6, 8]), ("row_start", [0, 2, 5, 100, 8]), ("group_start", [0, 3, 2]), ("group_start", [2, 0, 4])):
        a = Attn(ctx, c, 8, row_start, lens, groups, "f16")
        good = getattr(a, field).clone()
        setattr(a, field, torch.tensor(bad, dtype=torch.int32, device=DEV))
        out = torch.full_like(d, 7.0)
        a.plan()
        a.run(d.view(len(d), -1), out.view(len(d), -1), 0.125)
        torch.cuda.synchronize()
        assert bool((out == 7).all()), (field, bad)
        setattr(a, field, good)                             # the same workspace, planned again
        a.plan()
        a.run(d.view(len(d), -1), out.view(len(d), -1), 0.125)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(out).all()) and not bool((out == 7).any())


# ---- calls that small ones do not stand for (what each reaches is checked on the CPU)
def _cut_case(name):
    p = {k: v for k, v in CASES[name].items() if k not in ("name", "reaches")}
    print(f"cut: {name}", flush=True)
    return p, case(**p, seed=41)


@pytest.mark.parametrize("name", list(CASES))
def test_long_and_many(ctx, name):
    p, (c, row_start, q) = _cut_case(name)
    scale = float(np.float32(p["hd"] ** -0.5))
    ref, tol = reference(c, q.double(), row_start, p["lens"], scale, q.dtype, up=TWO[q.dtype])
    check(run(ctx, p["typ"], c, row_start, q, p["lens"], p["groups"], scale), ref, tol + below_normal(c, q, p["lens"]), name)


@pytest.mark.parametrize("name", [n for n in CASES if n.startswith("long walks") or "in a row" in n])
def test_long_walks_repeat_bit_for_bit(ctx, name):
    """Keys and values pass through LDS in many steps, which waves that have nothing to multiply help to fill: no answer depends on who
    came first."""
    p, (c, row_start, q) = _cut_case(name)
    a = Attn(ctx, c, p["heads"], row_start, p["lens"], p["groups"], p["typ"])
    d = q.to(DEV)
    outs = [torch.empty_like(d) for _ in range(30)]
    a.plan()
    for o in outs:
        a.run(d.view(len(d), -1), o.view(len(d), -1), p["hd"] ** -0.5)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(outs[0]).all()) and all(torch.equal(o, outs[0]) for o in outs)


def test_a_billion_rows_per_sequence(ctx):
    """The longest sequences that a table may describe, over two pages again and again: lengths near 2^30, and more steps in the call than are
    counted one by one. A piece adds up 2^17 steps one after the other, their sums by 2^17 roundings of at most 2^-24 of what has come together (half
    of it on average), the values by four times as many: 2^-8 and 2^-6 of a result whose values are all positive."""
    P, hd, S = 4096, 32, 8
    g = torch.Generator().manual_seed(5)
    c = Cache([P, P], 1, hd, P, torch.float16, 6)
    pages = [int(c.table_host[s, 0]) for s in range(2)]
    for i, page in enumerate(pages):
        c.buf[1][page] = (torch.rand(P * hd, generator=g) + 1 + 2 * i).half()
    per = (1 << 30) // P
    turn = [(s + 1) * per // 10 for s in range(S)]          # the page from which on a sequence has the second one
    c.table_host = np.where(np.arange(per)[None] < np.array(turn)[:, None], pages[0], pages[1]).astype(np.int32)
    c.upload()
    lens = [(1 << 30) - 37 * s for s in range(S)]
    q = torch.randn((S, 1, hd), generator=g).half()
    out = run(ctx, "f16", c, np.arange(S + 1), q, lens)
    k, v = ([b[p].view(P, hd).double() for p in pages] for b in c.buf)
    for s in range(S):
        w = [torch.exp(0.125 * (x @ q[s, 0].double())) for x in k]
        last = lens[s] - (per - 1) * P                      # rows of the last page
        some = [torch.full((P,), float(turn[s]), dtype=torch.float64), torch.full((P,), float(per - 1 - turn[s]), dtype=torch.float64)]
        some[1][:last] += 1
        ref = sum((n * x) @ y for n, x, y in zip(some, w, v)) / sum((n * x).sum() for n, x in zip(some, w))
        err = ((out[s, 0].double().cpu() - ref).abs() / ref).max()
        print(f"sequence {s}: off by {float(err):.2e}", flush=True)
        assert float(err) <= 2.0 ** -8 + 2.0 ** -6 + 2.0 ** -11


# ---- no rows: tensors of no elements have no address
def test_no_rows_without_tensors(ctx):
    c, row_start, q = case("f16", [20, 30], [0, 0], 4, 2, 64, 16, seed=33)
    old = [b.clone() for b in c.dev]
    rope = z2h.Rope(n_dims=64)
    ctx.rope_rows(rope, 0, 4, 64, z2h.F16, 0, 256, 0, 256, 0)
    ctx.paged_append(c.pages, rope, 0, 0, 0, z2h.F16, 0, 128, 0, 128, 4, 0, 256, 0, 256)
    a = Attn(ctx, c, 4, row_start, [20, 30], (), "f16")
    empty = torch.empty((0, 256), dtype=torch.float16, device=DEV)
    assert empty.data_ptr() == 0
    a.plan()
    a.run(empty, empty, 0.125)
    ctx.verify(0, 2, 1, 10, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    torch.cuda.synchronize()
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(old, c.dev))
    for call in (lambda: ctx.rope_rows(rope, 0, 0, 64, z2h.F16, 0, 256, 0, 256, 0), lambda: ctx.rope_rows(rope, 0, 4, 64, z2h.F16, 0, 255, 0, 256, 0),
                 lambda: ctx.verify(0, 2, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)):
        with pytest.raises(z2h.Z2HError):
            call()
