"""z2h_rope_rows and z2h_paged_append against 64-bit rotations: layouts, partial heads, context scaling, far positions, types,
strides, pages that end inside a chunk, padded rows and bad table entries, in place, another stream, a replayed graph."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, TYPES, Cache, check, context, half_step, ints, rotate, rotate_tol
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu

PLAIN = dict(factor=1.0, low=0.0, high=0.0, orig=0, mscale=1.0)
LINEAR = dict(PLAIN, factor=4.0)
PARTS = dict(factor=8.0, low=1.0, high=32.0, orig=4096, mscale=1.25)


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def _rope(base, dims, halves, sc):
    return z2h.Rope(base=base, n_dims=dims, halves=int(halves), factor=sc["factor"], low_turns=sc["low"], high_turns=sc["high"],
                    orig_ctx=sc["orig"], mscale=sc["mscale"])


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("halves", [False, True], ids=["pairs", "halves"])
@pytest.mark.parametrize("rows,heads,hd,dims,sc", [
    (1, 1, 32, 32, PLAIN), (16, 16, 128, 128, PLAIN), (7, 3, 64, 64, LINEAR), (5, 2, 128, 96, PARTS), (33, 5, 64, 30, PARTS),
    (3, 2, 64, 2, PLAIN), (2, 2, 32, 0, PLAIN), (9, 40, 128, 64, PARTS), (4, 2, 80, 20, PLAIN), (300, 8, 128, 128, LINEAR),
    (3, 2, 6, 4, PLAIN)])
def test_rope_rows(ctx, typ, halves, rows, heads, hd, dims, sc):
    print(f"rope {typ} {halves} {rows} {heads} {hd} {dims}", flush=True)
    code, dtype = TYPES[typ]
    g = torch.Generator().manual_seed(rows * 1000 + hd + dims)
    x = torch.randn((rows, heads, hd), generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g)
    pos[0] = 0
    base = 500000.0 if sc is PARTS else 10000.0
    ref = rotate(x.double(), pos, base, dims, halves, **sc)
    tol = rotate_tol(x.double(), ref, dims, halves, sc["mscale"], dtype)
    d, out, p = x.to(DEV), torch.full(x.shape, float("nan"), dtype=dtype, device=DEV), ints(pos)
    r = _rope(base, dims, halves, sc)
    ctx.rope_rows(r, rows, heads, hd, code, d.data_ptr(), heads * hd, out.data_ptr(), heads * hd, p.data_ptr())
    torch.cuda.synchronize()
    check(out, ref, tol, "rows")
    ctx.rope_rows(r, rows, heads, hd, code, d.data_ptr(), heads * hd, d.data_ptr(), heads * hd, p.data_ptr())   # in place
    torch.cuda.synchronize()
    assert torch.equal(d, out)


def test_rope_rows_strided_and_far(ctx):
    """Rows inside wider ones at an odd element offset, positions up to 2^31 - 1 and negative ones."""
    code, dtype = TYPES["f16"]
    g = torch.Generator().manual_seed(5)
    wide = torch.randn((6, 3 * 64 + 9), generator=g).to(dtype)
    pos = torch.tensor([2**31 - 1, 123456789, 5, -7, 0, -2**31])
    ref = rotate(wide[:, 3:195].reshape(6, 3, 64).double(), pos, 10000.0, 64, True)
    d = wide.to(DEV)
    out = torch.full((6, 250), 7.0, dtype=dtype, device=DEV)
    dpos = ints(pos)
    ctx.rope_rows(_rope(10000.0, 64, True, PLAIN), 6, 3, 64, code, d.data_ptr() + 6, 201, out.data_ptr() + 2, 250, dpos.data_ptr())
    torch.cuda.synchronize()
    check(out[:, 1:193].reshape(6, 3, 64), ref, rotate_tol(wide[:, 3:195].reshape(6, 3, 64).double(), ref, 64, True, 1.0, dtype))
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 193:] == 7).all()) and torch.equal(d.cpu(), wide)


# rotating back by the same positions (the rotation's transpose, so its gradient) gives the rows again
def test_rope_rows_transpose(ctx):
    g = torch.Generator().manual_seed(6)
    x = torch.randn((12, 4, 64), generator=g)
    pos = torch.randint(0, 100000, (12,), generator=g)
    r = _rope(10000.0, 48, True, PLAIN)
    d = x.to(DEV)
    there, back = ints(pos), ints(-pos)
    for p in (there, back):
        ctx.rope_rows(r, 12, 4, 64, z2h.F32, d.data_ptr(), 256, d.data_ptr(), 256, p.data_ptr())
    torch.cuda.synchronize()
    tol = 2 * rotate_tol(x.double(), x.double(), 48, True, 1.0, torch.float32) * 2 ** 0.5
    check(d, x.double(), tol)


@pytest.mark.parametrize("typ,cache_type", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("kvh,heads,hd,dims,page,halves,pad", [
    (1, 1, 32, 32, 16, False, 0), (4, 16, 128, 128, 16, False, 2), (2, 6, 64, 30, 32, True, 1), (8, 8, 128, 64, 64, True, 3),
    (3, 0, 64, 64, 16, True, 0)])
def test_paged_append(ctx, typ, cache_type, kvh, heads, hd, dims, page, halves, pad):
    print(f"append {typ} {cache_type} {kvh} {heads} {hd} {dims} {page}", flush=True)
    code, dtype = TYPES[typ]
    ctype = TYPES[cache_type][1]
    lens = [0, 15, 16, 33, 100]
    c = Cache(lens, kvh, hd, page, ctype, 3, room=40, stride_pad=8 * pad)
    g = torch.Generator().manual_seed(9)
    # chunks that start in the middle of a page and cross its end, one row each for others, padded rows between them
    seq = [0] * 37 + [1] + [-1] * pad + [2, 3] + [4] * 20 + [len(lens)] * pad
    pos = list(range(37)) + [15] + [3] * pad + [16, 33] + list(range(100, 120)) + [0] * pad
    n = len(seq)
    w = (heads + 2 * kvh) * hd + 8                          # one fused row: queries, keys, values, something else
    x = torch.randn((n, w), generator=g).to(dtype)
    d = x.to(DEV)
    qo = torch.full((n, heads * hd + 4), 5.0, dtype=dtype, device=DEV)
    e = d.element_size()
    r = _rope(10000.0, dims, halves, PARTS)
    dseq, dpos = ints(seq), ints(pos)
    ctx.paged_append(c.pages, r, n, dseq.data_ptr(), dpos.data_ptr(), code, d.data_ptr() + heads * hd * e, w,
                     d.data_ptr() + (heads + kvh) * hd * e, w, heads, d.data_ptr() if heads else 0, w,
                     qo.data_ptr() if heads else 0, heads * hd + 4)
    torch.cuda.synchronize()
    live = torch.tensor([0 <= s < len(lens) for s in seq])
    tpos = torch.tensor(pos)
    q, k, v = x[:, :heads * hd].reshape(n, heads, hd), x[:, heads * hd:(heads + kvh) * hd].reshape(n, kvh, hd), \
        x[:, (heads + kvh) * hd:(heads + 2 * kvh) * hd].reshape(n, kvh, hd)
    if heads:
        ref = rotate(q.double(), tpos, 10000.0, dims, halves, **PARTS)
        tol = rotate_tol(q.double(), ref, dims, halves, PARTS["mscale"], dtype)
        ref[~live] = 5.0
        check(qo[:, :heads * hd].reshape(n, heads, hd), ref, tol, "queries")
        assert bool((qo[:, heads * hd:] == 5).all())
    kr = rotate(k.double(), tpos, 10000.0, dims, halves, **PARTS)
    kt = rotate_tol(k.double(), kr, dims, halves, PARTS["mscale"], ctype)
    before = [b.clone() for b in c.buf]
    tols = [torch.zeros(b.shape, dtype=torch.float64) for b in c.buf]
    want = [b.double() for b in c.buf]
    size = kvh * page * hd
    for i in range(n):
        if live[i]:
            at = c.table_host[seq[i], pos[i] // page]
            for t, (val, lim) in enumerate(((kr[i], kt[i]), (v[i].double(), half_step(v[i].double(), ctype)))):
                want[t][at, :size].view(kvh, page, hd)[:, pos[i] % page] = val
                tols[t][at, :size].view(kvh, page, hd)[:, pos[i] % page] = lim
    for t in range(2):
        check(c.dev[t], want[t], tols[t], "kv"[t])           # every other row as it was (tolerance 0, NaN kept)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(before, c.buf))


def test_append_bad_entries_leave_the_cache(ctx):
    """Positions behind the table, negative ones and pages out of range: no cache row changes, queries are rotated."""
    c = Cache([64, 64], 2, 64, 16, torch.float16, 4, fill=1.0)
    c.table_host[1, 2], c.table_host[1, 3] = -5, 1 << 28
    c.upload()
    seq, pos = [0, 0, 1, 1, 0, 7, -3], [64, -1, 32, 63, 2**31 - 1, 0, 0]
    g = torch.Generator().manual_seed(2)
    x = torch.randn((7, 2, 64), generator=g).half()
    d, qo = x.to(DEV), torch.full((7, 2, 64), 9.0, dtype=torch.float16, device=DEV)
    old = [b.clone() for b in c.dev]
    dseq, dpos = ints(seq), ints(pos)
    ctx.paged_append(c.pages, _rope(10000.0, 64, False, PLAIN), 7, dseq.data_ptr(), dpos.data_ptr(), z2h.F16, d.data_ptr(), 128,
                     d.data_ptr(), 128, 2, d.data_ptr(), 128, qo.data_ptr(), 128)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(old, c.dev))
    ref = rotate(x.double(), torch.tensor(pos), 10000.0, 64, False)
    tol = rotate_tol(x.double(), ref, 64, False, 1.0, torch.float16)
    ref[5:] = 9.0
    check(qo, ref, tol)


def test_append_on_a_stream_and_in_a_replayed_graph(ctx):
    """A captured append reads new rows and positions at each replay; the same values as an eager call on the null stream."""
    caches = [Cache([40, 70], 2, 64, 16, torch.float16, 8, room=30, fill=0.0) for _ in range(2)]
    r = _rope(10000.0, 64, True, PLAIN)
    g = torch.Generator().manual_seed(3)
    x, seq, pos = torch.zeros((2, 3, 2, 64), device=DEV), ints([0, 1]), ints([0, 0])
    q = torch.zeros((2, 2, 64), device=DEV)

    def call(c, out, stream):
        ctx.paged_append(c.pages, r, 2, seq.data_ptr(), pos.data_ptr(), z2h.F32, x.data_ptr() + 512, 384, x.data_ptr() + 1024, 384, 2,
                         x.data_ptr(), 384, out.data_ptr(), 128, stream=stream)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        call(caches[0], q, side.cuda_stream)
    for step in range(4):
        x.copy_(torch.randn(x.shape, generator=g))
        pos.copy_(torch.tensor([40 + step, 70 + step]))
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(q)
        call(caches[1], eager, 0)
        torch.cuda.synchronize()
        assert torch.equal(q, eager) and all(torch.equal(a, b) for a, b in zip(caches[0].dev, caches[1].dev))


def test_refusals(ctx):
    c = Cache([16], 1, 32, 16, torch.float16, 1)
    t = torch.zeros((4, 64), device=DEV)
    zeros = ints([0] * 4)
    p, i = t.data_ptr(), zeros.data_ptr()
    ok = _rope(10000.0, 32, False, PLAIN)
    for bad in (dict(rope=_rope(10000.0, 34, False, PLAIN)), dict(rope=_rope(0.0, 32, False, PLAIN)), dict(n=-1), dict(heads=0),
                dict(type=8), dict(stride=31), dict(x=0), dict(out=0), dict(pos=0), dict(x=p + 2), dict(in_place=True)):
        a = dict(rope=ok, n=4, heads=1, type=z2h.F32, stride=32, x=p, out=p + 512, pos=i, in_place=False)
        a.update(bad)
        with pytest.raises(z2h.Z2HError):
            ctx.rope_rows(a["rope"], a["n"], a["heads"], 32, a["type"], a["x"], a["stride"], a["x"] if a["in_place"] else a["out"],
                          33 if a["in_place"] else 32, a["pos"])
    for bad in (dict(k=0), dict(v=0), dict(seq=0), dict(pos=0), dict(type=8), dict(q_out=0), dict(heads=0), dict(ks=31)):
        a = dict(k=p, v=p, seq=i, pos=i, type=z2h.F32, q_out=p + 512, heads=1, ks=32)
        a.update(bad)
        with pytest.raises(z2h.Z2HError):
            ctx.paged_append(c.pages, ok, 4, a["seq"], a["pos"], a["type"], a["k"], a["ks"], a["v"], 32, a["heads"], p, 32, a["q_out"], 32)
    ctx.rope_rows(ok, 0, 1, 32, z2h.F32, p, 32, p + 512, 32, i)                       # no rows: nothing to do
    ctx.paged_append(c.pages, ok, 0, i, i, z2h.F32, p, 32, p, 32)
