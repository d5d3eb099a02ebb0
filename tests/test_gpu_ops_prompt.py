"""z2h_prompt_attn against 64-bit attention: one row to long prompts, packed lengths around tiles, head groups, types, strides and
alignments, in place, rows of no sequence, values that are no numbers, streams, replayed graphs, and refusals."""
import math

import numpy as np
import pytest
import torch

from ops_helpers import DEV, TYPES, check, context, half_step, ints
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def reference(q, k, v, bounds, scale, dtype):
    """64-bit attention of q [rows][heads][hd] over k, v [rows][kv heads][hd] (host, float64) and a tolerance for a kernel of the given
    type; rows of no sequence are NaN in both.

    Per value, with p the softmax and A = sum p |v|: a score is a sum of hd products that are exact (16 bits) or rounded (fp32) and
    added in fp32, off by ds = scale (sum |q k|) 8 sqrt(hd) 2^-24 (a random walk of hd roundings, eight standard deviations' worth), which
    moves p by 2 ds relative (the weight and the sum). The exponent's argument (|s - max| up to 90) and the exponential round by
    94 * 2^-24. A weight meets the values to 2^-16 of it in bf16 (two numbers of 8 bits, the second's rounding left: 2^-9 * 2^-8 and a
    margin of 2) and 2^-21 in f16; fp32 weights are not rounded. The sums over n keys round like a random walk: 8 sqrt(n) 2^-24. The
    division: 2 * 2^-24. Then the output's own rounding."""
    R, nh, hd = q.shape
    grp = nh // k.shape[1]
    ref, tol = torch.full_like(q, math.nan), torch.full_like(q, math.nan)
    up = {torch.float32: 0.0, torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -16}[dtype]
    for a, b in zip(bounds[:-1], bounds[1:]):
        n = b - a
        if n <= 0:
            continue
        hidden = torch.ones((n, n), dtype=torch.bool).triu(1)
        seen = torch.arange(1, n + 1, dtype=torch.float64)
        for h in range(nh):
            qq, kk, vv = q[a:b, h], k[a:b, h // grp], v[a:b, h // grp]
            sc = (scale * (qq @ kk.T)).masked_fill(hidden, -math.inf)
            p = torch.softmax(sc, -1)
            ref[a:b, h] = p @ vv
            ds = abs(scale) * (qq.abs() @ kk.abs().T).masked_fill(hidden, 0).amax(-1) * 8 * math.sqrt(hd) * 2.0 ** -24
            rel = 2 * ds + 96 * 2.0 ** -24 + up + 8 * seen.sqrt() * 2.0 ** -24
            tol[a:b, h] = rel[:, None] * (p @ vv.abs())
    return ref, tol + half_step(ref, dtype) * (1 + 2.0 ** -10)


class Case:
    """Rows of a fused projection: queries, keys, values, and `pad` columns; `lead` elements before the first row."""

    def __init__(self, typ, lens, heads, kvh, hd, seed=0, pad=8, lead=0, qscale=1.0, extra=0, first=0):
        self.type, self.dtype = TYPES[typ]
        self.heads, self.kvh, self.hd, self.scale = heads, kvh, hd, hd ** -0.5
        self.bounds = [first, *(first + np.cumsum(lens)).tolist()]
        self.n = int(self.bounds[-1]) + extra
        self.width = (heads + 2 * kvh) * hd
        self.R = self.width + pad
        g = torch.Generator().manual_seed(seed)
        x = torch.randn((self.n, self.R), generator=g)
        x[:, :heads * hd] *= qscale
        self.host = x.to(self.dtype)
        self.lead = lead
        self.start = ints(self.bounds)

    def parts(self):
        x, nh, kvh, hd = self.host.double(), self.heads, self.kvh, self.hd
        return [t.reshape(self.n, -1, hd) for t in (x[:, :nh * hd], x[:, nh * hd:(nh + kvh) * hd], x[:, (nh + kvh) * hd:self.width])]

    def upload(self):
        flat = torch.zeros(self.lead + self.n * self.R + 8, dtype=self.dtype, device=DEV)
        flat[self.lead:self.lead + self.n * self.R] = self.host.reshape(-1).to(DEV)
        return flat

    def call(self, ctx, flat, out_ptr, out_stride, start=None, stream=None, scale=None):
        e, nh, kvh, hd = flat.element_size(), self.heads, self.kvh, self.hd
        p = flat.data_ptr() + self.lead * e
        ctx.prompt_attn(len(self.bounds) - 1, (self.start if start is None else start).data_ptr(), self.n, nh, kvh, hd,
                        self.scale if scale is None else scale, self.type, p, self.R, p + nh * hd * e, self.R, p + (nh + kvh) * hd * e, self.R,
                        out_ptr, out_stride, stream=stream)

    def run(self, ctx, stream=None):
        flat = self.upload()
        out = torch.full((self.n, self.heads * self.hd), 7.0, dtype=self.dtype, device=DEV)
        self.call(ctx, flat, out.data_ptr(), out.shape[1], stream=stream)
        torch.cuda.synchronize()
        return out.view(self.n, self.heads, self.hd)

    def check(self, out, what=""):
        ref, tol = reference(*self.parts(), self.bounds, float(np.float32(self.scale)), self.dtype)
        inside = ~torch.isnan(tol[:, 0, 0])
        check(out.cpu()[inside], ref[inside], tol[inside], what)
        assert bool((out.cpu()[~inside] == 7).all()), f"{what}: rows of no sequence were written"
        return ref, tol


LENS = [1, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 200, 2, 300]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", [(16, 4, 128), (8, 8, 64), (4, 1, 32), (14, 2, 128), (6, 2, 64), (64, 1, 64), (1, 1, 128), (24, 8, 32)])
def test_packed_lengths(ctx, typ, heads, kvh, hd):
    print(f"prompt {typ} heads {heads}/{kvh} hd {hd}", flush=True)
    c = Case(typ, LENS, heads, kvh, hd)
    c.check(c.run(ctx), typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 37, 511, 1025, 2600])
def test_one_prompt(ctx, typ, n):
    print(f"prompt {typ} n {n}", flush=True)
    c = Case(typ, [n], 4, 2, 128, seed=n)
    c.check(c.run(ctx), f"{typ} {n}")


@pytest.mark.parametrize("typ,hd", [("f32", 64), ("f16", 32), ("bf16", 128)])
def test_many_prompts(ctx, typ, hd):
    """More sequences than a wave has lanes, empty ones among them, first and last too."""
    rng = np.random.default_rng(1)
    lens = [0, 0] + [int(n) for n in rng.integers(0, 9, 200)] + [70, 0, 0]
    c = Case(typ, lens, 4, 2, hd)
    c.check(c.run(ctx), typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_few_heads_long_prompt(ctx, typ):
    """Fewer tiles than compute units: the keys are what there is to share out."""
    c = Case(typ, [1500, 40], 2, 1, 64)
    c.check(c.run(ctx), typ)


# sequences and heads at which a call is cut in each of its ways on this card: 16 row-heads per block, 128 with eight waves, 128 with four
CUTS = {"small": dict(lens=[90, 130, 40], heads=4, kvh=2), "pair": dict(lens=[1310], heads=16, kvh=4), "pair_f32": dict(lens=[1100, 1000], heads=16, kvh=8),
        "wide": dict(lens=[300, 1, 250, 77, 90, 33, 400, 180], heads=60, kvh=20)}


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cut", list(CUTS))
@pytest.mark.parametrize("hd,pad", [(128, 8), (64, 3), (32, 8)])
def test_every_cut(ctx, cut, typ, hd, pad):
    """Plain values, then a value that is not finite in the middle of the longest prompt's last rows."""
    print(f"prompt {cut} {typ} hd {hd}", flush=True)
    c = Case(typ, hd=hd, pad=pad, seed=3, **CUTS[cut])
    ref, tol = c.check(c.run(ctx), f"{cut} {typ}")
    s = int(np.argmax(CUTS[cut]["lens"]))
    end = c.bounds[s + 1]
    c.host[end - 3, (c.heads + c.kvh) * hd + 1] = math.inf
    c.host[end - 2, c.heads * hd] = math.nan
    out = c.run(ctx).cpu()
    rows = torch.ones(c.n, dtype=torch.bool)
    rows[end - 3:end] = False
    check(out[rows], ref[rows], tol[rows], f"{cut} {typ} rows that do not see them")
    grp = c.heads // c.kvh
    assert bool((out[end - 3, :grp, 1] == math.inf).all()) and bool(torch.isnan(out[end - 2:end, :grp]).all())
    assert bool(torch.isfinite(out[end - 3:end, grp:]).all())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_peaked(ctx, typ):
    """Scores far apart: softmax near one-hot, the running maximum moving often."""
    c = Case(typ, [300, 77], 4, 2, 64, qscale=20.0)
    c.check(c.run(ctx), typ)


def test_rising_scores(ctx):
    """Every key's score is above all before it by more than the maximum's slack, and the other way round."""
    for typ in ("f32", "f16", "bf16"):
        for sign in (1.0, -1.0):
            c = Case(typ, [400], 2, 1, 64)
            nh, hd = 2, 64
            c.host[:, :nh * hd] = 1.0
            ramp = sign * torch.arange(400, dtype=torch.float32)[:, None] * 0.25
            c.host[:, nh * hd:(nh + 1) * hd] = ramp.to(c.dtype)
            c.check(c.run(ctx), f"{typ} {sign}")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_strides_and_alignment(ctx, typ):
    """Rows at odd offsets with odd strides, 8-byte ones, and outputs in a wider row."""
    for pad, lead in ((5, 3), (4, 4), (8, 0), (3, 0), (8, 1)):
        c = Case(typ, [70, 5, 130], 4, 2, 64, pad=pad, lead=lead)
        flat = c.upload()
        out = torch.full((c.n, 263), 4.0, dtype=c.dtype, device=DEV)
        c.call(ctx, flat, out.data_ptr() + 5 * out.element_size(), 263)
        torch.cuda.synchronize()
        ref, tol = reference(*c.parts(), c.bounds, c.scale, c.dtype)
        check(out[:, 5:261].reshape(c.n, 4, 64), ref, tol, f"{typ} {pad} {lead}")
        assert bool((out[:, :5] == 4).all()) and bool((out[:, 261:] == 4).all())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[200, 3, 64], [1300]])
def test_in_place(ctx, typ, lens):
    c = Case(typ, lens, 4, 2, 64)
    want = c.run(ctx)
    flat = c.upload()
    c.call(ctx, flat, flat.data_ptr(), c.R)
    torch.cuda.synchronize()
    rows = flat[:c.n * c.R].view(c.n, c.R)
    assert torch.equal(rows[:, :256].reshape(c.n, 4, 64), want)
    assert torch.equal(rows[:, 256:].cpu(), c.host[:, 256:])


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[200, 3, 64], [1300]])
def test_in_place_with_values_that_are_not_finite(ctx, typ, lens):
    """Rows that are formed key by key read their queries while others are stored already."""
    c = Case(typ, lens, 8, 2, 64)
    a = (c.heads + c.kvh) * c.hd
    c.host[5::37, a + 3] = math.inf
    c.host[9::41, a + c.hd + 60] = -math.inf
    c.host[100, c.heads * c.hd + 7] = math.nan
    apart, flat = c.run(ctx), c.upload()
    c.call(ctx, flat, flat.data_ptr(), c.R)
    torch.cuda.synchronize()
    got = flat[:c.n * c.R].view(c.n, c.R)[:, :c.heads * c.hd].reshape(c.n, c.heads, c.hd)
    assert torch.equal(torch.isnan(got), torch.isnan(apart)) and bool(torch.isinf(apart).any()) and bool(torch.isnan(apart).any())
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(apart))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_rows_of_no_sequence(ctx, typ):
    """Rows before the first sequence and behind the last are left as they were, and what they hold reaches nobody."""
    c = Case(typ, [33, 100], 4, 2, 64, first=9, extra=50)
    c.host[:9] = math.nan
    c.host[c.bounds[-1]:] = math.nan
    c.check(c.run(ctx), typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [32, 128])
def test_no_numbers_in_later_rows_and_other_prompts(ctx, typ, hd):
    """NaN and infinities in the keys and values of a prompt's later rows and of other prompts: earlier rows as without them."""
    for bad in (math.nan, math.inf, -math.inf):
        c = Case(typ, [90, 130, 40], 4, 2, hd)
        ref, tol = reference(*c.parts(), c.bounds, float(np.float32(c.scale)), c.dtype)
        c.host[90 + 101, 4 * hd:] = bad                     # the middle prompt's row 101
        c.host[:90, 4 * hd:] = bad                          # the first one's all
        out = c.run(ctx).cpu()
        for rows in (slice(90, 90 + 101), slice(220, 260)):
            check(out[rows], ref[rows], tol[rows], f"{typ} {bad}")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_infinite_values_reach_the_rows_that_see_them(ctx, typ):
    c = Case(typ, [150, 20], 4, 2, 64)
    v = (4 + 2) * 64
    c.host[70, v + 5] = math.inf
    c.host[90, v + 64 + 9] = -math.inf
    c.host[100, v + 5] = -math.inf
    out = c.run(ctx)
    q, k, vv = c.parts()
    ref, tol = reference(q, k, vv, c.bounds, float(np.float32(c.scale)), c.dtype)
    # by the definition: a weight times infinity is infinity, both infinities together no number; columns of no infinity are untouched
    # (a product with the hidden rows' weight of 0 would have made them no numbers in `ref`)
    clean = vv.clone()
    clean[~torch.isfinite(clean)] = 0
    ref, tol = reference(q, k, clean, c.bounds, float(np.float32(c.scale)), c.dtype)
    ref[70:150, :2, 5] = math.inf
    ref[90:150, 2:, 9] = -math.inf
    ref[100:150, :2, 5] = math.nan
    check(out, ref, tol, typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[40, 300], [1200, 700]])
@pytest.mark.parametrize("hd", [32, 128])
def test_values_near_the_types_largest(ctx, typ, lens, hd):
    """Sums of weights times such values pass the largest number of fp32; their mean does not. (Rows formed key by key: every 64 keys the
    mean is scaled and its weights divided once more, three roundings of each, 3 sqrt(n / 64) 2^-24 times eight as a random walk, which
    the sums' 8 sqrt(n) 2^-24 of the tolerance holds beside their own 8 sqrt(64) 2^-24.)"""
    c = Case(typ, lens, 8, 2, hd, seed=hd)
    a, w = (c.heads + c.kvh) * hd, c.width
    big = torch.finfo(c.dtype).max / 2
    c.host[:, a:w] = (big * (1 + c.host[:, a:w].double().abs().remainder(0.5))).to(c.dtype)
    c.host[lens[0]:, a:w] *= -1
    c.host[:, a + 5] = 1.0
    c.check(c.run(ctx), f"{typ} {lens} {hd}")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_scores_that_are_no_numbers(ctx, typ):
    """A key whose score is minus infinity has no weight; infinity or NaN leaves the rows that see it without a number; a row that
    sees only minus infinities gives zeros."""
    c = Case(typ, [100], 2, 1, 64)
    c.host[:, :128] = c.host[:, :128].abs() + 0.5            # positive queries
    c.host[0, 128:192] = -math.inf                           # the first key: no weight for anyone
    c.host[40, 128:192] = math.inf                           # rows from 40 on have no number
    out = c.run(ctx).cpu()
    q, k, v = c.parts()
    ref, tol = reference(q[1:40], k[1:40], v[1:40], [0, 39], float(np.float32(c.scale)), c.dtype)
    check(out[1:40], ref, tol, typ)
    assert bool((out[0] == 0).all()) and bool(torch.isnan(out[40:]).all())


def test_scales(ctx):
    """Negative, zero, tiny and large factors; fp32 queries far from one."""
    for typ in ("f32", "f16", "bf16"):
        c = Case(typ, [130], 4, 2, 64)
        for scale in (-0.1, 0.0, 1e-30, 3.0):
            flat, out = c.upload(), torch.zeros((130, 256), dtype=c.dtype, device=DEV)
            c.call(ctx, flat, out.data_ptr(), 256, scale=scale)
            torch.cuda.synchronize()
            ref, tol = reference(*c.parts(), c.bounds, float(np.float32(scale)), c.dtype)
            check(out.view(130, 4, 64), ref, tol, f"{typ} {scale}")
    c = Case("f32", [100], 2, 1, 64)
    for s, scale in ((1e20, 1e-21), (1e-20, 1e19)):
        c.host[:, :128] = torch.randn((100, 128), generator=torch.Generator().manual_seed(3)) * s
        flat, out = c.upload(), torch.zeros((100, 128), device=DEV)
        c.call(ctx, flat, out.data_ptr(), 128, scale=scale)
        torch.cuda.synchronize()
        ref, tol = reference(*c.parts(), c.bounds, float(np.float32(scale)), c.dtype)
        check(out.view(100, 2, 64), ref, tol, f"{s}")


def test_offsets_beyond_32_bits(ctx):
    """Rows whose elements lie more than 2^31 apart."""
    n, stride, hd = 70, 1 << 25, 64
    c = Case("f16", [50, 20], 1, 1, hd)
    flat = torch.empty(n * stride, dtype=torch.float16, device=DEV)
    rows = flat.view(n, stride)
    rows[:, :3 * hd] = c.host[:, :3 * hd].to(DEV)
    p = flat.data_ptr()
    ctx.prompt_attn(2, c.start.data_ptr(), n, 1, 1, hd, c.scale, z2h.F16, p, stride, p + 2 * hd, stride, p + 4 * hd, stride, p + 6 * hd, stride)
    torch.cuda.synchronize()
    ref, tol = reference(*c.parts(), c.bounds, c.scale, c.dtype)
    check(rows[:, 3 * hd:4 * hd].reshape(n, 1, hd), ref, tol)


def test_bad_row_tables_stay_inside(ctx):
    """Entries out of range are clamped; descending ones give some values in their rows and never leave the buffers."""
    c = Case("f16", [40, 30, 30], 4, 2, 64)
    c.bounds = [0, 40, 70, 100]
    flat, out = c.upload(), torch.full((100, 256), 7.0, dtype=torch.float16, device=DEV)
    wide = ints([-5, 40, 70, 10 ** 6])
    c.call(ctx, flat, out.data_ptr(), 256, start=wide)
    torch.cuda.synchronize()
    c.check(out.view(100, 4, 64))
    guard = torch.full((300, 256), 7.0, dtype=torch.float16, device=DEV)
    for table in ([90, 20, 60, 10], [100, 0, 0, 0], [50, 50, 50, 50], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -1]):
        bad = ints(table)
        c.call(ctx, flat, guard.data_ptr() + 100 * 512, 256, start=bad)
        torch.cuda.synchronize()
    assert bool((guard[:100] == 7).all()) and bool((guard[200:] == 7).all())


def test_streams_graphs_and_repeats(ctx):
    """Two calls at once on two streams, a captured call replayed on new rows, and many repeats: bit for bit."""
    cases = [Case("bf16", [700, 33, 1], 16, 4, 128, seed=1), Case("f32", [260, 100], 8, 2, 64, seed=2)]
    want = [c.run(ctx) for c in cases]
    flats, outs = [c.upload() for c in cases], [torch.zeros_like(w) for w in want]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, c, f, o in zip(streams, cases, flats, outs):
            c.call(ctx, f, o.data_ptr(), c.heads * c.hd, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(w, o) for w, o in zip(want, outs))
    c, f, o = cases[0], flats[0], outs[0]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        c.call(ctx, f, o.data_ptr(), c.heads * c.hd, stream=side.cuda_stream)
    for seed, lens in ((5, [700, 33, 1]), (6, [1, 400, 333]), (7, [0, 734, 0])):
        d = Case("bf16", lens, 16, 4, 128, seed=seed)
        f[:d.n * d.R] = d.host.reshape(-1).to(DEV)
        c.start.copy_(d.start)
        o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, d.run(ctx))
        torch.randn(1000, device=DEV).sum().item()


def test_refusals_and_nothing_to_do(ctx):
    c = Case("f16", [20, 30], 4, 2, 64)
    flat, out = c.upload(), torch.full((50, 256), 3.0, dtype=torch.float16, device=DEV)
    p, o = flat.data_ptr(), out.data_ptr()
    good = dict(n_seq=2, start=c.start.data_ptr(), n=50, heads=4, kvh=2, hd=64, scale=0.1, type=z2h.F16, q=p, qs=c.R, k=p + 512, ks=c.R,
                v=p + 768, vs=c.R, out=o, os=256)
    call = lambda x: ctx.prompt_attn(x["n_seq"], x["start"], x["n"], x["heads"], x["kvh"], x["hd"], x["scale"], x["type"], x["q"], x["qs"], x["k"],
                                     x["ks"], x["v"], x["vs"], x["out"], x["os"])
    for bad in (dict(heads=3), dict(heads=0), dict(heads=260), dict(kvh=0), dict(hd=48), dict(hd=256), dict(n=-1), dict(n_seq=-1), dict(n=1 << 26),
                dict(scale=math.nan), dict(scale=math.inf), dict(type=8), dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(qs=255), dict(ks=127),
                dict(vs=127), dict(os=255), dict(q=p + 1), dict(out=p, os=256), dict(start=0), dict(n_seq=1 << 24)):
        with pytest.raises(z2h.Z2HError):
            call({**good, **bad})
    for none in (dict(n=0), dict(n_seq=0), dict(n=0, q=0, k=0, v=0, out=0, start=0)):
        call({**good, **none})
    torch.cuda.synchronize()
    assert bool((out == 3).all())
