"""z2h_moe_rows against a 64-bit restatement: routing by hand, ties, masked experts, rows without experts, the products at odd and
large widths, types, strides, in place, rows that hold no numbers, streams, replayed graphs, and refusals."""
import math

import numpy as np
import pytest
import torch

from ops_helpers import DEV, TYPES, check, context, half_step
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def route(logits, bias, k, renorm):
    """logits [n][E] float64: (experts, weights) of every row, in the order of the definition."""
    sels, ws = [], []
    for z in logits:
        sel, w = np.full(k, -1), np.zeros(k)
        if np.isnan(z).any() or (z == np.inf).any() or (bias is not None and np.isnan(bias).any()):
            w[:] = np.nan
        elif (z > -np.inf).any():
            e = np.exp(z - z.max())
            p = e / e.sum()
            score = np.where(z > -np.inf, p + bias if bias is not None else z, -np.inf)
            order = [i for i in np.argsort(-score, kind="stable") if z[i] > -np.inf][:k]
            sel[:len(order)] = order
            w[:len(order)] = p[order] / (p[order].sum() if renorm else 1.0)
        sels.append(sel), ws.append(w)
    return np.array(sels), np.array(ws)


def layer(x, gate, up, down, sel, w, dtype):
    """The layer in 64 bits on given routes, and a tolerance.

    A dot product of n terms in fp32, its terms exact products of 16-bit numbers: sums round like a random walk, 8 sqrt(n) 2^-24 of
    sum |terms|. fp32 rows meet the weights to 2^-22 of the largest of their neighbours, 2^-21 with a margin (their tests draw rows of one
    size); h, kept in fp32, meets `down` to 2^-21 (f16: of its largest neighbour) or 2^-16 (bf16). With dg and du the errors of gate's and
    up's products, h = silu(g) u is off by 1.1 |u| dg + |silu(g)| du (|silu'| <= 1.1) and 12 roundings of its own (the exponential, the
    division); the output by sum w |down| dh, its own dot product, its weights (their softmax in fp32: 8 * 2^-24 and 2 * 2^-24 E), and its
    type's rounding."""
    n, D = x.shape
    out, tol = (torch.zeros((n, D), dtype=torch.float64, device=x.device) for _ in range(2))
    e24 = 2.0 ** -24
    ux = 2.0 ** -21 if dtype == torch.float32 else 0.0
    uh = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -21
    E = gate.shape[0]
    for t in range(n):
        big = x[t].abs().max()
        for e, we in zip(sel[t].tolist(), w[t].tolist()):
            if e < 0:
                if math.isnan(we):
                    out[t] = math.nan
                continue
            F = gate.shape[1]
            g, u = gate[e] @ x[t], up[e] @ x[t]
            rd = 8 * math.sqrt(D) * e24
            dg = rd * (gate[e].abs() @ x[t].abs()) + ux * big * gate[e].abs().sum(-1)
            du = rd * (up[e].abs() @ x[t].abs()) + ux * big * up[e].abs().sum(-1)
            s = g * torch.sigmoid(g)
            h = s * u
            dh = 1.1 * u.abs() * dg + s.abs() * du + 1.1 * dg * du + 12 * e24 * h.abs()
            y = down[e] @ h
            dy = down[e].abs() @ dh + (8 * math.sqrt(F) * e24 + (10 + 2 * E) * e24) * (down[e].abs() @ h.abs())
            dy = dy + uh * (down[e].abs() @ h.abs() if dtype == torch.bfloat16 else h.abs().max() * down[e].abs().sum(-1))
            out[t] += we * y
            tol[t] += we * dy
    return out, tol + half_step(out, dtype) * (1 + 2.0 ** -10)


class Layer:
    def __init__(self, typ, E, F, D, n, k, seed=0, renorm=False, bias=False, xscale=1.0):
        self.type, self.dtype = TYPES[typ]
        self.wtype = torch.bfloat16 if typ == "bf16" else torch.float16
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=g)
        self.gate, self.up = ((rnd(E, F, D) * D ** -0.5).to(self.wtype) for _ in range(2))
        self.down = (rnd(E, D, F) * F ** -0.5).to(self.wtype)
        self.x, self.logits = (rnd(n, D) * xscale).to(self.dtype), rnd(n, E) * 1.5
        self.bias = rnd(E) * 0.05 if bias else None
        self.E, self.F, self.D, self.n, self.k, self.renorm = E, F, D, n, k, renorm
        self.dev = [t.to(DEV) for t in (self.gate, self.up, self.down)]
        self.ex = z2h.Experts(gate=self.dev[0].data_ptr(), up=self.dev[1].data_ptr(), down=self.dev[2].data_ptr(),
                              type=TYPES["bf16" if typ == "bf16" else "f16"][0], n_expert=E, n_ff=F, n_embd=D)

    def put(self, ctx):
        """Buffers of a call; the workspace holds what no call left there."""
        d = dict(x=self.x.to(DEV), logits=self.logits.to(DEV), bias=None if self.bias is None else self.bias.to(DEV),
                 out=torch.full((self.n, self.D), 7.0, dtype=self.dtype, device=DEV), sel=torch.full((self.n, self.k), -7, dtype=torch.int32, device=DEV),
                 w=torch.full((self.n, self.k), -7.0, device=DEV))
        d["ws"] = torch.full((ctx.moe_rows_ws_bytes(self.ex, self.n, self.k),), 255, dtype=torch.uint8, device=DEV)
        return d

    def call(self, ctx, d, stream=None, xs=None, os=None, x=None, out=None):
        ctx.moe_rows(self.ex, self.n, self.k, self.renorm, d["logits"].data_ptr(), 0 if d["bias"] is None else d["bias"].data_ptr(), self.type,
                     x or d["x"].data_ptr(), xs or self.D, out or d["out"].data_ptr(), os or self.D, d["sel"].data_ptr(), d["w"].data_ptr(),
                     d["ws"].data_ptr(), d["ws"].numel(), stream=stream)

    def want(self):
        sel, w = route(self.logits.double().numpy(), None if self.bias is None else self.bias.double().numpy(), self.k, self.renorm)
        return sel, w, *layer(self.x.double(), self.gate.double(), self.up.double(), self.down.double(), sel, w, self.dtype)

    def check(self, ctx, what=""):
        d = self.put(ctx)
        self.call(ctx, d)
        torch.cuda.synchronize()
        sel, w, ref, tol = self.want()
        assert np.array_equal(d["sel"].cpu().numpy(), sel), f"{what}: experts"
        assert np.allclose(d["w"].cpu().numpy(), w, rtol=(10 + 2 * self.E) * 2.0 ** -24, atol=1e-37, equal_nan=True), f"{what}: weights"
        check(d["out"], ref, tol, what)
        return d


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 5, 16, 17, 33, 64, 128])
def test_rows(ctx, typ, n):
    print(f"moe {typ} rows {n}", flush=True)
    Layer(typ, 8, 96, 128, n, 2, seed=n, renorm=n % 2 == 0, bias=n % 3 == 0).check(ctx, f"{typ} {n}")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("E,F,D,k", [(1, 8, 8, 1), (2, 8, 2056, 2), (4, 40, 24, 3), (16, 136, 264, 1), (32, 200, 520, 4), (3, 2056, 72, 2),
                                     (60, 24, 56, 8), (257, 16, 32, 16), (1024, 8, 8, 5), (5, 520, 4104, 2), (2, 4120, 16, 1)])
def test_widths(ctx, typ, E, F, D, k):
    print(f"moe {typ} E {E} F {F} D {D} k {k}", flush=True)
    for n in (1, 7, 40):
        Layer(typ, E, F, D, n, k, seed=E + n, renorm=n == 7, bias=n == 40).check(ctx, f"{typ} {E} {F} {D} {k} rows {n}")


def test_the_benchmark_models_layer(ctx):
    for typ, n in (("f32", 1), ("f16", 16), ("bf16", 3)):
        Layer(typ, 32, 1536, 2048, n, 4, bias=True).check(ctx, typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_all_rows_take_one_expert(ctx, typ):
    """More rows of an expert than a tile of products has; the others' weights are not needed."""
    for n in (16, 17, 64, 100, 128):
        m = Layer(typ, 4, 72, 136, n, 1, seed=n)
        m.logits[:, 2] = 9.0
        m.check(ctx, f"{typ} {n}")


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("E,F,D,k,n", [(12, 1032, 264, 4, 100), (200, 264, 520, 8, 128), (300, 40, 72, 16, 90), (6, 2056, 2056, 3, 48), (64, 8, 40, 6, 64)])
def test_few_experts_take_most_rows(ctx, typ, E, F, D, k, n):
    """Experts with many rows beside ones with few, in parts of equal work that begin and end inside an expert."""
    print(f"moe {typ} E {E} F {F} D {D} k {k} rows {n}", flush=True)
    m = Layer(typ, E, F, D, n, k, seed=E)
    m.logits[:, 1::5] += 2.5 * torch.arange(1, (E + 3) // 5 + 1).remainder(4)
    m.logits[:, E - 1] += 6.0
    m.check(ctx, f"{typ} {E} {F} {D} {k} {n}")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 17, 40])
def test_wide_rows_and_many_hidden_dims(ctx, typ, n):
    """Rows of more than one pass of columns, more tiles of hidden dims per block than take a pass together (4101 tiles; from 17 rows on on
    256 blocks at most)."""
    print(f"moe {typ} rows {n}, wide", flush=True)
    E, F, D, k = 1, 32808, 2064, 1
    m = Layer(typ, E, 8, 8, n, k, seed=n, renorm=True)
    g = torch.Generator(device=DEV).manual_seed(n)
    gate, up = ((torch.randn((E, F, D), generator=g, device=DEV) * D ** -0.5).to(m.wtype) for _ in range(2))
    down = (torch.randn((E, D, F), generator=g, device=DEV) * F ** -0.5).to(m.wtype)
    x = torch.randn((n, D), generator=g, device=DEV).to(m.dtype)
    m.F, m.D, m.x = F, D, x
    m.ex = z2h.Experts(gate=gate.data_ptr(), up=up.data_ptr(), down=down.data_ptr(), type=m.ex.type, n_expert=E, n_ff=F, n_embd=D)
    d = m.put(ctx)
    m.call(ctx, d)
    torch.cuda.synchronize()
    ref, tol = layer(x.double(), gate.double(), up.double(), down.double(), np.zeros((n, 1), np.int64), np.ones((n, 1)), m.dtype)
    check(d["out"], ref.cpu(), tol.cpu(), typ)


def test_offsets_beyond_32_bits(ctx):
    """The last of 33 experts of 8192 x 8192 lies 2^31 elements behind the first, and so do the second row of x and that of the output."""
    print("moe offsets", flush=True)
    E, F, D, n, far = 33, 8192, 8192, 2, (1 << 31) + 8
    m = Layer("f16", E, 8, 8, n, 1, renorm=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    w = [torch.zeros((E, F, D), dtype=torch.float16, device=DEV) for _ in range(3)]
    for t in w:
        t[E - 1] = (torch.randn((F, D), generator=g, device=DEV) * D ** -0.5).half()
    x = torch.zeros(far + D, dtype=torch.float16, device=DEV)
    x[:D], x[far:] = (torch.randn(D, generator=g, device=DEV).half() for _ in range(2))
    out = torch.full((far + D,), 7.0, dtype=torch.float16, device=DEV)
    m.logits[:] = -1.0
    m.logits[:, E - 1] = 5.0
    m.F, m.D = F, D
    m.x = torch.stack([x[:D], x[far:]])
    m.ex = z2h.Experts(gate=w[0].data_ptr(), up=w[1].data_ptr(), down=w[2].data_ptr(), type=m.ex.type, n_expert=E, n_ff=F, n_embd=D)
    d = m.put(ctx)
    m.call(ctx, d, xs=far, os=far, x=x.data_ptr(), out=out.data_ptr())
    torch.cuda.synchronize()
    ref, tol = layer(m.x.double(), *(t[E - 1:].double() for t in w), np.zeros((n, 1), np.int64), np.ones((n, 1)), m.dtype)
    check(torch.stack([out[:D], out[far:]]), ref.cpu(), tol.cpu(), "far")
    assert bool((out[D:far] == 7).all())


def test_ties_go_to_the_lower_index(ctx):
    m = Layer("f32", 70, 16, 32, 6, 4)
    m.logits[0] = 0.0
    m.logits[1] = -3.0
    m.logits[2, :] = torch.arange(70) // 10
    m.logits[3, [5, 66, 64, 1]] = 8.0
    m.logits[4] = -0.0
    m.logits[4, ::2] = 0.0
    m.check(ctx)
    m = Layer("f32", 70, 16, 32, 2, 16, bias=True)
    m.logits[:] = 0.0
    m.bias[:] = 0.0
    m.bias[40] = 1.0
    m.check(ctx)


def test_masked_experts_and_rows_without_any(ctx):
    """Minus infinities: experts that are never taken, fewer than top_k left, none left; the lowest finite value is a value."""
    for typ in ("f32", "f16", "bf16"):
        for renorm in (False, True):
            m = Layer(typ, 16, 24, 40, 6, 4, renorm=renorm, bias=True)
            m.logits[0, :8] = -math.inf
            m.logits[1, 2:] = -math.inf
            m.logits[2] = -math.inf
            m.logits[3] = -math.inf
            m.logits[3, 11] = -3e38
            m.logits[4] = torch.finfo(torch.float32).min
            d = m.check(ctx, typ)
            assert bool((d["out"][2] == 0).all()) and d["sel"][2].tolist() == [-1] * 4


def test_no_numbers(ctx):
    """Rows whose logits are no numbers or infinite have no number; a row of x that holds one has results that are not finite; the other
    rows are as without them."""
    for typ in ("f32", "f16", "bf16"):
        m = Layer(typ, 8, 24, 40, 7, 2)
        sel, w, ref, tol = m.want()
        m.logits[1, 3] = math.nan
        m.logits[2, 0] = math.inf
        m.x[4, 7] = math.inf
        m.x[5, 39] = math.nan
        d = m.put(ctx)
        m.call(ctx, d)
        torch.cuda.synchronize()
        out = d["out"].cpu()
        assert bool(torch.isnan(out[1:3]).all()) and d["sel"][1:3].tolist() == [[-1, -1]] * 2 and bool(torch.isnan(d["w"][1:3]).all())
        assert not bool(torch.isfinite(out[4:6]).any())
        rows = [0, 3, 6]
        check(out[rows], ref[rows], tol[rows], typ)
    m = Layer("f32", 8, 24, 40, 3, 2, bias=True)
    m.bias[2] = math.nan
    d = m.put(ctx)
    m.call(ctx, d)
    torch.cuda.synchronize()
    assert bool(torch.isnan(d["out"]).all()) and bool((d["sel"] == -1).all())


def test_sizes_of_rows_and_products(ctx):
    """fp32 rows far from one, f16 rows whose products leave f16's range and come back."""
    for s in (1e-12, 1e-4, 1e4, 1e9):
        m = Layer("f32", 4, 40, 264, 5, 2, xscale=s)
        m.check(ctx, f"{s}")
    m = Layer("f16", 4, 40, 264, 5, 2, xscale=3000.0)        # h around 10^7
    m.down = (m.down.float() * 2.0 ** -12).half()
    m.dev[2].copy_(m.down)
    m.check(ctx, "large products")
    m = Layer("f16", 4, 40, 264, 5, 2, xscale=1e-3)
    m.check(ctx, "small products")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_strides_alignment_and_in_place(ctx, typ):
    m = Layer(typ, 8, 40, 136, 9, 2)
    sel, w, ref, tol = m.want()
    d = m.put(ctx)
    e = d["x"].element_size()
    for lead, stride in ((3, 301), (0, 139), (1, 136), (8, 144)):
        wide = torch.zeros(lead + 9 * stride, dtype=m.dtype, device=DEV)
        view = wide[lead:].view(9, stride)
        view[:, :136] = d["x"]
        out = torch.full((9, 143), 4.0, dtype=m.dtype, device=DEV)
        m.call(ctx, d, x=wide.data_ptr() + lead * e, xs=stride, out=out.data_ptr() + 5 * e, os=143)
        torch.cuda.synchronize()
        check(out[:, 5:141], ref, tol, f"{typ} {lead} {stride}")
        assert bool((out[:, :5] == 4).all()) and bool((out[:, 141:] == 4).all())
        m.call(ctx, d, x=wide.data_ptr() + lead * e, xs=stride, out=wide.data_ptr() + lead * e, os=stride)
        torch.cuda.synchronize()
        assert torch.equal(view[:, :136], out[:, 5:141])


def test_without_sel_and_weights(ctx):
    m = Layer("f16", 8, 40, 64, 3, 2)
    d = m.put(ctx)
    ctx.moe_rows(m.ex, 3, 2, False, d["logits"].data_ptr(), 0, m.type, d["x"].data_ptr(), 64, d["out"].data_ptr(), 64, 0, 0, d["ws"].data_ptr(),
                 d["ws"].numel())
    torch.cuda.synchronize()
    _, _, ref, tol = m.want()
    check(d["out"], ref, tol)


def test_streams_graphs_and_repeats(ctx):
    """Two layers at once on two streams, a captured layer replayed on new rows and logits, many repeats: bit for bit."""
    ms = [Layer("f16", 16, 264, 520, 12, 3, seed=1), Layer("f32", 8, 96, 136, 5, 2, seed=2, renorm=True)]
    ds = [m.put(ctx) for m in ms]
    for m, d in zip(ms, ds):
        m.call(ctx, d)
    torch.cuda.synchronize()
    want = [d["out"].clone() for d in ds]
    streams = [torch.cuda.Stream() for _ in ms]
    for d in ds:
        d["out"].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for st, m, d in zip(streams, ms, ds):
            m.call(ctx, d, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(w, d["out"]) for w, d in zip(want, ds))
    m, d = ms[0], ds[0]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        m.call(ctx, d, stream=side.cuda_stream)
    for seed in (3, 4, 5, 6):
        g = torch.Generator().manual_seed(seed)
        m.x, m.logits = torch.randn((12, 520), generator=g).half(), torch.randn((12, 16), generator=g) * seed
        d["x"].copy_(m.x), d["logits"].copy_(m.logits)
        graph.replay()
        torch.cuda.synchronize()
        sel, w, ref, tol = m.want()
        assert np.array_equal(d["sel"].cpu().numpy(), sel)
        check(d["out"], ref, tol, f"replay {seed}")
        torch.randn(1000, device=DEV).sum().item()


def test_refusals_and_nothing_to_do(ctx):
    m = Layer("f16", 8, 24, 40, 3, 2)
    d = m.put(ctx)
    p = {k: (0 if v is None else v.data_ptr()) for k, v in d.items()}
    good = dict(ex=m.ex, n=3, k=2, logits=p["logits"], type=z2h.F16, x=p["x"], xs=40, out=p["out"], os=40, ws=p["ws"], nb=d["ws"].numel())
    call = lambda a: ctx.moe_rows(a["ex"], a["n"], a["k"], 0, a["logits"], 0, a["type"], a["x"], a["xs"], a["out"], a["os"], 0, 0, a["ws"], a["nb"])
    for bad in (dict(n=-1), dict(n=129), dict(k=0), dict(k=9), dict(logits=0), dict(type=z2h.BF16), dict(type=8), dict(x=0), dict(out=0), dict(xs=39),
                dict(os=39), dict(x=p["x"] + 1), dict(out=p["x"], os=48), dict(ws=0), dict(ws=p["ws"] + 16), dict(nb=255)):
        with pytest.raises(z2h.Z2HError):
            call({**good, **bad})
    for field, value in (("gate", 0), ("up", m.ex.up + 8), ("down", 0), ("type", z2h.F32), ("type", z2h.BF16), ("n_expert", 0), ("n_expert", 1025),
                         ("n_ff", 20), ("n_ff", 0), ("n_embd", 36), ("n_embd", 65544)):
        ex = z2h.Experts.from_buffer_copy(m.ex)
        setattr(ex, field, value)
        with pytest.raises(z2h.Z2HError):
            call({**good, "ex": ex})
    call({**good, "n": 0, "x": 0, "out": 0, "logits": 0, "ws": 0, "nb": 0})
    torch.cuda.synchronize()
    assert bool((d["out"] == 7).all())
