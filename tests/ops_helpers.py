"""Inputs and 64-bit references of the operators on device tensors, shared by their GPU tests."""
import math

import numpy as np
import torch

from zonos2_amd import configs, z2h

DEV = "cuda:0"
TYPES = {"f32": (z2h.F32, torch.float32), "f16": (z2h.F16, torch.float16), "bf16": (z2h.BF16, torch.bfloat16)}


def context():
    """The operators need a context's device and error string, no weights."""
    cfg = configs.ModelConfig("operators", n_layer=1, n_embd=256, n_head=4, n_head_kv=2, head_dim=64, n_expert=0, top_k=0,
                              n_ff=256, bulk=configs.F16)
    return z2h.Context(cfg.hparams(), 1, 256)


def half_step(ref, dtype):
    """Half a step of the output type at the reference's size, its smallest subnormal step at the least."""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2) + f.tiny * f.eps


def ints(a):
    return torch.as_tensor(np.asarray(a, np.int32)).to(DEV)


def check(got, ref, tol, what=""):
    """Elementwise |got - ref| <= tol; NaN only where the reference has it."""
    got = got.double().cpu()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in {int((torch.isnan(got) != nan).sum())} other places"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    ok = ~(nan | inf)
    err, lim = (got - ref).abs()[ok], (tol if torch.is_tensor(tol) else torch.full_like(ref, tol))[ok]
    if err.numel():
        worst = (err / lim).max()
        assert bool((err <= lim).all()), f"{what}: error {float(err.max()):.3e}, {float(worst):.2f} of the tolerance"


# ---- rotary positions
def rotate(x, pos, base, dims, halves, factor=1.0, low=0.0, high=0.0, orig=0, mscale=1.0):
    """x [rows][heads][hd] float64, pos int64: rotated in 64 bits."""
    i = torch.arange(dims // 2, dtype=torch.float64)
    theta = torch.tensor(base, dtype=torch.float64) ** (-2.0 * i / max(dims, 1))
    keep = ((orig * theta / (2 * math.pi) - low) / (high - low)).clamp(0, 1) if orig else torch.zeros_like(theta)
    ang = pos.double()[:, None] * theta * (keep + (1 - keep) / factor)
    c, s = mscale * ang.cos()[:, None], mscale * ang.sin()[:, None]
    y = x.clone()
    a, b = (slice(0, dims // 2), slice(dims // 2, dims)) if halves else (slice(0, dims, 2), slice(1, dims, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def rotate_tol(x, ref, dims, halves, mscale, dtype):
    """Of the fp32 arithmetic, in units of mscale (|x| + |y|) 2^-24: cos and sin 2.5 (the reduced angle's rounding, at most
    pi/4, the polynomial's last sums), their product with mscale 1, the two products and their difference 2: 8 covers
    the sum with a margin. Then the rounding to the output's type. Dims that are not rotated are copied: half a step."""
    t = torch.zeros_like(x)
    a, b = (slice(0, dims // 2), slice(dims // 2, dims)) if halves else (slice(0, dims, 2), slice(1, dims, 2))
    t[..., a] = t[..., b] = 8 * 2.0 ** -24 * mscale * (x[..., a].abs() + x[..., b].abs())
    return t + half_step(ref, dtype) * (1 + 2.0 ** -10)


# ---- a paged cache
class Cache:
    """Pages of one layer on the device: random values where a sequence has rows, `fill` everywhere else. seq_rows: rows per
    sequence; shared: (first sequence, last, prefix rows) of groups whose whole prefix pages are the same ones and whose
    copies of the page that the prefix ends in hold the same rows."""

    def __init__(self, seq_rows, kvh, hd, page, dtype, seed, shared=(), room=0, fill=float("nan"), stride_pad=0):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        S = len(seq_rows)
        per = max(1, max((n + room + page - 1) // page for n in seq_rows))
        n_pages = S * per + 2
        ids = rng.permutation(n_pages)
        table = ids[:S * per].reshape(S, per).astype(np.int32).copy()
        for a, b, n in shared:
            table[a + 1:b, :n // page] = table[a, :n // page]
        self.kvh, self.hd, self.page, self.dtype = kvh, hd, page, dtype
        size = kvh * page * hd
        self.page_stride = size + stride_pad
        self.buf = [torch.full((n_pages, self.page_stride), fill, dtype=dtype) for _ in range(2)]
        view = [b[:, :size].view(n_pages, kvh, page, hd) for b in self.buf]
        for c in view:
            for s, n in enumerate(seq_rows):
                for i in range((n + page - 1) // page):
                    m = min(page, n - i * page)
                    c[table[s, i], :, :m] = torch.randn((kvh, m, hd), generator=g).to(dtype)
            for a, b, n in shared:
                if n % page:
                    for s in range(a + 1, b):
                        c[table[s, n // page], :, :n % page] = c[table[a, n // page], :, :n % page]
        self.table_host = table
        self.upload()

    def upload(self):
        self.dev = [b.to(DEV) for b in self.buf]
        self.table = ints(self.table_host)
        n_pages = self.buf[0].shape[0]
        self.pages = z2h.Pages(k=self.dev[0].data_ptr(), v=self.dev[1].data_ptr(), page_stride=self.page_stride,
                               type=z2h.BF16 if self.dtype == torch.bfloat16 else z2h.F16, n_pages=n_pages, page_rows=self.page,
                               n_head_kv=self.kvh, head_dim=self.hd, table=self.table.data_ptr(), n_seq=self.table_host.shape[0],
                               table_len=self.table_host.shape[1])

    def cell(self, which, seq, pos):
        """The [kvh][hd] view of one row in the host buffers."""
        b = self.buf[which][self.table_host[seq, pos // self.page]]
        return b[:self.kvh * self.page * self.hd].view(self.kvh, self.page, self.hd)[:, pos % self.page]

    def rows(self, seq, n):
        """k, v [n][kvh][hd] in 64 bits."""
        size = self.kvh * self.page * self.hd
        t = self.table_host[seq, :(n + self.page - 1) // self.page]
        return [b[t][:, :size].view(-1, self.kvh, self.page, self.hd).transpose(1, 2).reshape(-1, self.kvh, self.hd)[:n].double()
                for b in self.buf]


def attention(cache, q, row_start, kv_len, scale, dtype):
    """64-bit attention of q [rows][heads][hd] (float64, host), and a tolerance for a kernel of the given output type.

    Per value, with p the softmax and A = sum p |v|: a score's error is ds = scale (sum |q k|) (2^-24 sqrt(hd) * 8 + uq)
    (fp32 sums of exact products; uq: fp32 queries carried as two f16, 2^-21; f16 and bf16 queries are exact), which moves
    p by 2 ds relative at most (the weight and the sum). The exponent's argument (|s - max| up to 90) and exp round by
    2^-24 * (90 + 4). p is rounded to the cache's type before it meets the values, half a step up: 2^-11 f16, 2^-8
    bf16; for fp32 outputs it is carried as two f16, 2^-21. The sums over n keys, and over their partial results, round like
    a random walk: 8 sqrt(n) 2^-24 (eight standard deviations of a uniform rounding are 4.7 half steps). Then the output's
    own rounding."""
    R, nh, hd = q.shape
    grp = nh // cache.kvh
    ref, tol = torch.zeros_like(q), torch.zeros_like(q)
    up = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    uq = 2.0 ** -21 if dtype == torch.float32 else 0.0
    for s in range(len(kv_len)):
        r0, m, n = row_start[s], row_start[s + 1] - row_start[s], kv_len[s]
        if m == 0 or n == 0:
            continue
        k, v = cache.rows(s, n)
        for j in range(m):
            see = n - m + j + 1
            if see <= 0:
                continue
            kk, vv = (t[:see].repeat_interleave(grp, 1).transpose(0, 1) for t in (k, v))      # [nh][see][hd]
            x = q[r0 + j][:, None]
            sc = scale * (x * kk).sum(-1)
            p = torch.softmax(sc, -1)
            ref[r0 + j] = (p[..., None] * vv).sum(1)
            ds = abs(scale) * (x * kk).abs().sum(-1).amax(-1) * (8 * 2.0 ** -24 * math.sqrt(hd) + uq)
            rel = 2 * ds + 94 * 2.0 ** -24 + up + 8 * math.sqrt(see) * 2.0 ** -24
            tol[r0 + j] = rel[:, None] * (p[..., None] * vv.abs()).sum(1)
    return ref, tol + half_step(ref, dtype) * (1 + 2.0 ** -10)


class Attn:
    """One planned attention call."""

    def __init__(self, ctx, cache, heads, row_start, kv_len, groups, type_name, stream=0):
        self.ctx, self.cache, self.heads, self.stream = ctx, cache, heads, stream
        self.type, self.dtype = TYPES[type_name]
        self.R, self.G = int(row_start[-1]), len(groups)
        self.row_start, self.kv_len = ints(row_start), ints(kv_len)
        # groups: (first sequence, last, prefix rows), adjacent or with gaps; gaps become groups that share nothing
        start, prefix, at = [], [], 0
        for a, b, n in groups:
            if a > at:
                start.append(at), prefix.append(0)
            start.append(a), prefix.append(n)
            at = b
        self.G = len(start)
        self.group_start, self.prefix = ints(start + [at]), ints(prefix if prefix else [0])
        self.ws = torch.empty(ctx.paged_ws_bytes(cache.pages, heads, self.R, self.G), dtype=torch.uint8, device=DEV)

    def plan(self, stream=None):
        self.ctx.paged_plan(self.cache.pages, self.heads, self.R, self.row_start.data_ptr(), self.kv_len.data_ptr(), self.G,
                            self.group_start.data_ptr(), self.prefix.data_ptr(), self.ws.data_ptr(), self.ws.numel(),
                            stream=self.stream if stream is None else stream)

    def run(self, q, out, scale, stream=None):
        self.ctx.paged_attn(self.cache.pages, self.heads, self.R, self.G, scale, self.type, q.data_ptr(), q.stride(0),
                            out.data_ptr(), out.stride(0), self.ws.data_ptr(), self.ws.numel(),
                            stream=self.stream if stream is None else stream)


# ---- verification, in the order of its definition
def verify(draft, n_draft, target, temperature, draft_probs, u_accept, u_draw):
    """numpy arrays; returns (n_accept, codes)."""
    S, C, V = target.shape[0], target.shape[2], target.shape[3]
    accepted, codes = np.zeros(S, np.int32), np.zeros((S, C), np.int32)

    def probs(s, k, c):
        x = target[s, k, c].astype(np.float64)
        if temperature is None:
            return x
        if not temperature[s] > 0:
            return np.eye(1, V, int(x.argmax()))[0]
        e = np.exp((x - x.max()) / np.float64(temperature[s]))
        return e / e.sum()

    def pick(w, u):
        cum = np.cumsum(w)
        i = int(np.searchsorted(cum, u * cum[-1], side="right"))
        return i if i < V else int(np.nonzero(w > 0)[0][-1])

    for s in range(S):
        k, bad = 0, -1
        while k < n_draft[s] and bad < 0:
            for c in range(C):
                x = int(draft[s, k, c])
                inside = 0 <= x < V
                qx = 0.0 if not inside else 1.0 if draft_probs is None else float(draft_probs[s, k, c, x])
                if not (inside and u_accept[s, k, c] * qx < probs(s, k, c)[x]):
                    bad = c
                    break
            else:
                k += 1
        accepted[s] = k
        for c in range(C):
            w = probs(s, k, c)
            if c < bad:
                codes[s, c] = draft[s, k, c]
                continue
            if c == bad:
                x = int(draft[s, k, c])
                q = draft_probs[s, k, c].astype(np.float64) if draft_probs is not None else \
                    np.eye(1, V, x)[0] if 0 <= x < V else np.zeros(V)
                rest = np.maximum(w - q, 0.0)
                w = rest if rest.sum() > 0 else w
            codes[s, c] = pick(w, u_draw[s, c])
    return accepted, codes
