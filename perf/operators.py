"""The work of the operators around a paged key / value cache, as measured cases: rotary positions, appending rotated rows
to pages, attention of a batch whose requests share long prefixes (a voice prompt, a system prompt), and verifying
drafted frames.

`run` computes them either in their plain form (elementary torch operations, in 32 bits, angles and draws in 64) or,
with `own`, by the calls that a program makes of the Python binding of include/z2h.h (zonos2_amd.z2h).
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCALING = {                       # factor, low_turns, high_turns, orig_ctx, mscale
    "none": (1.0, 0.0, 0.0, 0, 1.0),
    "linear": (4.0, 0.0, 0.0, 0, 1.0),
    "parts": (8.0, 1.0, 32.0, 4096, 1.2079441541679836),
}


def listed():
    return [
        # the query rows of one decode step of 16 requests (this model family's heads)
        dict(name="rope16_f32", op="rope", rows=16, heads=16, hd=128, dims=128, halves=False, base=10000.0, scaling="none",
             type="f32", pos=4096),
        # a long document's rows, half layout, the first half of each head, stretched context
        dict(name="rope4099_bf16", op="rope", rows=4099, heads=32, hd=128, dims=64, halves=True, base=500000.0,
             scaling="parts", type="bf16", pos=1 << 20),
        # a decode step of 16 requests: one row each, fp32 projections into f16 pages, queries rotated on the way
        dict(name="append16_f32", op="append", seqs=16, rows=1, heads=16, kv_heads=4, hd=128, dims=128, halves=False,
             base=10000.0, scaling="none", type="f32", cache="f16", page=16, past=2048, pad=0),
        # prompt chunks of a mixed pass beside padded rows, bf16
        dict(name="append2088_bf16", op="append", seqs=8, rows=261, heads=32, kv_heads=8, hd=128, dims=96, halves=True,
             base=500000.0, scaling="linear", type="bf16", cache="bf16", page=64, past=3000, pad=24),
        # one request in the middle of its speech: nothing shared, latency counts
        dict(name="attn1_f32", op="attn", groups=1, seqs=1, rows=1, prefix=0, own_low=700, own_high=700, heads=16,
             kv_heads=4, hd=128, page=16, type="f32"),
        # a full server: 64 requests of one voice whose prompt is shared, lengths of their own far apart
        dict(name="attn64_f16", op="attn", groups=1, seqs=64, rows=1, prefix=2048, own_low=16, own_high=2048, heads=16,
             kv_heads=4, hd=128, page=16, type="f16"),
        # drafts of four frames to verify, 8 requests of each of three voices, odd lengths, smaller heads
        dict(name="attn24x5_bf16", op="attn", groups=3, seqs=8, rows=5, prefix=1111, own_low=5, own_high=333, heads=8,
             kv_heads=8, hd=64, page=32, type="bf16"),
        # prompt chunks behind a shared prefix: 4 requests, 333 rows each
        dict(name="attn4x333_f16", op="attn", groups=1, seqs=4, rows=333, prefix=1500, own_low=333, own_high=700, heads=16,
             kv_heads=4, hd=128, page=64, type="f16"),
        # many requests behind one very long prompt
        dict(name="attn256_bf16", op="attn", groups=1, seqs=256, rows=1, prefix=16384, own_low=32, own_high=512, heads=32,
             kv_heads=8, hd=128, page=64, type="bf16"),
        # 16 requests with four drafted frames each, logits of the model family's nine codebooks, drafts without
        # probabilities of their own (looked up, not drawn)
        dict(name="verify16_frames", op="verify", seqs=16, drafts=4, codebooks=9, vocab=1025, logits=True, draft_probs=False),
        # a text model's tokens, both models' probabilities in hand
        dict(name="verify64_probs", op="verify", seqs=64, drafts=5, codebooks=1, vocab=32000, logits=False, draft_probs=True),
        # few requests, a large vocabulary, logits
        dict(name="verify8_logits", op="verify", seqs=8, drafts=7, codebooks=1, vocab=131072, logits=True, draft_probs=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max((work(c) for c in listed()), key=lambda w: w["flops"])
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= top["flops"] and w["bytes"] <= top["bytes"]:
            return case


def _draw(rng):
    op = rng.choice(["rope", "append", "append", "attn", "attn", "attn", "attn", "verify", "verify"])
    if op == "verify":
        if rng.random() < 0.5:
            return dict(op=op, seqs=_log(rng, 1, 64), drafts=rng.randint(1, 6), codebooks=9, vocab=rng.choice([1025, 1026]),
                        logits=rng.random() < 0.7, draft_probs=rng.random() < 0.5)
        vocab = _log(rng, 300, 131072)
        return dict(op=op, seqs=_log(rng, 1, 64 if vocab < 16384 else 8), drafts=rng.randint(1, 7), codebooks=1,
                    vocab=vocab, logits=rng.random() < 0.5, draft_probs=rng.random() < 0.5)
    hd = rng.choice([32, 64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8])
    typ = rng.choice(["f32", "f16", "bf16"])
    if op == "attn":
        rows = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 300)])
        groups = rng.choice([1, 1, rng.randint(2, 5)])
        seqs = max(1, _log(rng, 1, 128) // groups // (1 if rows < 9 else 8))
        high = _log(rng, rows + 1, 3000)
        return dict(op=op, groups=groups, seqs=seqs, rows=rows, prefix=rng.choice([0, _log(rng, 17, 8192), _log(rng, 17, 8192)]),
                    own_low=max(rows, high // rng.randint(1, 16)), own_high=high, heads=heads, kv_heads=kv_heads, hd=hd,
                    page=rng.choice([16, 32, 64, 128]), type=typ)
    dims = rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)])
    case = dict(op=op, heads=heads, hd=hd, dims=dims, halves=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]),
                scaling=rng.choice(list(SCALING)), type=typ)
    if op == "rope":
        return dict(case, rows=_log(rng, 1, 4000), pos=_log(rng, 100, 1 << 20))
    return dict(case, seqs=_log(rng, 1, 64), rows=rng.choice([1, 1, _log(rng, 2, 64)]), kv_heads=kv_heads,
                cache="bf16" if typ == "bf16" else "f16", page=rng.choice([16, 32, 64, 128]), past=_log(rng, 16, 3000),
                pad=rng.choice([0, 0, rng.randint(1, 40)]))


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 12345)
    return g


def _randn(g, shape, typ="f32", scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(TYPES[typ])


def _ints(a):
    return torch.from_numpy(np.asarray(a, np.int32)).to(DEV)


def _append_rows(case, rng):
    """(sequence, position) of every row; padded rows have sequence -1."""
    seq, pos = [], []
    for s in range(case["seqs"]):
        p0 = int(rng.integers(0, case["past"] + 1))
        seq += [s] * case["rows"]
        pos += range(p0, p0 + case["rows"])
    return seq + [-1] * case["pad"], pos + [0] * case["pad"]


def _attn_lens(case, rng):
    """Rows of its own of every sequence, behind the shared prefix: log-uniform, the last `rows` of them this call's."""
    lo, hi = case["own_low"], case["own_high"]
    n = case["groups"] * case["seqs"]
    return np.maximum(case["rows"], np.exp(rng.uniform(math.log(lo), math.log(hi), n)).round().astype(int))


def _inputs(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    op = case["op"]
    if op == "rope":
        return dict(x=_randn(g, (case["rows"], case["heads"], case["hd"]), case["type"]),
                    pos=_ints(rng.integers(0, case["pos"], case["rows"])))
    if op == "append":
        seq, pos = _append_rows(case, rng)
        P, hd, kvh, n = case["page"], case["hd"], case["kv_heads"], len(seq)
        per = (case["past"] + case["rows"] + P - 1) // P
        n_pages = per * case["seqs"] + 3
        # one fused projection's rows, as the model's matmul leaves them: queries, keys, values
        fused = _randn(g, (n, (case["heads"] + 2 * kvh) * hd), case["type"])
        table = rng.permutation(n_pages)[:per * case["seqs"]].reshape(-1, per)
        k, v = (_randn(g, (n_pages, kvh, P, hd), case["cache"]) for _ in range(2))
        return dict(fused=fused, seq=_ints(seq), pos=_ints(pos), table=_ints(table), k_pages=k, v_pages=v,
                    q_out=torch.zeros((n, case["heads"], hd), device=DEV, dtype=TYPES[case["type"]]))
    if op == "attn":
        P, hd, kvh = case["page"], case["hd"], case["kv_heads"]
        S, pre = case["groups"] * case["seqs"], case["prefix"]
        lens = pre + _attn_lens(case, rng)
        shared = pre // P                    # whole pages of the prefix; the page that it ends in is each one's own copy
        per = int((lens.max() + P - 1) // P)
        used = [int((n + P - 1) // P) for n in lens]
        n_pages = case["groups"] * shared + sum(u - shared for u in used) + 1
        ids = iter(rng.permutation(n_pages).tolist())
        table = np.full((S, per), 0, np.int32)
        heads_ = [[next(ids) for _ in range(shared)] for _ in range(case["groups"])]
        for s in range(S):
            table[s, :shared] = heads_[s // case["seqs"]]
            table[s, shared:used[s]] = [next(ids) for _ in range(used[s] - shared)]
        cache = "bf16" if case["type"] == "bf16" else "f16"
        k, v = (_randn(g, (n_pages, kvh, P, hd), cache) for _ in range(2))
        if pre % P:
            # the copies of the page that the prefix ends in hold the same rows of it
            for s in range(S):
                first = table[s - s % case["seqs"], shared]
                for c in (k, v):
                    c[table[s, shared], :, :pre % P] = c[first, :, :pre % P]
        q = _randn(g, (S * case["rows"], case["heads"], hd), case["type"], 1.5)
        return dict(q=q, k_pages=k, v_pages=v, table=_ints(table), lens=lens, kv_len=_ints(lens), row_start=_ints(np.arange(S + 1) * case["rows"]),
                    group_start=_ints(np.arange(case["groups"] + 1) * case["seqs"]), prefix_len=_ints([pre] * case["groups"]))
    S, K, C, V = case["seqs"], case["drafts"], case["codebooks"], case["vocab"]
    # the target's logits are peaked; the draft's are the target's with an error, so that most drafts hold
    logits = _randn(g, (S, K + 1, C, V), scale=2.5)
    noisy = torch.softmax(logits[:, :K] + _randn(g, (S, K, C, V), scale=0.3 if C == 1 else 0.05), -1)
    if case["draft_probs"]:
        draft = torch.multinomial(noisy.reshape(-1, V), 1, generator=g).reshape(S, K, C)
    else:
        draft = noisy.argmax(-1)
        logits[:, :K].scatter_add_(-1, draft[..., None], torch.full((S, K, C, 1), 9.0 if V < 5000 else 13.0, device=DEV))
    st = dict(draft=draft.int(), n_draft=_ints(rng.integers(max(0, K - 2), K + 1, S)),
              u_accept=torch.rand((S, K, C), generator=g, device=DEV, dtype=torch.float64),
              u_draw=torch.rand((S, C), generator=g, device=DEV, dtype=torch.float64))
    st["temperature"] = torch.rand((S,), generator=g, device=DEV) * 0.4 + 0.7 if case["logits"] else None
    st["target"] = logits if case["logits"] else torch.softmax(logits, -1)
    st["draft_probs"] = noisy if case["draft_probs"] else None
    return st


# ---------------------------------------------------------------- the framework's calls
_ctx = []


def _binding():
    pkg = str(Path("zonos2.cpp_amd").resolve())
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from zonos2_amd import z2h
    return z2h


def _context():
    """A program's context: the operators take its device and leave their errors with it."""
    if not _ctx:
        from zonos2_amd import configs
        cfg = configs.ModelConfig("operators", n_layer=1, n_embd=256, n_head=4, n_head_kv=2, head_dim=64, n_expert=0, top_k=0,
                                  n_ff=256, bulk=configs.F16)
        _ctx.append(_binding().Context(cfg.hparams(), 1, 256))
    return _ctx[0]


def _handles(case, st):
    """What a program sets up once: the description of its pages and of the rotation, workspaces, output buffers, and
    for a step's attention the plan that every layer of the step uses."""
    z, op = _binding(), case["op"]
    ctx = _context()
    types = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16}
    stream = torch.cuda.current_stream().cuda_stream
    st["ctx"], st["type"] = ctx, types[case.get("type", "f32")]
    if op in ("rope", "append"):
        f, lo, hi, orig, ms = SCALING[case["scaling"]]
        st["rope"] = z.Rope(base=case["base"], n_dims=case["dims"], halves=int(case["halves"]), factor=f, low_turns=lo,
                            high_turns=hi, orig_ctx=orig, mscale=ms)
    if op == "rope":
        st["out"] = torch.empty_like(st["x"])
    if op in ("append", "attn"):
        k, t = st["k_pages"], st["table"]
        cache = types["bf16" if k.dtype == torch.bfloat16 else "f16"]
        st["pages"] = z.Pages(k=k.data_ptr(), v=st["v_pages"].data_ptr(), page_stride=k.stride(0), type=cache, n_pages=k.shape[0],
                              page_rows=k.shape[2], n_head_kv=k.shape[1], head_dim=k.shape[3], table=t.data_ptr(),
                              n_seq=t.shape[0], table_len=t.shape[1])
    if op == "attn":
        n, nh, G = st["q"].shape[0], case["heads"], case["groups"]
        st["out"] = torch.empty_like(st["q"])
        st["ws"] = torch.empty(ctx.paged_ws_bytes(st["pages"], nh, n, G), dtype=torch.uint8, device=DEV)
        ctx.paged_plan(st["pages"], nh, n, st["row_start"].data_ptr(), st["kv_len"].data_ptr(), G, st["group_start"].data_ptr(),
                       st["prefix_len"].data_ptr(), st["ws"].data_ptr(), st["ws"].numel(), stream=stream)
    if op == "verify":
        S, C = case["seqs"], case["codebooks"]
        st["n_accept"] = torch.empty((S,), dtype=torch.int32, device=DEV)
        st["codes"] = torch.empty((S, C), dtype=torch.int32, device=DEV)
        st["ws"] = torch.empty(ctx.verify_ws_bytes(S, case["drafts"], C, case["vocab"]), dtype=torch.uint8, device=DEV)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    return _handles(case, st) if own else st


def _own(st):
    case, ctx = st["case"], st["ctx"]
    op = case["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "rope":
        x, out, w = st["x"], st["out"], case["heads"] * case["hd"]
        ctx.rope_rows(st["rope"], case["rows"], case["heads"], case["hd"], st["type"], x.data_ptr(), w, out.data_ptr(), w,
                      st["pos"].data_ptr(), stream=stream)
        return out
    if op == "append":
        f, hd, nh, kvh = st["fused"], case["hd"], case["heads"], case["kv_heads"]
        R, p, e = f.shape[1], f.data_ptr(), f.element_size()
        ctx.paged_append(st["pages"], st["rope"], f.shape[0], st["seq"].data_ptr(), st["pos"].data_ptr(), st["type"],
                         p + nh * hd * e, R, p + (nh + kvh) * hd * e, R, nh, p, R, st["q_out"].data_ptr(), nh * hd, stream=stream)
        return st["q_out"], st["k_pages"], st["v_pages"]
    if op == "attn":
        q, w = st["q"], case["heads"] * case["hd"]
        ctx.paged_attn(st["pages"], case["heads"], q.shape[0], case["groups"], case["hd"] ** -0.5, st["type"], q.data_ptr(), w,
                       st["out"].data_ptr(), w, st["ws"].data_ptr(), st["ws"].numel(), stream=stream)
        return st["out"]
    ptr = lambda t: 0 if t is None else t.data_ptr()
    ctx.verify(case["seqs"], case["drafts"], case["codebooks"], case["vocab"], st["draft"].data_ptr(), st["n_draft"].data_ptr(),
               st["target"].data_ptr(), ptr(st["temperature"]), ptr(st["draft_probs"]), st["u_accept"].data_ptr(),
               st["u_draw"].data_ptr(), st["n_accept"].data_ptr(), st["codes"].data_ptr(), st["ws"].data_ptr(), st["ws"].numel(),
               stream=stream)
    return st["n_accept"], st["codes"]


# ---------------------------------------------------------------- the plain forms
def _rotate(case, x, pos):
    """x [rows][heads][hd] in 32 bits, rotated by its positions' angles."""
    n = case["dims"]
    factor, lo, hi, orig, ms = SCALING[case["scaling"]]
    theta = torch.pow(torch.tensor(case["base"], dtype=torch.float64, device=DEV),
                      -2.0 * torch.arange(n // 2, dtype=torch.float64, device=DEV) / n)
    keep = torch.clamp((orig * theta / (2 * math.pi) - lo) / (hi - lo), 0, 1) if orig else torch.zeros_like(theta)
    a = pos.double()[:, None] * (theta * (keep + (1 - keep) / factor))
    c, s = (ms * torch.cos(a)).float()[:, None], (ms * torch.sin(a)).float()[:, None]
    x = x.float()
    y = x.clone()
    first, second = (slice(0, n // 2), slice(n // 2, n)) if case["halves"] else (slice(0, n, 2), slice(1, n, 2))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    return y


def _plain_attn(st):
    case = st["case"]
    kvh, hd, m = case["kv_heads"], case["hd"], case["rows"]
    grp = case["heads"] // kvh
    out = torch.empty_like(st["q"])
    for s, n in enumerate(st["lens"].tolist()):
        t = st["table"][s, :(n + case["page"] - 1) // case["page"]].long()
        k, v = (c[t].transpose(0, 1).reshape(kvh, -1, hd)[:, :n].float() for c in (st["k_pages"], st["v_pages"]))
        q = st["q"][s * m:(s + 1) * m].float().reshape(m, kvh, grp, hd).transpose(0, 1).reshape(kvh, m * grp, hd)
        sc = torch.bmm(q, k.transpose(1, 2).contiguous()) * hd ** -0.5
        if m > 1:
            seen = n - m + torch.arange(m, device=DEV).repeat_interleave(grp)
            sc = torch.where(torch.arange(n, device=DEV) <= seen[:, None], sc, torch.full_like(sc, -math.inf))
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.bmm(p, v.contiguous()) / p.sum(-1, keepdim=True)
        out[s * m:(s + 1) * m] = o.reshape(kvh, m, grp, hd).transpose(0, 1).reshape(m, -1, hd).to(out.dtype)
    return out


def _plain_verify(st):
    case = st["case"]
    S, K, C, V = case["seqs"], case["drafts"], case["codebooks"], case["vocab"]
    p = st["target"].double()
    if st["temperature"] is not None:
        p = p / st["temperature"].double()[:, None, None, None]
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    x = st["draft"].long()
    px = p[:, :K].gather(-1, x[..., None])[..., 0]
    q = st["draft_probs"]
    qx = torch.ones_like(px) if q is None else q.gather(-1, x[..., None])[..., 0].double()
    judged = torch.arange(K, device=DEV)[:, None] < st["n_draft"].long()[:, None, None]
    fail = ((st["u_accept"] * qx >= px) & judged).reshape(S, K * C)
    first = torch.where(fail.any(-1), fail.int().argmax(-1), st["n_draft"].long() * C)      # the code that fails, in order
    frame, code = first // C, first % C
    at = torch.arange(S, device=DEV)
    w = p[at, frame]                                                                        # [S][C][V]
    rejected = frame < st["n_draft"]
    fr = frame.clamp(max=K - 1)
    qr = torch.zeros((S, V), dtype=torch.float64, device=DEV).scatter_(1, x[at, fr, code][:, None], 1.0) if q is None \
        else q[at, fr, code].double()
    rest = (w[at, code] - qr).clamp(min=0)
    use = rejected & (rest.sum(-1) > 0)
    w[at, code] = torch.where(use[:, None], rest, w[at, code])
    cum = w.cumsum(-1)
    past = cum > st["u_draw"][..., None] * cum[..., -1:]
    last = V - 1 - (w.flip(-1) > 0).int().argmax(-1)
    drawn = torch.where(past.any(-1), past.int().argmax(-1), last)
    kept = torch.arange(C, device=DEV)[None] < torch.where(rejected, code, 0)[:, None]
    return frame.int(), torch.where(kept, x[at, fr], drawn).int()


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    op = case["op"]
    if op == "rope":
        return _rotate(case, state["x"], state["pos"]).to(state["x"].dtype)
    if op == "append":
        nh, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
        n = case["seqs"] * case["rows"]                          # the padded rows are the last
        f = state["fused"][:n]
        pos = state["pos"][:n].long()
        page = state["table"][state["seq"][:n].long(), pos // case["page"]].long()
        r = pos % case["page"]
        k = f[:, nh * hd:(nh + kvh) * hd].reshape(n, kvh, hd)
        state["k_pages"][page, :, r] = _rotate(case, k, pos).to(state["k_pages"].dtype)
        state["v_pages"][page, :, r] = f[:, (nh + kvh) * hd:].reshape(n, kvh, hd).to(state["v_pages"].dtype)
        state["q_out"][:n] = _rotate(case, f[:, :nh * hd].reshape(n, nh, hd), pos).to(state["q_out"].dtype)
        return state["q_out"], state["k_pages"], state["v_pages"]
    if op == "attn":
        return _plain_attn(state)
    return _plain_verify(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 2 * n * SIZE[case["type"]] + 4 * case["rows"], "flops": 3 * n}
    if op == "append":
        n, hd = case["seqs"] * case["rows"], case["hd"]
        q, k = n * case["heads"] * hd, n * case["kv_heads"] * hd
        e = SIZE[case["type"]]
        return {"bytes": 2 * q * e + 2 * k * (e + SIZE[case["cache"]]) + 12 * n, "flops": 3 * (q + k)}
    if op == "attn":
        lo, hi = case["own_low"], case["own_high"]
        S, m, pre = case["groups"] * case["seqs"], case["rows"], case["prefix"]
        mean = lo if lo == hi else (hi - lo) / math.log(hi / lo)                            # of log-uniform lengths
        mean = max(mean, m)
        keys = case["groups"] * pre + S * mean
        seen = S * m * (pre + mean - (m - 1) / 2)
        q = S * m * case["heads"] * case["hd"]
        return {"bytes": int(keys * 2 * case["kv_heads"] * case["hd"] * 2 + 2 * q * SIZE[case["type"]]),
                "flops": int(4 * seen * case["heads"] * case["hd"])}
    S, K, C, V = case["seqs"], case["drafts"], case["codebooks"], case["vocab"]
    # logits: every row's sum; probabilities: the rows that are drawn from, and the rest of one row of the draft's
    rows = S * ((K + 1) * C if case["logits"] else C) + (S if case["draft_probs"] else 0)
    return {"bytes": 4 * rows * V + S * (K * C * 12 + C * 12), "flops": (10 if case["logits"] else 3) * rows * V}


# ---------------------------------------------------------------- the same in 64 bits
def _exact_rotate(case, x, pos):
    """Complex multiplication by mscale e^(i pos theta')."""
    n = case["dims"]
    factor, lo, hi, orig, ms = SCALING[case["scaling"]]
    i = np.arange(n // 2, dtype=np.float64)
    theta = np.exp(-2.0 * i / n * math.log(case["base"]))
    if orig:
        turns = orig * theta / (2 * math.pi)
        keep = np.minimum(1.0, np.maximum(0.0, (turns - lo) / (hi - lo)))
        theta = keep * theta + (1.0 - keep) * theta / factor
    else:
        theta = theta / factor
    z = torch.from_numpy(ms * np.exp(1j * pos.astype(np.float64)[:, None] * theta)).to(DEV)[:, None]
    x = x.double()
    r = x[..., :n]
    pair = r.reshape(*r.shape[:-1], 2, n // 2).transpose(-1, -2) if case["halves"] else r.reshape(*r.shape[:-1], n // 2, 2)
    t = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    t = (t.transpose(-1, -2) if case["halves"] else t).reshape(r.shape)
    return torch.cat([t, x[..., n:]], -1)


def exact(case, seed):
    st = _inputs(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_rotate(case, st["x"], st["pos"].cpu().numpy())
    if op == "append":
        nh, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
        seq, pos = st["seq"].cpu().numpy(), st["pos"].cpu().numpy()
        table = st["table"].cpu().numpy()
        q, k, v = st["fused"].double().split([nh * hd, kvh * hd, kvh * hd], 1)
        q = _exact_rotate(case, q.reshape(-1, nh, hd), pos)
        k = _exact_rotate(case, k.reshape(-1, kvh, hd), pos)
        q[torch.from_numpy(seq).to(DEV) < 0] = 0.0
        K, V = st["k_pages"].double(), st["v_pages"].double()
        rows = np.nonzero(seq >= 0)[0]
        page = torch.from_numpy(table[seq[rows], pos[rows] // case["page"]].astype(np.int64)).to(DEV)
        r = torch.from_numpy(pos[rows] % case["page"]).long().to(DEV)
        i = torch.from_numpy(rows).to(DEV)
        K[page, :, r] = k[i]
        V[page, :, r] = v.reshape(-1, kvh, hd)[i]
        return q, K, V
    if op == "attn":
        m, kvh, hd = case["rows"], case["kv_heads"], case["hd"]
        grp = case["heads"] // kvh
        out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
        for s, n in enumerate(st["lens"].tolist()):
            pages = st["table"][s, :-(-n // case["page"])].tolist()
            K, V = (torch.cat([c[p] for p in pages], 1)[:, :n].double() for c in (st["k_pages"], st["v_pages"]))
            hidden = torch.ones((m, n), dtype=torch.bool, device=DEV).triu(n - m + 1)
            for h in range(case["heads"]):
                sc = (st["q"][s * m:(s + 1) * m, h].double() @ K[h // grp].T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                out[s * m:(s + 1) * m, h] = torch.softmax(sc, -1) @ V[h // grp]
        return out
    # integers: every sequence by itself, in the order of the definition
    S, C = case["seqs"], case["codebooks"]
    host = {n: (None if t is None else t.cpu().numpy()) for n, t in st.items()}
    accepted, codes = np.zeros(S, np.int32), np.zeros((S, C), np.int32)

    def probs(s, k, c):
        row = host["target"][s, k, c].astype(np.float64)
        if host["temperature"] is None:
            return row
        e = np.exp((row - row.max()) / float(host["temperature"][s]))
        return e / e.sum()

    def pick(w, u):
        cum = np.cumsum(w)
        i = int(np.searchsorted(cum, u * cum[-1], side="right"))
        return i if i < len(w) else int(np.nonzero(w > 0)[0][-1])

    for s in range(S):
        k, bad = 0, -1
        while k < host["n_draft"][s] and bad < 0:
            for c in range(C):
                x = host["draft"][s, k, c]
                qx = 1.0 if host["draft_probs"] is None else float(host["draft_probs"][s, k, c, x])
                if host["u_accept"][s, k, c] * qx >= probs(s, k, c)[x]:
                    bad = c
                    break
            else:
                k += 1
        accepted[s] = k
        for c in range(C):
            w = probs(s, k, c)
            if c < bad:
                codes[s, c] = host["draft"][s, k, c]
                continue
            if c == bad:
                q = np.eye(1, case["vocab"], int(host["draft"][s, k, c]))[0] if host["draft_probs"] is None else host["draft_probs"][s, k, c]
                rest = np.maximum(w - q, 0.0)
                w = rest if rest.sum() > 0 else w
            codes[s, c] = pick(w, host["u_draw"][s, c])
    return torch.from_numpy(accepted).to(DEV), torch.from_numpy(codes).to(DEV)
