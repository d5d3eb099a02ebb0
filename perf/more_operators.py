"""The work of a prompt's attention, of a mixture-of-experts layer for a few rows, and of a paged cache's upkeep, as measured
cases: attention of whole prompts packed one behind the other, routing with the experts' products, sequences that take over
others' cache rows (with copies of the pages that both go on writing to), and moving a cache's pages together.

`run` computes them either in their plain form (elementary torch operations, in 32 bits, routing in 64) or, with `own`, by
the calls that a program makes of the Python binding of include/z2h.h (zonos2_amd.z2h).
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


def listed():
    return [
        # one short prompt in fp32 rows, as the model's projections leave them: latency counts
        dict(name="prompt37_f32", op="prompt", seqs=1, low=37, high=37, heads=16, kv_heads=4, hd=128, type="f32"),
        # the prompts of one mixed pass: eight of 256 rows
        dict(name="prompt8x256_f16", op="prompt", seqs=8, low=256, high=256, heads=16, kv_heads=4, hd=128, type="f16"),
        # a server's queue of prompts, lengths far apart, smaller heads
        dict(name="prompt24_bf16", op="prompt", seqs=24, low=16, high=2000, heads=32, kv_heads=8, hd=64, type="bf16"),
        # one long document
        dict(name="prompt8191_bf16", op="prompt", seqs=1, low=8191, high=8191, heads=32, kv_heads=8, hd=128, type="bf16"),
        # one request's frame through the benchmark model's experts, fp32 rows
        dict(name="moe1_f32", op="moe", rows=1, embd=2048, ff=1536, experts=32, top_k=4, renorm=False, bias=True, type="f32"),
        # a step of 16 requests
        dict(name="moe16_f16", op="moe", rows=16, embd=2048, ff=1536, experts=32, top_k=4, renorm=False, bias=True, type="f16"),
        # a frame and four drafts, 16 experts of which a row takes one
        dict(name="moe5_bf16", op="moe", rows=5, embd=2048, ff=4096, experts=16, top_k=1, renorm=False, bias=False, type="bf16"),
        # a full server, many small experts, weights made to sum to one
        dict(name="moe64_bf16", op="moe", rows=64, embd=2048, ff=1032, experts=64, top_k=6, renorm=True, bias=False, type="bf16"),
        # a voice prompt taken over by four new requests: small pages, latency counts
        dict(name="fork4_f16", op="fork", prompts=1, forks=4, rows=700, room=40, page=16, layers=24, kv_heads=4, hd=128, type="f16", spare=64),
        # 16 beams of each of four requests begin anew behind what their best has
        dict(name="fork64_bf16", op="fork", prompts=4, forks=16, rows=1999, room=64, page=64, layers=24, kv_heads=4, hd=128, type="bf16", spare=200),
        # a small cache after a few requests ended
        dict(name="compact300_f16", op="compact", seqs=12, rows=350, shared=100, page=16, gone=0.4, layers=4, kv_heads=4, hd=128, type="f16"),
        # a full server's cache: half of the requests ended
        dict(name="compact1500_f16", op="compact", seqs=48, rows=1800, shared=512, page=64, gone=0.5, layers=24, kv_heads=4, hd=128, type="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    every = [work(c) for c in listed()]
    flops, size = max(w["flops"] for w in every), max(w["bytes"] for w in every)
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= flops and w["bytes"] <= size and _scores(case) <= 2.2e9:
            return case


def _scores(case):
    return case["seqs"] * case["heads"] * case["high"] ** 2 if case["op"] == "prompt" else 0


def _draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "moe", "moe", "moe", "fork", "compact"])
    hd, kv_heads = rng.choice([32, 64, 128, 128]), rng.choice([1, 2, 4, 8])
    if op == "prompt":
        high = _log(rng, 1, 6000)
        return dict(op=op, seqs=rng.choice([1, 1, _log(rng, 2, 64)]), low=max(1, high // rng.choice([1, 2, 16, 100])), high=high,
                    heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads, hd=hd, type=rng.choice(["f32", "f16", "bf16"]))
    if op == "moe":
        experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
        return dict(op=op, rows=_log(rng, 1, 64), embd=8 * _log(rng, 32, 512), ff=8 * _log(rng, 16, 512 if experts < 33 else 128), experts=experts,
                    top_k=rng.choice([1, 2, 4, min(8, experts)]), renorm=rng.random() < 0.5, bias=rng.random() < 0.5,
                    type=rng.choice(["f32", "f16", "bf16"]))
    page = rng.choice([16, 32, 64, 128])
    rest = dict(page=page, layers=rng.choice([1, 4, 24, 28]), kv_heads=rng.choice([1, 2, 4]), hd=hd, type=rng.choice(["f16", "bf16"]))
    if op == "fork":
        return dict(op=op, prompts=rng.randint(1, 6), forks=_log(rng, 1, 24), rows=_log(rng, 10, 2000), room=rng.choice([0, 1, _log(rng, 2, 200)]),
                    spare=rng.randint(1, 300), **rest)
    rows = _log(rng, 40, 1800)
    return dict(op=op, seqs=rng.randint(2, 48), rows=rows, shared=rng.choice([0, rows // 3, rows // 2]), gone=rng.choice([0.1, 0.3, 0.5, 0.8]), **rest)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 54321)
    return g


def _randn(g, shape, typ="f32", scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(TYPES[typ])


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _cache(case, g, n_pages):
    """k and v of all layers, each [layers][n_pages][kv_heads][page][hd]."""
    shape = (case["layers"], n_pages, case["kv_heads"], case["page"], case["hd"])
    out = []
    for _ in range(2):
        t = torch.empty(shape, dtype=TYPES[case["type"]], device=DEV)
        t.normal_(generator=g)
        out.append(t)
    return out


def _prompt_inputs(case, g, rng):
    # the same lengths for every seed, in another order
    lo, hi, S = case["low"], case["high"], case["seqs"]
    lens = np.exp(np.random.default_rng(S).uniform(math.log(lo), math.log(hi), S)).round().astype(int)
    lens[0] = hi
    lens = rng.permutation(lens)
    start = np.concatenate([[0], np.cumsum(lens)])
    n, nh, kvh, hd = int(start[-1]), case["heads"], case["kv_heads"], case["hd"]
    # one fused projection's rows: queries, keys, values, and behind them the heads' gates
    fused = _randn(g, (n, (nh + 2 * kvh) * hd + (nh + 7) // 8 * 8), case["type"])
    fused[:, :nh * hd] *= 1.5
    return dict(fused=fused, start=_ints(start), lens=lens)


def _moe_inputs(case, g, rng):
    E, F, D = case["experts"], case["ff"], case["embd"]
    typ = "bf16" if case["type"] == "bf16" else "f16"
    gate, up = (_randn(g, (E, F, D), typ, D ** -0.5) for _ in range(2))
    down = _randn(g, (E, D, F), typ, F ** -0.5)
    return dict(gate=gate, up=up, down=down, x=_randn(g, (case["rows"], D), case["type"]),
                logits=_randn(g, (case["rows"], E), "f32", 1.5), bias=_randn(g, (E,), "f32", 0.02) if case["bias"] else None)


def _pages_of(rows, page):
    return (rows + page - 1) // page


def _fork_inputs(case, g, rng):
    """Prompts in sequences of their own; behind them the sequences that take them over, which still hold a few pages of what
    they had."""
    P, S = case["page"], case["prompts"] * (1 + case["forks"])
    rows = rng.integers(max(1, case["rows"] - P), case["rows"] + 1, case["prompts"])
    total = _pages_of(case["rows"] + case["room"], P)
    old = rng.integers(0, 3, S - case["prompts"]).clip(max=total)
    n_pages = case["prompts"] * total + len(old) * (1 + _pages_of(case["room"], P) + 2) + case["spare"]
    ids = iter(rng.permutation(n_pages).tolist())
    table = np.full((S, total), -1, np.int32)
    refs = np.zeros(n_pages, np.int32)
    for s in range(S):
        n = _pages_of(int(rows[s]), P) if s < case["prompts"] else int(old[s - case["prompts"]])
        table[s, :n] = [next(ids) for _ in range(n)]
        refs[table[s, :n]] += 1
    dst = np.arange(case["prompts"], S)
    src = (dst - case["prompts"]) // case["forks"]
    k, v = _cache(case, g, n_pages)
    return dict(k=k, v=v, table=_ints(table), refs=_ints(refs), src=_ints(src), dst=_ints(dst), rows=_ints(rows[src]),
                room=_ints(rows[src] + case["room"]))


def _compact_inputs(case, g, rng):
    """Sequences that came one after the other and grew a page at a time, a prefix shared by all; some of them ended."""
    P, S = case["page"], case["seqs"]
    lens = rng.permutation(np.linspace(max(case["rows"] // 2, case["shared"] + 1), case["rows"], S).round().astype(int))
    shared, total = case["shared"] // P, _pages_of(case["rows"], P)
    need = [int(_pages_of(int(n), P)) for n in lens]
    n_pages = shared + sum(n - shared for n in need) + 8
    table = np.full((S, total), -1, np.int32)
    table[:, :shared] = np.arange(shared)
    at = shared
    for j in range(shared, total):
        for s in range(S):
            if j < need[s]:
                table[s, j] = at
                at += 1
    gone = rng.permutation(S)[:min(S - 1, max(1, int(round(S * case["gone"]))))]
    table[gone] = -1
    refs = np.bincount(table[table >= 0], minlength=n_pages)
    k, v = _cache(case, g, n_pages)
    return dict(k=k, v=v, table=_ints(table), refs=_ints(refs))


def _inputs(case, seed):
    make = {"prompt": _prompt_inputs, "moe": _moe_inputs, "fork": _fork_inputs, "compact": _compact_inputs}[case["op"]]
    return make(case, _gen(seed), np.random.default_rng(seed))


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case, kept={})


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
        z = _binding()
        from zonos2_amd import configs
        cfg = configs.ModelConfig("operators", n_layer=1, n_embd=256, n_head=4, n_head_kv=2, head_dim=64, n_expert=0, top_k=0,
                                  n_ff=256, bulk=configs.F16)
        _ctx.append(z.Context(cfg.hparams(), 1, 256))
    return _ctx[0]


def _keep(st):
    """What a program sets up once and keeps beside its data: descriptions, output buffers, workspaces."""
    z, ctx, case, kept = _binding(), _context(), st["case"], st["kept"]
    types = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16}
    kept["type"] = types[case["type"]]
    if case["op"] == "prompt":
        kept["out"] = torch.empty((st["fused"].shape[0], case["heads"] * case["hd"]), dtype=st["fused"].dtype, device=DEV)
    elif case["op"] == "moe":
        n, k = case["rows"], case["top_k"]
        kept["experts"] = z.Experts(gate=st["gate"].data_ptr(), up=st["up"].data_ptr(), down=st["down"].data_ptr(),
                                    type=types["bf16" if case["type"] == "bf16" else "f16"], n_expert=case["experts"], n_ff=case["ff"],
                                    n_embd=case["embd"])
        kept["out"] = torch.empty_like(st["x"])
        kept["sel"] = torch.empty((n, k), dtype=torch.int32, device=DEV)
        kept["weights"] = torch.empty((n, k), dtype=torch.float32, device=DEV)
        kept["ws"] = torch.empty(ctx.moe_rows_ws_bytes(kept["experts"], n, k), dtype=torch.uint8, device=DEV)
    else:
        k, t = st["k"], st["table"]
        kept["pages"] = z.Pages(k=k.data_ptr(), v=st["v"].data_ptr(), page_stride=k.stride(1), type=kept["type"], n_pages=k.shape[1],
                                page_rows=k.shape[3], n_head_kv=k.shape[2], head_dim=k.shape[4], table=t.data_ptr(), n_seq=t.shape[0],
                                table_len=t.shape[1])
        n = st["src"].numel() if case["op"] == "fork" else 0
        kept["ws"] = torch.empty(ctx.pages_ws_bytes(kept["pages"], n), dtype=torch.uint8, device=DEV)
        if n:
            kept["held"] = torch.empty_like(st["src"])
        else:
            kept["table"], kept["refs"] = torch.empty_like(t), torch.empty_like(st["refs"])
            kept["n_used"] = torch.empty(1, dtype=torch.int32, device=DEV)
    return kept


def _own(st):
    case, kept, ctx = st["case"], st["kept"] or _keep(st), _context()
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "prompt":
        f, out, nh, kvh, hd = st["fused"], kept["out"], case["heads"], case["kv_heads"], case["hd"]
        R, p, e = f.shape[1], f.data_ptr(), f.element_size()
        ctx.prompt_attn(case["seqs"], st["start"].data_ptr(), f.shape[0], nh, kvh, hd, hd ** -0.5, kept["type"], p, R, p + nh * hd * e, R,
                        p + (nh + kvh) * hd * e, R, out.data_ptr(), nh * hd, stream=stream)
        return out
    ws, n_ws = kept["ws"].data_ptr(), kept["ws"].numel()
    if case["op"] == "moe":
        x, out, D = st["x"], kept["out"], case["embd"]
        ctx.moe_rows(kept["experts"], case["rows"], case["top_k"], case["renorm"], st["logits"].data_ptr(),
                     st["bias"].data_ptr() if case["bias"] else 0, kept["type"], x.data_ptr(), D, out.data_ptr(), D, kept["sel"].data_ptr(),
                     kept["weights"].data_ptr(), ws, n_ws, stream=stream)
        return out, kept["sel"], kept["weights"]
    layers, stride = case["layers"], st["k"].stride(0)
    if case["op"] == "fork":
        ctx.pages_fork(kept["pages"], layers, stride, st["refs"].data_ptr(), st["src"].numel(), st["src"].data_ptr(), st["dst"].data_ptr(),
                       st["rows"].data_ptr(), st["room"].data_ptr(), kept["held"].data_ptr(), ws, n_ws, stream=stream)
        return st["table"], st["refs"], kept["held"], st["k"], st["v"]
    ctx.pages_compact(kept["pages"], layers, stride, st["refs"].data_ptr(), kept["table"].data_ptr(), kept["refs"].data_ptr(),
                      kept["n_used"].data_ptr(), ws, n_ws, stream=stream)
    return kept["table"], kept["refs"], kept["n_used"], st["k"], st["v"]


# ---------------------------------------------------------------- the plain forms
def _plain_prompt(st):
    """All prompts side by side, padded to the longest."""
    case, f = st["case"], st["fused"]
    S, nh, kvh, hd = case["seqs"], case["heads"], case["kv_heads"], case["hd"]
    grp, L = nh // kvh, int(st["lens"].max())
    start = st["start"].long()
    at = torch.arange(L, device=DEV)
    live = at < (start[1:] - start[:-1])[:, None]                               # [S][L]
    rows = f[torch.where(live, start[:-1, None] + at, 0)].float()               # [S][L][...]
    q, k, v, _ = rows.split([nh * hd, kvh * hd, kvh * hd, (nh + 7) // 8 * 8], -1)
    q = q.reshape(S, L, kvh, grp, hd).permute(0, 2, 3, 1, 4).reshape(S * kvh, grp * L, hd).contiguous()
    k = k.reshape(S, L, kvh, hd).permute(0, 2, 3, 1).reshape(S * kvh, hd, L).contiguous()
    v = v.reshape(S, L, kvh, hd).transpose(1, 2).reshape(S * kvh, L, hd).contiguous()
    p = torch.bmm(q, k).mul_(hd ** -0.5).view(S * kvh, grp, L, L)
    p.masked_fill_(at > at[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(S * kvh, grp * L, L), v).view(S * kvh, grp, L, hd) / total
    o = o.view(S, nh, L, hd).transpose(1, 2)                                    # [S][L][nh][hd]
    s = torch.arange(S, device=DEV).repeat_interleave(start[1:] - start[:-1], output_size=f.shape[0])
    return o[s, torch.arange(f.shape[0], device=DEV) - start[s]].reshape(-1, nh * hd).to(f.dtype)


def _plain_moe(st):
    case, x = st["case"], st["x"].float()
    E, F, D, n, k = case["experts"], case["ff"], case["embd"], case["rows"], case["top_k"]
    z = st["logits"].double()
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    score = p + st["bias"].double() if case["bias"] else p
    sel = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, sel)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = w.float()
    silu = lambda a: a / (1 + torch.exp(-a))
    if n * k <= E:                       # the chosen experts' weights, one copy per route
        at = sel.reshape(-1)
        xr = x.repeat_interleave(k, 0)[..., None]
        h = silu(torch.bmm(st["gate"][at].float(), xr)) * torch.bmm(st["up"][at].float(), xr)
        y = torch.bmm(st["down"][at].float(), h).view(n, k, D)
        out = (w[..., None] * y).sum(1)
    else:                                # all experts on all rows, weights of 0 for the others
        h = silu(x @ st["gate"].float().view(E * F, D).T) * (x @ st["up"].float().view(E * F, D).T)
        full = torch.zeros((n, E), device=DEV).scatter_(1, sel, w)
        h = (h.view(n, E, F) * full[..., None]).transpose(0, 1).contiguous()
        out = torch.bmm(h, st["down"].float().transpose(1, 2).contiguous()).sum(0)
    return out.to(st["x"].dtype), sel.int(), w


def _plain_fork(st):
    case, table, refs = st["case"], st["table"], st["refs"]
    P, T = case["page"], table.shape[1]
    src, dst, rows, room = (st[n].long() for n in ("src", "dst", "rows", "room"))
    at = torch.arange(T, device=DEV)
    given, taken = table[dst].long(), table[src].long()
    whole, part = rows // P, (rows % P > 0).long()
    pages = torch.maximum((room + P - 1) // P, whole + part)
    shared = at < whole[:, None]
    count = torch.zeros(refs.numel() + 1, dtype=torch.int64, device=DEV)        # the last: entries that name no page
    count[:-1] = refs
    count.index_add_(0, torch.where(given >= 0, given, refs.numel()).view(-1), torch.full((given.numel(),), -1, device=DEV))
    count.index_add_(0, torch.where(shared, taken, refs.numel()).view(-1), torch.ones((given.numel(),), dtype=torch.int64, device=DEV))
    free = torch.sort((count[:-1] > 0).int(), stable=True).indices              # free pages first, ascending
    need = pages - whole
    new = (~shared) & (at < pages[:, None])
    rank = (need.cumsum(0) - need)[:, None] + at - whole[:, None]
    page = free[rank.clamp(0, refs.numel() - 1)]
    count.index_add_(0, torch.where(new, page, refs.numel()).view(-1), torch.ones((given.numel(),), dtype=torch.int64, device=DEV))
    table[dst] = torch.where(shared, taken, torch.where(new, page, -1)).int()
    refs.copy_(count[:-1])
    # the rows behind the last whole page (prompts that end with a page copy none: their first page onto itself)
    i = whole.clamp(max=T - 1)[:, None]
    a, b = (torch.where(part > 0, t.gather(1, i)[:, 0], taken[:, 0]) for t in (taken, page))
    mine = (torch.arange(P, device=DEV) < (rows % P)[:, None])[None, :, None, :, None]
    for c in (st["k"], st["v"]):
        c[:, b] = torch.where(mine, c[:, a], c[:, b])
    return table, refs, (pages * P).clamp(max=T * P).minimum(room.maximum(rows)).int(), st["k"], st["v"]


def _plain_compact(st):
    table, refs = st["table"].long(), st["refs"].long()
    n, n_max = refs.numel(), refs.numel()
    used = refs > 0
    n_used = used.sum()
    ids = torch.arange(n, device=DEV)
    moves = used & (ids >= n_used)
    holes = ~used & (ids < n_used)
    # the i-th page behind goes into the i-th hole
    order = torch.sort((~moves).int(), stable=True).indices
    hole = torch.sort((~holes).int(), stable=True).indices
    m = moves.sum()
    rank = moves.long().cumsum(0) - 1
    to = torch.where(moves, hole[rank.clamp(min=0)], ids)
    new_refs = torch.zeros(n_max, dtype=torch.int64, device=DEV)
    new_refs.index_add_(0, to, torch.where(used, refs, 0))
    new_table = torch.where(table >= 0, to[table.clamp(min=0)], -1)
    k = int(m)
    for c in (st["k"], st["v"]):
        c[:, hole[:k]] = c[:, order[:k]]
    return new_table.int(), new_refs.int(), n_used.int().view(1), st["k"], st["v"]


def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_prompt, "moe": _plain_moe, "fork": _plain_fork, "compact": _plain_compact}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _mean(lo, hi):
    return lo if lo == hi else (hi - lo) / math.log(hi / lo)                    # of log-uniform lengths


def _mean_square(lo, hi):
    return lo * lo if lo == hi else (hi * hi - lo * lo) / (2 * math.log(hi / lo))


def work(case):
    op = case["op"]
    if op == "prompt":
        lo, hi, S = case["low"], case["high"], case["seqs"]
        rest = S - 1 if S > 1 else 0                                            # one of several has the largest length
        n = rest * _mean(lo, hi) + hi
        seen = (rest * (_mean_square(lo, hi) + _mean(lo, hi)) + hi * hi + hi) / 2
        return {"bytes": int(n * 2 * (case["heads"] + case["kv_heads"]) * case["hd"] * SIZE[case["type"]]),
                "flops": int(4 * seen * case["heads"] * case["hd"])}
    if op == "moe":
        E, F, D, n, k = case["experts"], case["ff"], case["embd"], case["rows"], case["top_k"]
        touched = E * (1 - (1 - k / E) ** n)                                    # experts that a row takes, routing even
        return {"bytes": int(touched * 3 * F * D * 2 + 2 * n * D * SIZE[case["type"]] + 4 * n * (E + 2 * k)), "flops": int(6 * n * k * F * D)}
    row = case["layers"] * 2 * case["kv_heads"] * case["hd"] * 2                # bytes of a cache row in all layers
    P = case["page"]
    if op == "fork":
        n = case["prompts"] * case["forks"]
        total = _pages_of(case["rows"] + case["room"], P)
        part = (P - 1) / 2
        return {"bytes": int(2 * n * part * row + 4 * n * (3 * total + 5)), "flops": 0}
    S, shared, total = case["seqs"], case["shared"] // P, _pages_of(case["rows"], P)
    gone = min(S - 1, max(1, int(round(S * case["gone"]))))
    mean = (max(case["rows"] // 2, case["shared"] + 1) + case["rows"]) / 2 / P - shared
    pages = shared + S * mean
    freed = gone * mean
    moved = freed * (1 - freed / pages)                                         # of holes spread evenly, those in front
    return {"bytes": int(2 * moved * P * row + 8 * (S * total + pages)), "flops": 0}


# ---------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    return {"prompt": _exact_prompt, "moe": _exact_moe, "fork": _exact_fork, "compact": _exact_compact}[case["op"]](case, _inputs(case, seed))


def _exact_prompt(case, st):
    """Every prompt and head by itself."""
    nh, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    f, bounds = st["fused"], st["start"].tolist()
    out = torch.empty((f.shape[0], nh * hd), dtype=torch.float64, device=DEV)
    for a, b in zip(bounds[:-1], bounds[1:]):
        hidden = torch.ones((b - a, b - a), dtype=torch.bool, device=DEV).triu(1)
        for h in range(nh):
            g = h // (nh // kvh)
            q = f[a:b, h * hd:(h + 1) * hd].double()
            k = f[a:b, (nh + g) * hd:(nh + g + 1) * hd].double()
            v = f[a:b, (nh + kvh + g) * hd:(nh + kvh + g + 1) * hd].double()
            out[a:b, h * hd:(h + 1) * hd] = torch.softmax((q @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1) @ v
    return out


def _exact_moe(case, st):
    """Every row by itself, expert by expert."""
    k = case["top_k"]
    logits = st["logits"].cpu().numpy().astype(np.float64)
    bias = st["bias"].cpu().numpy().astype(np.float64) if case["bias"] else 0.0
    out, sels, weights = [], [], []
    for t in range(case["rows"]):
        e = np.exp(logits[t] - logits[t].max())
        p = e / e.sum()
        sel = np.argsort(-(p + bias), kind="stable")[:k]
        w = p[sel] / (p[sel].sum() if case["renorm"] else 1.0)
        x, y = st["x"][t].double(), 0.0
        for e, we in zip(sel.tolist(), w.tolist()):
            g = st["gate"][e].double() @ x
            y = y + we * (st["down"][e].double() @ (g * torch.sigmoid(g) * (st["up"][e].double() @ x)))
        out.append(y), sels.append(sel), weights.append(w)
    return torch.stack(out), torch.from_numpy(np.array(sels, np.int32)).to(DEV), torch.from_numpy(np.array(weights)).to(DEV)


def _exact_fork(case, st):
    """Sequence by sequence, as the definition has it."""
    P = case["page"]
    table, refs, src, dst, rows, room = (st[n].cpu().numpy().copy() for n in ("table", "refs", "src", "dst", "rows", "room"))
    for d in dst:
        for p in table[d][table[d] >= 0]:
            refs[p] -= 1
        table[d] = -1
    held = []
    for s, d, r in zip(src, dst, rows):
        refs[table[s, :r // P]] += 1
    free = iter(np.nonzero(refs == 0)[0].tolist())
    K, V = st["k"].double(), st["v"].double()
    for s, d, r, want in zip(src, dst, rows, room):
        table[d, :r // P] = table[s, :r // P]
        for j in range(r // P, -(-max(want, r) // P)):
            table[d, j] = next(free)
            refs[table[d, j]] = 1
        if r % P:
            for c in (K, V):
                c[:, table[d, r // P], :, :r % P] = c[:, table[s, r // P], :, :r % P]
        held.append(max(want, r))
    return (*(torch.from_numpy(np.asarray(a, np.int32)).to(DEV) for a in (table, refs, held)), K, V)


def _exact_compact(case, st):
    table, refs = st["table"].cpu().numpy().copy(), st["refs"].cpu().numpy().copy()
    n = int((refs > 0).sum())
    K, V = st["k"].double(), st["v"].double()
    behind = [p for p in range(n, len(refs)) if refs[p]]
    for a, b in zip(behind, [p for p in range(n) if not refs[p]]):
        K[:, b], V[:, b] = K[:, a], V[:, a]
        table[table == a] = b
        refs[b], refs[a] = refs[a], 0
    return (*(torch.from_numpy(np.asarray(t, np.int32)).to(DEV) for t in (table, refs, [n])), K, V)
