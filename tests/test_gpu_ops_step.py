"""The model's layers over a paged cache (z2h_step_paged): rows of several sequences, some of which share a prefix, against the
oracle's mixed step over one band per sequence; and a speculative loop of it with z2h_verify.

The bar is that of the quantised models end to end (cos >= 0.9999, max-abs 5e-2 per row): the oracle rounds queries to f16 and the
paged attention does not, which moves scores by up to 2^-11 of their size, and the encoding before every projection turns such a
difference into a step of one level now and then."""
import dataclasses

import numpy as np
import pytest
import torch

import ops_helpers as H
import oracle_py as O
from helpers import assert_close
from zonos2_amd import configs, synth, z2h
from zonos2_amd.z2h import Context, Model, Pages, Z2HError

pytestmark = pytest.mark.gpu
BAR = {"maxabs": 5e-2}
EINVAL, ESTATE = 1, 4


def _config(shape):
    if shape == "hd128":
        return dataclasses.replace(configs.zonos2_24l(configs.Q4_K), n_layer=2, expert_used=[4, 4])
    return configs.C1()[0]


def _ids(cfg, n, rng):
    return np.concatenate([rng.integers(0, cfg.audio_vocab, (n, cfg.n_codebooks)),
                           rng.integers(0, cfg.text_vocab + 1, (n, 1))], axis=1).astype(np.int32)


class Paged:
    """Pages of all layers, NaN where nothing was written; table rows by hand."""

    def __init__(self, cfg, table, page, n_pages):
        self.cfg, self.page = cfg, page
        shape = (cfg.n_layer, n_pages, cfg.n_head_kv, page, cfg.head_dim)
        self.k = torch.full(shape, float("nan"), dtype=torch.float16, device=H.DEV)
        self.v = torch.full(shape, float("nan"), dtype=torch.float16, device=H.DEV)
        self.table = np.asarray(table, np.int32)
        self.d_table = H.ints(self.table)
        self.stride = n_pages * cfg.n_head_kv * page * cfg.head_dim
        self.pages = Pages(self.k.data_ptr(), self.v.data_ptr(), cfg.n_head_kv * page * cfg.head_dim, z2h.F16, n_pages, page,
                           cfg.n_head_kv, cfg.head_dim, *self.table.shape, self.d_table.data_ptr())

    def write(self, layer, seq, row0, k, v):
        for i in range(k.shape[0]):
            p, r = self.table[seq, (row0 + i) // self.page], (row0 + i) % self.page
            self.k[layer, p, :, r] = torch.from_numpy(k[i].view(np.float16)).to(H.DEV)
            self.v[layer, p, :, r] = torch.from_numpy(v[i].view(np.float16)).to(H.DEV)

    def read(self, layer, seq, row0, n):
        at = [(int(self.table[seq, r // self.page]), r % self.page) for r in range(row0, row0 + n)]
        return tuple(np.stack([t[layer, p, :, r].float().cpu().numpy() for p, r in at]) for t in (self.k, self.v))

    def workspace(self, ctx, n_rows, n_group):
        n = ctx.step_paged_ws_bytes(self.pages, n_rows, n_group)
        self.ws = torch.zeros(n, dtype=torch.uint8, device=H.DEV)
        return self.ws.data_ptr(), n


def _rows(row_start, kv_len):
    seq = np.concatenate([np.full(row_start[s + 1] - row_start[s], s) for s in range(len(kv_len))]).astype(np.int32)
    pos = np.concatenate([np.arange(kv_len[s] - (row_start[s + 1] - row_start[s]), kv_len[s]) for s in range(len(kv_len))])
    return seq, pos.astype(np.int32)


@pytest.mark.parametrize("shape,page", [("c1", 16), ("c1", 64), ("hd128", 32)])
def test_shared_prefix_against_bands(shape, page):
    cfg = _config(shape)
    model = synth.generate_model(cfg, 49)
    m = Model(cfg.hparams(), model)
    rng = np.random.default_rng(5)
    prefix = 64                                                      # sequences 0 .. 2 share it
    past = [64 + 10, 64 + 3, 64, 130, 7]                             # rows in the cache before; sequence 4 sits out
    new = [1, 5, 40, 1, 0]
    kv_len = [p + n for p, n in zip(past, new)]
    row_start = np.cumsum([0] + new)
    per, shared = 192 // page, prefix // page
    table = np.full((5, per), -1, np.int32)                          # entries behind a sequence's rows are out of range
    free = iter(range(2, 5 * per + 2))
    for s, n in enumerate(kv_len):
        for i in range((n + page - 1) // page):
            table[s, i] = table[0, i] if s in (1, 2) and i < shared else next(free)
    pg = Paged(cfg, table, page, 5 * per + 3)
    ctx = Context(None, 4, 256, model=m)
    om = O.OracleModel(cfg.hparams(), model)
    okv = O.OracleKV(om, 5, 256)
    for L in range(cfg.n_layer):
        pre = synth.kv_rows(cfg, L, 9, prefix, 70)
        for s in range(5):
            k, v = synth.kv_rows(cfg, L, s, past[s], 71)
            if s < 3:
                k[:prefix], v[:prefix] = pre
            okv.write(L, s, 0, k, v)
            pg.write(L, s, 0, k, v)
    seq, pos = _rows(row_start, kv_len)
    n = len(seq)
    ids = _ids(cfg, n, rng)
    emap = np.full(n, -1, np.int32)
    emap[row_start[2]] = 0                                           # a chunk that begins with a speaker row
    emb = rng.standard_normal((1, cfg.n_embd)).astype(np.float32)
    out = np.array([0, 1, 2, 3, 4, 5, 25, n - 2, n - 1], np.int32)
    ws = pg.workspace(ctx, n, 1)
    before = pg.k.clone()
    got = ctx.step_paged(pg.pages, pg.stride, row_start, kv_len, ids, out, *ws, group_start=[0, 3], prefix_len=[prefix],
                         emb_map=emap, emb=emb)
    want = O.step_mixed(om, okv, seq, pos, ids, emb_map=emap, emb=emb)[out]
    for i, r in enumerate(out):
        assert_close(f"row {r}", got[i], want[i], **BAR)
    for s in range(5):
        for L in range(cfg.n_layer):
            if new[s]:
                for a, b, what in zip(pg.read(L, s, past[s], new[s]), okv.read(L, s, past[s], new[s]), "KV"):
                    assert_close(f"{what} rows of {s} L{L}", a, b.view(np.float16).astype(np.float32), **BAR)
    # nothing else of the cache was touched
    written = torch.zeros(pg.k.shape[1], page, dtype=torch.bool)
    for s, r in zip(seq, pos):
        written[table[s, r // page], r % page] = True
    same = (pg.k.view(torch.int16) == before.view(torch.int16)).permute(1, 3, 0, 2, 4).flatten(2).all(-1).cpu()
    assert bool(same[~written].all())
    # and the same pass without groups reads every prefix by itself
    again = ctx.step_paged(pg.pages, pg.stride, row_start, kv_len, ids, out, *ws, emb_map=emap, emb=emb)
    for i, r in enumerate(out):
        assert_close(f"row {r} without groups", again[i], want[i], **BAR)
    ctx.close(); m.close()


def test_prefix_and_its_readers_in_one_pass():
    cfg = _config("c1")
    model = synth.generate_model(cfg, 49)
    m = Model(cfg.hparams(), model)
    rng = np.random.default_rng(6)
    page, prefix, more = 16, 48, [0, 9, 1, 30]
    new = [prefix] + more[1:]
    kv_len = [prefix] + [prefix + x for x in more[1:]]
    table = np.full((4, 6), -1, np.int32)
    table[:, :3] = [5, 3, 9]
    for s in (1, 2, 3):
        table[s, 3:6] = 10 + 3 * s + np.arange(3)
    pg = Paged(cfg, table, page, 24)
    ctx = Context(None, 4, 256, model=m)
    row_start = np.cumsum([0] + new)
    ids = _ids(cfg, row_start[-1], rng)
    out = row_start[1:] - 1
    got = ctx.step_paged(pg.pages, pg.stride, row_start, kv_len, ids, out, *pg.workspace(ctx, len(ids), 1), group_start=[0, 4],
                         prefix_len=[prefix])
    # the oracle runs the prefix in every reader's band
    om = O.OracleModel(cfg.hparams(), model)
    for s in range(4):
        okv = O.OracleKV(om, 1, 256)
        own = ids[row_start[s]:row_start[s + 1]]
        rows = np.concatenate([ids[:prefix], own]) if s else own
        want = O.step_mixed(om, okv, np.zeros(len(rows), np.int32), np.arange(len(rows), dtype=np.int32), rows)
        assert_close(f"last row of {s}", got[s], want[-1], **BAR)
    ctx.close(); m.close()


def test_drafts_step_and_verify():
    """Rounds of drafts over shared pages: a pass over each sequence's frame and its drafts leaves the logits on the device, the
    verification judges them, and the next round begins behind the frames kept. The judgement is exactly that of the logits; the
    logits of a frame are those of a pass that brings it alone."""
    cfg = _config("c1")
    m = Model(cfg.hparams(), synth.generate_model(cfg, 49))
    rng = np.random.default_rng(7)
    C, V, K, S, page, prefix = cfg.n_codebooks, cfg.audio_vocab, 3, 3, 16, 32
    table = np.stack([np.r_[[0, 1], 2 + 6 * s + np.arange(6)] for s in range(S)]).astype(np.int32)
    pg, alone = Paged(cfg, table, page, 24), Paged(cfg, table, page, 24)
    ctx = Context(None, 4, 256, model=m)
    text = np.full((1, 1), cfg.text_vocab, np.int32)
    frame = lambda codes: np.concatenate([np.asarray(codes, np.int32).reshape(1, C), text], 1)
    prompt = _ids(cfg, prefix, rng)
    for p in (pg, alone):
        p.ws1 = p.workspace(ctx, prefix, 1)
        p.keep = p.ws
        ctx.step_paged(p.pages, p.stride, [0, prefix, prefix, prefix], [prefix, 0, 0], prompt, [], *p.ws1)
    last = [frame(rng.integers(0, V, C)) for _ in range(S)]
    length = [prefix] * S
    temperature = torch.full((S,), 0.7, device=H.DEV)
    ws = pg.workspace(ctx, S * (K + 1), 1)
    n_ws = ctx.verify_ws_bytes(S, K, C, V)
    v_ws = torch.zeros(n_ws, dtype=torch.uint8, device=H.DEV)
    target = torch.zeros(S, K + 1, C, V, device=H.DEV)
    for rnd in range(3):
        draft = rng.integers(0, V, (S, K, C)).astype(np.int32)
        ua, ud = rng.random((S, K, C)), rng.random((S, C))
        # what the model itself says, frame by frame in passes of one row; in round 1 its likeliest frames are the first drafts
        ws1 = alone.workspace(ctx, S, 1)
        x, said = [l.copy() for l in last], []
        for k in range(2):
            said.append(ctx.step_paged(alone.pages, alone.stride, range(S + 1), [n + k + 1 for n in length], np.concatenate(x), range(S),
                                       *ws1, group_start=[0, S], prefix_len=[prefix]).reshape(S, C, V))
            if rnd == 1:
                draft[:, k] = said[k].argmax(-1)
                ua[:, k] = 0.0
            x = [frame(draft[s, k]) for s in range(S)]
        ids = np.concatenate([np.concatenate([last[s]] + [frame(draft[s, k]) for k in range(K)]) for s in range(S)])
        ctx.step_paged(pg.pages, pg.stride, [(K + 1) * s for s in range(S + 1)], [n + K + 1 for n in length], ids, range(S * (K + 1)), *ws,
                       group_start=[0, S], prefix_len=[prefix], d_logits=target.data_ptr())
        d = dict(draft=H.ints(draft), ua=torch.tensor(ua, device=H.DEV), ud=torch.tensor(ud, device=H.DEV),
                 n=torch.zeros(S, dtype=torch.int32, device=H.DEV), codes=torch.zeros(S, C, dtype=torch.int32, device=H.DEV))
        ctx.verify(S, K, C, V, d["draft"].data_ptr(), 0, target.data_ptr(), temperature.data_ptr(), 0, d["ua"].data_ptr(),
                   d["ud"].data_ptr(), d["n"].data_ptr(), d["codes"].data_ptr(), v_ws.data_ptr(), n_ws)
        torch.cuda.synchronize()
        logits = target.cpu()
        n, codes = d["n"].cpu().numpy(), d["codes"].cpu().numpy()
        want_n, want_codes = H.verify(draft, np.full(S, K), logits.numpy().astype(np.float64), np.full(S, np.float32(0.7)), None, ua, ud)
        assert np.array_equal(n, want_n) and np.array_equal(codes, want_codes)
        assert rnd != 1 or (n >= 2).all()
        for s in range(S):
            for k in range(2):
                assert_close(f"frame {length[s] + k} of {s}", logits[s, k].numpy(), said[k][s], **BAR)
        for s in range(S):                                           # the kept frames' rows stay; the next round overwrites the others
            rows = [last[s]] + [frame(draft[s, k]) for k in range(n[s])]
            ctx.step_paged(alone.pages, alone.stride, [0] * (s + 1) + [len(rows)] * (S - s),
                           [length[s] + len(rows) if t == s else 0 for t in range(S)], np.concatenate(rows), [],
                           *alone.workspace(ctx, len(rows), 0))
            length[s] += len(rows)
            last[s] = frame(codes[s])
    ctx.close(); m.close()


def test_refusals():
    cfg = _config("c1")
    m = Model(cfg.hparams(), synth.generate_model(cfg, 49))
    rng = np.random.default_rng(8)
    pg = Paged(cfg, [[0, 1], [0, 2]], 16, 3)
    ctx = Context(None, 4, 256, model=m)
    ids = _ids(cfg, 3, rng)
    ws, n_ws = pg.workspace(ctx, 3, 1)
    good = dict(pages=pg.pages, layer_stride=pg.stride, row_start=[0, 1, 3], kv_len=[17, 20], ids=ids, out_rows=[0], d_ws=ws, ws_bytes=n_ws,
                group_start=[0, 2], prefix_len=[16])

    def pages(**kw):
        p = Pages.from_buffer_copy(pg.pages)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    bad_id = ids.copy()
    bad_id[1, 0] = cfg.audio_vocab + 5
    for bad in (dict(kv_len=[0, 20]), dict(kv_len=[17, 33]), dict(kv_len=[17, 17]), dict(row_start=[0, 4, 3]), dict(row_start=[1, 1, 3]),
                dict(row_start=[0, 1, 2]), dict(ids=ids[:0], row_start=[0, 0, 0]), dict(ids=bad_id), dict(out_rows=[3]), dict(out_rows=[-1]), dict(layer_stride=pg.stride - 8),
                dict(layer_stride=pg.stride + 4), dict(d_ws=ws + 16), dict(ws_bytes=n_ws - 1), dict(d_ws=0), dict(group_start=[0, 3]),
                dict(group_start=[1, 0]), dict(prefix_len=[-1]), dict(emb_map=[0, -1, -1]), dict(pages=pages(type=z2h.BF16)),
                dict(pages=pages(n_head_kv=cfg.n_head_kv + 1)), dict(pages=pages(head_dim=64)), dict(pages=pages(page_rows=24)),
                dict(pages=pages(k=0)), dict(emb_map=[0, 1, -1], emb=np.zeros((1, cfg.n_embd), np.float32))):
        with pytest.raises(Z2HError) as e:
            ctx.step_paged(**{**good, **bad})
        assert e.value.code == EINVAL and str(e.value), bad
    ctx.set_capture(True)
    with pytest.raises(Z2HError) as e:
        ctx.step_paged(**good)
    assert e.value.code == ESTATE
    ctx.set_capture(False)
    assert np.isfinite(pg.k.float().cpu().numpy()).sum() == 0        # no refused call wrote a row
    ctx.close(); m.close()
