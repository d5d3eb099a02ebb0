"""z2h_verify against its definition in 64 bits (integers, equal): probabilities and logits, drafts with and without
probabilities of their own, one codebook and nine, vocabularies from one code to more than a block's share, draws at the
border, rows without mass, a replayed graph; and that the frames are distributed as the target's."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, context, ints, verify
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def _dev(a, dtype=None):
    return None if a is None else torch.as_tensor(a if dtype is None else np.asarray(a, dtype)).to(DEV)


def _run(ctx, draft, n_draft, target, temperature, draft_probs, u_accept, u_draw, stream=0):
    S, K1, C, V = target.shape
    t = [_dev(draft, np.int32), _dev(n_draft, np.int32), _dev(target, np.float32), _dev(temperature, np.float32),
         _dev(draft_probs, np.float32), _dev(u_accept, np.float64), _dev(u_draw, np.float64)]
    n, codes = torch.full((S,), -9, dtype=torch.int32, device=DEV), torch.full((S, C), -9, dtype=torch.int32, device=DEV)
    ws = torch.empty(ctx.verify_ws_bytes(S, K1 - 1, C, V), dtype=torch.uint8, device=DEV)
    p = [0 if x is None else x.data_ptr() for x in t]
    ctx.verify(S, K1 - 1, C, V, p[0], p[1], p[2], p[3], p[4], p[5], p[6], n.data_ptr(), codes.data_ptr(), ws.data_ptr(), ws.numel(),
               stream=stream)
    torch.cuda.synchronize()
    return n.cpu().numpy(), codes.cpu().numpy()


def _case(S, K, C, V, logits, probs, seed, noise=0.4):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((S, K + 1, C, V)) * 2).astype(np.float32)
    y = x[:, :K] + noise * rng.standard_normal((S, K, C, V)).astype(np.float32)
    e = np.exp(y - (y.max(-1, keepdims=True) if K else 0))
    q = (e / e.sum(-1, keepdims=True)).astype(np.float32) if K else np.zeros((S, 0, C, V), np.float32)
    draft = np.array([[[rng.choice(V, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in f] for f in s] for s in q]).reshape(S, K, C)
    if not probs:
        draft = y.argmax(-1) if K else draft
        for s, k, c in np.ndindex(S, K, C):
            x[s, k, c, draft[s, k, c]] += 6
    e = np.exp(x - x.max(-1, keepdims=True))
    target = x if logits else (e / e.sum(-1, keepdims=True)).astype(np.float32)
    T = rng.uniform(0.6, 1.2, S).astype(np.float32) if logits else None
    if logits and S > 2:
        T[1] = 0.0                                          # greedy
    return dict(draft=draft.astype(np.int32), n_draft=rng.integers(0, K + 1, S).astype(np.int32), target=target, temperature=T,
                draft_probs=q if probs else None, u_accept=rng.random((S, K, C)), u_draw=rng.random((S, C)))


@pytest.mark.parametrize("S,K,C,V", [(1, 0, 1, 1), (1, 1, 1, 1), (3, 2, 2, 2), (5, 4, 9, 1025), (16, 3, 9, 1026), (4, 5, 1, 255), (4, 5, 1, 257),
                                     (64, 1, 1, 300), (2, 3, 1, 20000), (2, 2, 1, 131072), (1, 1, 2, 70001), (300, 2, 1, 64)])
@pytest.mark.parametrize("logits", [True, False], ids=["logits", "probs"])
@pytest.mark.parametrize("probs", [True, False], ids=["drawn", "given"])
def test_verify(ctx, S, K, C, V, logits, probs):
    print(f"verify {S} {K} {C} {V} {logits} {probs}", flush=True)
    c = _case(S, K, C, V, logits, probs, S * 131 + K * 17 + V)
    n, codes = _run(ctx, **c)
    want_n, want = verify(**c)
    np.testing.assert_array_equal(n, want_n)
    np.testing.assert_array_equal(codes, want)
    if S >= 16 and K >= 2:                                  # the case has sequences that end early and whole ones
        assert (want_n < c["n_draft"]).any() and (want_n == c["n_draft"]).any()


def test_all_frames_by_default_and_clamped(ctx):
    c = _case(6, 3, 2, 50, False, True, 4)
    c["n_draft"] = np.full(6, 3, np.int32)
    want = verify(**c)
    for nd in (None, np.full(6, 100, np.int32)):
        got = _run(ctx, **dict(c, n_draft=nd))
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
    c["n_draft"] = np.full(6, -4, np.int32)
    got, want = _run(ctx, **c), verify(**dict(c, n_draft=np.zeros(6, np.int32)))
    np.testing.assert_array_equal(got[1], want[1])
    assert (got[0] == 0).all()


def test_borders(ctx):
    """Exact masses: u on a cumulative sum goes to the next code, u q = p is not kept, equal rows leave nothing to draw
    from the rest, zeros are never drawn, a drafted code out of range is not kept."""
    V = 600
    p = np.zeros((8, 2, 1, V), np.float32)
    p[:, :, 0, [3, 300, 598]] = [0.25, 0.5, 0.25]
    q = p[:, :1].copy()
    draft = np.full((8, 1, 1), 300, np.int32)
    ua, ud = np.zeros((8, 1, 1)), np.zeros((8, 1))
    ud[:, 0] = [0.0, 0.25, np.nextafter(0.25, 0), 0.75, np.nextafter(1, 0), 0.5, 0.0, 0.9]
    ua[4] = 0.999
    draft[5] = 7                                            # p = q = 0 there: u q = p, not kept, nothing left: drawn from p
    draft[6], draft[7] = -1, V                              # out of range
    q[3, 0, 0, 300] = 0.875                                 # u q = 0.4375 < 0.5: kept; below, u q = 0.5: not kept
    ua[3] = 0.5
    q[2, 0, 0, 300], ua[2] = 1.0, 0.5
    q[2, 0, 0, 3] = 0.0
    c = dict(draft=draft, n_draft=np.ones(8, np.int32), target=p, temperature=None, draft_probs=q, u_accept=ua, u_draw=ud)
    n, codes = _run(ctx, **c)
    np.testing.assert_array_equal(n, [1, 1, 0, 1, 1, 0, 0, 0])
    np.testing.assert_array_equal(codes[:, 0], [3, 300, 3, 598, 598, 300, verify(**c)[1][6, 0], verify(**c)[1][7, 0]])
    np.testing.assert_array_equal(codes, verify(**c)[1])


def test_no_numbers_stay_in_range(ctx):
    """NaN, infinities and rows without mass give some code in [0, V)."""
    for logits in (True, False):
        c = _case(6, 2, 2, 700, logits, True, 8)
        c["target"][0] = np.nan
        c["target"][1] = -np.inf if logits else 0.0
        c["target"][2, :, :, 5] = np.inf
        c["draft_probs"][3] = np.nan
        c["u_draw"][4] = np.nan
        if logits:
            c["temperature"][5] = np.nan
        n, codes = _run(ctx, **c)
        assert ((n >= 0) & (n <= 2)).all() and ((codes >= 0) & (codes < 700)).all()


def test_one_huge_logit_and_masked_ones(ctx):
    c = _case(4, 2, 1, 3000, True, False, 2)
    c["target"][:, :, :, 1000:] = -np.inf                   # masked codes have no mass
    c["draft"][0, 0, 0] = 2000
    c["n_draft"][:] = 2
    c["target"][1, :, :, 77] = 1e30
    n, codes = _run(ctx, **c)
    want_n, want = verify(**c)
    np.testing.assert_array_equal(n, want_n)
    np.testing.assert_array_equal(codes, want)
    assert n[0] == 0 and (codes < 1000).all()


def test_frames_follow_the_target(ctx):
    """40000 sequences with one drafted frame from q: the first frame's codes follow p (each count within 5 standard
    deviations), though q is far from it."""
    rng = np.random.default_rng(77)
    S, V = 40000, 6
    p = np.array([0.05, 0.3, 0.1, 0.25, 0.0, 0.3], np.float32)
    q = np.array([0.3, 0.1, 0.2, 0.1, 0.2, 0.1], np.float32)
    draft = rng.choice(V, p=q.astype(np.float64) / q.astype(np.float64).sum(), size=(S, 1, 1)).astype(np.int32)
    c = dict(draft=draft, n_draft=np.ones(S, np.int32), target=np.broadcast_to(p, (S, 2, 1, V)).copy(), temperature=None,
             draft_probs=np.broadcast_to(q, (S, 1, 1, V)).copy(), u_accept=rng.random((S, 1, 1)), u_draw=rng.random((S, 1)))
    n, codes = _run(ctx, **c)
    first = np.where(n == 1, draft[:, 0, 0], codes[:, 0])
    counts = np.bincount(first, minlength=V)
    pd = p.astype(np.float64) / p.astype(np.float64).sum()
    assert (np.abs(counts - S * pd) <= 5 * np.sqrt(S * pd * (1 - pd)) + 1e-9).all(), counts
    assert abs((n == 1).mean() - np.minimum(p, q).sum()) < 5 * 0.5 / np.sqrt(S)


def test_replayed_graph(ctx):
    c = _case(8, 3, 9, 1025, True, True, 6)
    t = {k: _dev(v) for k, v in c.items()}
    n, codes = torch.zeros(8, dtype=torch.int32, device=DEV), torch.zeros((8, 9), dtype=torch.int32, device=DEV)
    ws = torch.empty(ctx.verify_ws_bytes(8, 3, 9, 1025), dtype=torch.uint8, device=DEV)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        ctx.verify(8, 3, 9, 1025, *(t[k].data_ptr() for k in ("draft", "n_draft", "target", "temperature", "draft_probs", "u_accept", "u_draw")),
                   n.data_ptr(), codes.data_ptr(), ws.data_ptr(), ws.numel(), stream=side.cuda_stream)
    for seed in (6, 7, 8, 9):
        c = _case(8, 3, 9, 1025, True, True, seed)
        for k, v in c.items():
            t[k].copy_(torch.as_tensor(v))
        graph.replay()
        torch.cuda.synchronize()
        want_n, want = verify(**c)
        np.testing.assert_array_equal(n.cpu().numpy(), want_n)
        np.testing.assert_array_equal(codes.cpu().numpy(), want)
        torch.randn(1000, device=DEV).sum().item()


def test_refusals(ctx):
    t = torch.zeros(4096, dtype=torch.float64, device=DEV)
    p = t.data_ptr()
    ok = dict(S=1, K=1, C=1, V=10, draft=p, target=p, ua=p, ud=p, n=p, codes=p, ws=p, wb=t.numel() * 8)
    for bad in (dict(S=-1), dict(K=-1), dict(C=0), dict(V=0), dict(V=(1 << 20) + 1), dict(draft=0), dict(target=0), dict(ua=0), dict(ud=0),
                dict(n=0), dict(codes=0), dict(ws=0), dict(ws=p + 8), dict(wb=8)):
        a = dict(ok, **bad)
        with pytest.raises(z2h.Z2HError):
            ctx.verify(a["S"], a["K"], a["C"], a["V"], a["draft"], 0, a["target"], 0, 0, a["ua"], a["ud"], a["n"], a["codes"], a["ws"], a["wb"])
    with pytest.raises(z2h.Z2HError):
        ctx.verify_ws_bytes(1, 1, 1, 0)
    ctx.verify(0, 1, 1, 10, p, 0, p, 0, 0, p, p, p, p, p, t.numel() * 8)
