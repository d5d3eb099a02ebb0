"""The operators on device tensors in calls of more blocks than one launch may have."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, Cache, context, half_step, ints, rotate, rotate_tol
from zonos2_amd import z2h

pytestmark = pytest.mark.gpu
SLICE = 1 << 23                                             # blocks of 256 threads per launch


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()
    torch.cuda.empty_cache()


def _at(n):
    """Rows to look at: both ends, and both sides of a launch's end."""
    r = np.unique(np.concatenate([np.arange(50), np.arange(SLICE - 50, SLICE + 50), np.arange(n - 50, n), np.random.default_rng(1).integers(0, n, 500)]))
    return torch.from_numpy(r[r < n])


def test_rope_rows(ctx):
    n = 2 * SLICE + 3
    print(f"rope {n} rows", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((n, 1, 2), generator=g, device=DEV).half()
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device=DEV, dtype=torch.int32)
    out = torch.full_like(x, float("nan"))
    ctx.rope_rows(z2h.Rope(base=10000.0, n_dims=2), n, 1, 2, z2h.F16, x.data_ptr(), 2, out.data_ptr(), 2, pos.data_ptr())
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all())
    i = _at(n).to(DEV)
    a = x[i].double().cpu()
    ref = rotate(a, pos[i].long().cpu(), 10000.0, 2, False)
    assert bool(((out[i].double().cpu() - ref).abs() <= rotate_tol(a, ref, 2, False, 1.0, torch.float16)).all())


def test_append(ctx):
    """Padding but for the rows at the ends and around the launch's end."""
    n, hd = SLICE + 200, 32
    print(f"append {n} rows", flush=True)
    live = torch.cat([torch.arange(20), torch.arange(SLICE - 20, SLICE + 20), torch.arange(n - 20, n)])
    c = Cache([128, 128], 1, hd, 16, torch.float16, 3, fill=0.0)
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn((n, 2 * hd), generator=g, device=DEV).half()
    seq, pos = torch.full((n,), -1, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    seq[live.to(DEV)] = ints(np.arange(len(live)) % 2)
    pos[live.to(DEV)] = ints(np.arange(len(live)) // 2)
    ctx.paged_append(c.pages, z2h.Rope(base=10000.0, n_dims=hd), n, seq.data_ptr(), pos.data_ptr(), z2h.F16, x.data_ptr(), 2 * hd,
                     x.data_ptr() + 2 * hd, 2 * hd)
    torch.cuda.synchronize()
    rows = x[live.to(DEV)].double().cpu()
    k = rotate(rows[:, None, :hd], pos[live.to(DEV)].long().cpu(), 10000.0, hd, False)
    tol = rotate_tol(rows[:, None, :hd], k, hd, False, 1.0, torch.float16)
    for i in range(len(live)):
        s, p = i % 2, i // 2
        page, r = c.table_host[s, p // 16], p % 16
        got = [b[page].view(1, 16, hd)[:, r].double().cpu() for b in c.dev]
        assert bool(((got[0] - k[i]).abs() <= tol[i]).all()), i
        assert torch.equal(got[1][0], rows[i, hd:]), i
    for b, old in zip(c.dev, c.buf):                         # the rows behind those appended
        for s in range(2):
            assert torch.equal(b[c.table_host[s, 3:8]].cpu(), old[c.table_host[s, 3:8]])


def test_attention_of_the_most_rows_and_heads(ctx):
    """2^20 rows of 64 heads, one cache row each, in place; the last four behind a shared prefix, so that results are joined in the last launch."""
    S, H, hd, P, N = 1 << 20, 64, 32, 4096, 64
    print(f"attention {S} rows of {H} heads", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn((N, 1, P, hd), generator=g, device=DEV).half() for _ in range(2))
    at = torch.arange(S, device=DEV)
    table = torch.stack([at % N, (at + 1) % N], 1).int().contiguous()
    table[-4:, 0] = 7
    kv_len = torch.ones(S, dtype=torch.int32, device=DEV)
    kv_len[-4:] = P + 1
    pages = z2h.Pages(k=k.data_ptr(), v=v.data_ptr(), page_stride=P * hd, type=z2h.F16, n_pages=N, page_rows=P, n_head_kv=1, head_dim=hd,
                      table=table.data_ptr(), n_seq=S, table_len=2)
    row_start = torch.arange(S + 1, device=DEV, dtype=torch.int32)
    group, prefix = ints([S - 4, S]), ints([P])
    q = torch.zeros((S, H * hd), dtype=torch.float16, device=DEV)        # every key alike: the mean of the values
    ws = torch.empty(ctx.paged_ws_bytes(pages, H, S, 1), dtype=torch.uint8, device=DEV)
    ctx.paged_plan(pages, H, S, row_start.data_ptr(), kv_len.data_ptr(), 1, group.data_ptr(), prefix.data_ptr(), ws.data_ptr(), ws.numel())
    ctx.paged_attn(pages, H, S, 1, 0.1, z2h.F16, q.data_ptr(), H * hd, q.data_ptr(), H * hd, ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    out = q.view(S, H, hd)
    want = v[table[:, 0].long(), 0, 0]                                   # one key: its value itself
    for r in range(0, S - 4, 1 << 16):
        e = min(r + (1 << 16), S - 4)
        assert torch.equal(out[r:e], want[r:e, None].expand(-1, H, -1)), r
    for s in range(S - 4, S):
        rows = torch.cat([v[7, 0], v[int(table[s, 1]), 0, :1]]).double()
        ref = rows.mean(0)
        tol = half_step(ref, torch.float16) * 1.001 + rows.abs().mean(0) * (8 * P ** 0.5 + 100) * 2.0 ** -24
        assert bool(((out[s].double() - ref).abs() <= tol).all()), s


def test_verify_of_more_rows_than_a_launch_has_blocks(ctx):
    """Long rows of logits, each with one largest code, without temperature: a frame is kept where its draft is that code."""
    S, K, V = 700001, 2, 8193
    print(f"verify {S} sequences", flush=True)
    rows = S * (K + 1)
    assert rows > 1 << 21
    target = torch.zeros((rows, V), device=DEV)
    hot = torch.arange(rows, device=DEV) * 7919 % V
    target[torch.arange(rows, device=DEV), hot] = 1.0
    best = hot.view(S, K + 1)
    draft = best[:, :K].clone()
    at = torch.arange(S, device=DEV)
    draft[at % 3 == 0, 0] = (best[at % 3 == 0, 0] + 1) % V   # nothing kept
    draft[at % 3 == 1, 1] = (best[at % 3 == 1, 1] + 1) % V   # one frame kept
    u, draw, T = (torch.full(s, 0.5, dtype=t, device=DEV) for s, t in (((S, K), torch.float64), ((S, 1), torch.float64), ((S,), torch.float32)))
    T.zero_()
    n, codes = torch.full((S,), -9, dtype=torch.int32, device=DEV), torch.full((S,), -9, dtype=torch.int32, device=DEV)
    ws = torch.empty(ctx.verify_ws_bytes(S, K, 1, V), dtype=torch.uint8, device=DEV)
    d = draft.int().contiguous()
    ctx.verify(S, K, 1, V, d.data_ptr(), 0, target.data_ptr(), T.data_ptr(), 0, u.data_ptr(), draw.data_ptr(), n.data_ptr(), codes.data_ptr(),
               ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    want = at % 3
    assert torch.equal(n.long(), want) and torch.equal(codes.long(), best[at, want])
