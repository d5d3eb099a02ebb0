"""How many bits z2h_moe_rows keeps between its products, where a difference of nearly equal values shows them."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, check, context, half_step
from test_gpu_ops_moe import Layer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = context()
    yield c
    c.close()


def near_pairs(n, seed):
    """n pairs of hidden values silu(g) u of bf16 numbers g and u that differ by 2^-15 to 2^-13 of themselves: [n][2][g, u] and their h."""
    steps = 1 + np.arange(128) / 128
    g = np.concatenate([0.5 * steps, steps, 2 * steps])
    g, u = (a.ravel() for a in np.meshgrid(g, steps))
    h = g / (1 + np.exp(-g)) * u
    order = np.argsort(h, kind="stable")
    gap = np.diff(h[order]) / h[order][1:]
    at = np.nonzero((gap > 2.0 ** -15) & (gap < 2.0 ** -13))[0]
    at = np.random.default_rng(seed).permutation(at)[:n]
    pick = np.stack([order[at], order[at + 1]], 1)
    return np.stack([g[pick], u[pick]], -1), h[pick]


@pytest.mark.parametrize("n", [1, 5, 20])
def test_hidden_values_keep_24_bits_with_bf16_experts(ctx, n):
    """out_d = h_2d - h_(2d+1) of neighbours 2^-14 apart; row t has its gates and ups in column t, so that their products with it are exact.

    Each h is off by 12 roundings of 2^-24 of its own (the exponential, the division, the product) and by one as it meets `down`; its parts are
    multiplied by 1 or -1 and summed in fp32, where no sum exceeds h: 8 roundings more. 34 2^-24 h for both, then the output's half step, 2^-8
    of a difference of 2^-13 h."""
    D = 512
    m = Layer("bf16", 1, 8, 8, n, 1, renorm=True)
    m.F, m.D = 2 * D, D
    gate, up, down = torch.zeros((1, m.F, D)), torch.zeros((1, m.F, D)), torch.zeros((1, D, m.F))
    ref, size = torch.empty((n, D), dtype=torch.float64), torch.empty((n, D), dtype=torch.float64)
    for t in range(n):
        gu, h = near_pairs(D, t)
        gate[0, :, t], up[0, :, t] = (torch.from_numpy(gu[..., i].ravel()).float() for i in range(2))
        ref[t], size[t] = torch.from_numpy(h[:, 0] - h[:, 1]), torch.from_numpy(h.max(1))
    d = torch.arange(D)
    down[0, d, 2 * d], down[0, d, 2 * d + 1] = 1.0, -1.0
    m.x = torch.eye(n, D).bfloat16()
    for t, src in zip((gate, up, down), ("gate", "up", "down")):
        assert torch.equal(t.bfloat16().float(), t), src
    dev = [t.bfloat16().to(DEV) for t in (gate, up, down)]
    m.ex.gate, m.ex.up, m.ex.down = (t.data_ptr() for t in dev)
    m.ex.n_ff, m.ex.n_embd = m.F, D
    put = m.put(ctx)
    m.call(ctx, put)
    torch.cuda.synchronize()
    check(put["out"], ref, 34 * 2.0 ** -24 * size + half_step(ref, torch.bfloat16) * (1 + 2.0 ** -10), f"{n} rows")
