"""How many bits z2h_moe_rows keeps: of hidden values, where a difference of nearly equal ones shows them, and in routing, where a bias keeps a
row's most probable expert out or decides between nearly equal ones."""
import numpy as np
import pytest
import torch

from ops_helpers import DEV, check, context, half_step
from test_gpu_ops_moe import Layer, route

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


def routed(ctx, logits, bias, k, renorm):
    m = Layer("f32", logits.shape[1], 8, 8, logits.shape[0], k, renorm=renorm)
    m.logits, m.bias = logits, bias
    d = m.put(ctx)
    m.call(ctx, d)
    torch.cuda.synchronize()
    return d["sel"].cpu().numpy(), d["w"].cpu().double().numpy()


def check_weights(got, want):
    """Formed in 64 bits and rounded once: half a step of fp32, its smallest one at the least."""
    assert np.allclose(got, want, rtol=2.0 ** -24 * (1 + 2.0 ** -10), atol=2.0 ** -149), np.abs(got / np.where(want, want, 1) - 1).max()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_a_bias_keeps_the_most_probable_expert_out(ctx, typ):
    """The chosen experts' probabilities are e^-120 and less: their shares of each other are not."""
    for n in (1, 9):
        m = Layer(typ, 3, 16, 24, n, 2, renorm=True)
        m.logits, m.bias = torch.tensor([[0.0, -120.0, -121.0]]).repeat(n, 1), torch.tensor([-2.0, 0.0, 0.0])
        d = m.check(ctx, typ)
        check_weights(d["w"].cpu().double().numpy(), np.array([[1.0, np.exp(-1.0)]] * n) / (1 + np.exp(-1.0)))


def test_shares_of_probabilities_below_64_bits(ctx):
    """800 and more below the largest logit p is 0 to 64 bits, so that the index decides; the shares of the chosen are still theirs."""
    logits, bias = torch.tensor([[0.0, -801.0, -800.0], [3e38, -5.0, -4.0], [0.0, -3e38, -3e38]]), torch.tensor([-2.0, 0.0, 0.0])
    sel, w = routed(ctx, logits, bias, 2, True)
    assert sel.tolist() == [[1, 2]] * 3
    e = np.exp(-1.0)
    check_weights(w, np.array([[e / (1 + e), 1 / (1 + e)]] * 2 + [[0.5, 0.5]]))


def test_order_of_small_probabilities(ctx):
    """Under a bias of zeros the order is that of the probabilities, however small."""
    logits = torch.tensor([[0.0, -120.0, -110.0], [-300.0, 0.0, -200.0], [-104.5, -104.25, 0.0]])
    sel, w = routed(ctx, logits, torch.zeros(3), 2, False)
    assert sel.tolist() == [[0, 2], [1, 2], [2, 1]]
    check_weights(w, route(logits.double().numpy(), np.zeros(3), 2, False)[1])


@pytest.mark.parametrize("E", [3, 64, 70, 300, 1024])
@pytest.mark.parametrize("n", [1, 5, 20])
def test_routing_is_in_64_bits(ctx, E, n):
    """Probabilities far below the largest one, which a bias keeps out, and nearly equal ones, whose order biases of their differences' size
    decide: experts as in 64 bits, weights rounded once."""
    print(f"routing E {E} rows {n}", flush=True)
    g = torch.Generator().manual_seed(100 * E + n)
    top, k = E // 2, min(E - 1, 8)
    for low, high in ((-130.0, -100.0), (-104.0, -87.0), (-650.0, -600.0), (-1e-6, 1e-6)):
        logits = low + (high - low) * torch.rand((n, E), generator=g)
        if high < 0:
            logits[:, top] = 0.0
        for scale in (0.0, (high - low) / E if high > 0 else 1e-40):
            bias = torch.randn(E, generator=g) * scale
            bias[top] = -2.0
            for renorm in (False, True):
                sel, w = routed(ctx, logits, bias, k, renorm)
                want = route(logits.double().numpy(), bias.double().numpy(), k, renorm)
                assert np.array_equal(sel, want[0]), (low, scale, renorm)
                check_weights(w, want[1])
