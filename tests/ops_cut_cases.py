"""Calls of the paged attention that take it where small ones do not: walks of many steps, shares that have parts of several strips, plans of more
tiles and spans than a block has threads, tables longer than its LDS holds. What each is there for (`reaches`) is checked on the CPU from
the rules that the plan uses, and the results on the GPU. Blocks: those of 256 compute units."""
import numpy as np

BLOCKS = 512


def _lens(seed, n, lo, hi):
    return [int(x) for x in np.exp(np.random.default_rng(seed).uniform(np.log(lo), np.log(hi), n)).round()]


def _cases():
    # one shared prefix of 160 steps for two tiles of 16 key heads: pieces of many steps; the second tile leaves a wave without rows
    yield dict(name="long walks of four waves", typ="f16", lens=[10240 + 3 * s for s in range(1, 27)], rows=[1] * 26, heads=128, kvh=16, hd=64, page=64,
               groups=[(0, 26, 10240)], reaches=lambda narrow, wide: wide["longest"] >= 5 and wide["small"] >= 1)
    yield dict(name="long walks of four waves, fp32", typ="f32", lens=[10240 + 3 * s for s in range(1, 24)], rows=[1] * 23, heads=64, kvh=16, hd=128, page=16,
               groups=[(0, 23, 10240)], reaches=lambda narrow, wide: wide["longest"] >= 5 and wide["small"] >= 1)
    yield dict(name="long walks of one wave", typ="bf16", lens=_lens(2, 24, 3000, 9000), rows=[1] * 24, heads=32, kvh=16, hd=64, page=32, groups=(),
               reaches=lambda narrow, wide: narrow["longest"] >= 12)
    # more strips than shares: parts of several strips in a share
    yield dict(name="many narrow strips", typ="f16", lens=_lens(3, 330, 1, 700), rows=[1] * 330, heads=16, kvh=8, hd=64, page=16, groups=(),
               reaches=lambda narrow, wide: narrow["head"] > 0 and narrow["several"] > 400)
    yield dict(name="many narrow strips, fp32", typ="f32", lens=_lens(4, 100, 1, 500) + [64] + _lens(14, 229, 1, 500), rows=[1] * 330, heads=16, kvh=8, hd=128, page=64, stride_pad=24,
               groups=[(0, 100, 1), (100, 330, 40)], reaches=lambda narrow, wide: narrow["head"] > 0 and narrow["several"] > 400)
    yield dict(name="many wide strips", typ="f16", lens=[n + 12 for n in _lens(5, 90, 1, 600)], rows=[12] * 90, heads=32, kvh=8, hd=64, page=16, groups=(),
               reaches=lambda narrow, wide: wide["head"] > 0 and wide["several"] > 100 and wide["small"] > 0)
    yield dict(name="many wide strips, fp32", typ="f32", lens=[n + 40 for n in _lens(6, 75, 1, 400)], rows=[40] * 75, heads=16, kvh=8, hd=32, page=128, stride_pad=8,
               groups=(), reaches=lambda narrow, wide: wide["head"] > 0 and wide["several"] > 100)
    yield dict(name="wide and narrow strips in a row", typ="bf16", lens=[n + 37 for n in _lens(7, 160, 1, 900)], rows=[37, 1] * 80, heads=32, kvh=8, hd=64, page=32,
               groups=[(0, 40, 30)], reaches=lambda narrow, wide: wide["head"] > 0 and narrow["longest"] >= 1)
    # one strip far longer than all others, wide and narrow: few whole shares fit
    yield dict(name="uneven lengths", typ="f16", lens=[12000] + _lens(8, 63, 1, 60), rows=[20] + [1] * 63, heads=16, kvh=8, hd=32, page=16, groups=(),
               reaches=lambda narrow, wide: narrow["longest"] >= 1 and wide["longest"] >= 3)
    # more spans and tiles than the plan's threads, and than its table in LDS
    yield dict(name="many sequences", typ="f32", lens=[9 + n % 40 for n in range(1400)] + [n % 12 for n in range(100)], rows=[n % 3 for n in range(1500)], heads=4, kvh=2, hd=32, page=16,
               groups=[(i, i + 5, 9) for i in range(0, 1400, 7)], reaches=lambda narrow, wide: narrow["tiles"] > 1024)
    yield dict(name="more narrow tiles than LDS holds", typ="f16", lens=_lens(9, 9000, 1, 70), rows=[1] * 9000, heads=1, kvh=1, hd=32, page=16, groups=(),
               reaches=lambda narrow, wide: narrow["tiles"] > 8192 and narrow["head"] > 0)
    yield dict(name="more wide tiles than LDS holds", typ="bf16", lens=_lens(10, 8500, 1, 130), rows=[1] * 8500, heads=33, kvh=1, hd=32, page=32, groups=(),
               reaches=lambda narrow, wide: wide["tiles"] > 8192 and wide["head"] > 0 and wide["several"] > 1000)


CASES = {c["name"]: c for c in _cases()}


def group_tables(case):
    """group_start, prefix_len as the attention's test helper passes them: sequences between groups become groups that share nothing."""
    start, prefix, at = [], [], 0
    for a, b, n in case["groups"]:
        if a > at:
            start.append(at), prefix.append(0)
        start.append(a), prefix.append(n)
        at = b
    return start + [at], prefix
