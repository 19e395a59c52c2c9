"""attention_scored's masks in combinations: documents that begin before the key axis or end behind it, with prefixes, lengths and offsets, against the
float64 definition with the bounds of tests/test_attention_scored_gpu.py."""
import random

import pytest
import torch

from test_attention_scored_gpu import TYPES, _both, _i32

pytestmark = pytest.mark.gpu

# A prefix counts from its document's first boundary, also where that lies before the key axis (a cache whose oldest frames were dropped).
CASES = [
    (1, 2, 1, 64, 26, 26, 6, dict(causal=True, docs=_i32([[-3, 8, 11, 20]]), prefix=_i32([[6, 8, 4]]), lengths=_i32([22]))),
    (2, 2, 2, 96, 150, 150, None, dict(causal=True, docs=_i32([[-40, 100, 150], [-1, 0, 170]]), prefix=_i32([[60, 20], [1, 90]]))),
    (2, 4, 2, 32, 9, 80, 3, dict(causal=True, docs=_i32([[-20, 75], [-2 ** 31, 2 ** 31 - 1]]), prefix=_i32([[95, ], [2 ** 31 - 1]]), offset=_i32([60, 71]))),
    (2, 2, 1, 128, 33, 70, None, dict(causal=True, docs=_i32([[-5, -2, 60], [-30, 40, 90]]), prefix=_i32([[9, 50], [100, -7]]), offset=_i32([37, 20]))),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[:7]}")
def test_prefixes_of_documents_that_begin_before_the_keys(dev, case, dt):
    _both(dev, TYPES[dt], *case[:6], W=case[6], **case[7])


@pytest.mark.parametrize("seed", range(40))
def test_drawn_masks(dev, seed):
    """Heads, sizes and every option drawn; boundaries, lengths and offsets from a little outside the axis."""
    r = random.Random(seed)
    G = r.choice([1, 2, 3])
    H, B, dk = G * r.choice([1, 2, 3]), r.choice([1, 2, 5]), r.choice([r.randint(1, 128), 64, 96, 128])
    Tk = r.choice([r.randint(1, 40), r.randint(40, 200)])
    Tq = r.choice([Tk, r.randint(1, Tk)])
    kw = {"causal": True} if r.random() < 0.6 else {}
    if r.random() < 0.6:
        n = r.randint(1, 5)
        kw["docs"] = _i32([sorted(r.randint(-6, Tk + 6) for _ in range(n + 1)) for _ in range(B)])
    if r.random() < 0.3:
        kw["window"] = r.randint(0, Tk)
    elif "causal" in kw and r.random() < 0.7:
        row = lambda n: [r.randint(-4, Tk + 6) for _ in range(n)]  # noqa: E731
        kw["prefix"] = _i32([row(kw["docs"].shape[1] - 1) for _ in range(B)] if "docs" in kw else row(B))
    if r.random() < 0.4:
        kw["lengths"] = _i32([r.randint(-1, Tk + 2) for _ in range(B)])
    if Tq < Tk and r.random() < 0.6:
        kw["offset"] = r.choice([r.randint(0, Tk - Tq), _i32([r.randint(-Tq - 2, Tk + 2) for _ in range(B)])])
    if r.random() < 0.3:
        kw["softcap"] = r.choice([2.0, 30.0, 300.0])
    _both(dev, r.choice(list(TYPES.values())), B, H, G, dk, Tq, Tk, W=r.choice([None, 0, r.randint(1, Tk + 20)]), p=r.choice([0.0, 0.0, 0.3]), seed=seed, **kw)
