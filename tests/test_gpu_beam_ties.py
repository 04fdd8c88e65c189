"""Beam selection where fp32 rounding gives different logits one score: the lower token comes first, whichever
logits a part's list kept."""
import numpy as np
import pytest

from tests.test_gpu_beam import run
from tinygpt_b200 import workloads as W

pytestmark = pytest.mark.gpu


def order(x, score, beams, ulps=0):
    """Tokens of one live beam by the definition, its lse moved by some units in the last place."""
    top = x.max().astype(np.float64)
    lse = np.float32(top + np.log(np.exp(x.astype(np.float64) - top).sum()))
    for _ in range(abs(ulps)):
        lse = np.nextafter(lse, np.float32(np.inf if ulps > 0 else -np.inf))
    s = (x - lse) + np.float32(score)
    return np.lexsort((np.arange(len(x)), -s))[:beams].tolist()


def background(V, dtype, seed):
    x = np.random.default_rng(seed).standard_normal(V).astype(np.float32)
    return W.bf16_bits_to_f32(W.to_bf16_bits(x)) if dtype == "bf16" else x


def above(v, dtype, steps=1):
    """The logit some representable values above v."""
    for _ in range(steps):
        v = np.nextafter(v, np.float32(np.inf)) if dtype == "f32" else W.bf16_bits_to_f32(W.to_bf16_bits(np.array([v * np.float32(1 + 2.0 ** -7)])))[0]
    return v


# (beams, score, {token: steps above 6.0}): what a list keeps ends among equal logits, or does not; a lower
# token with a smaller logit of the same score is left out, or is not
CASES = [
    (1, -400.0, {100: 0, 900: 1, 1300: 1}),
    (1, -400.0, {100: 0, 900: 1}),
    (4, -30000.0, {11: 0, 500: 1, 777: 1, 4000: 1, 9000: 1, 15000: 1}),
    (4, -30000.0, {11: 0, 12: 0, 500: 2, 777: 1, 4000: 2, 9000: 1, 15000: 1, 19000: 3}),
    (4, -30000.0, {11: 3, 500: 2, 777: 1, 4000: 1, 9000: 1, 15000: 0}),
    (2, -30000.0, {19000: 5, 18000: 4, 17000: 3, 16000: 2, 15000: 1, 14000: 0}),
    (8, -30000.0, {t: int(t > 9000) for t in range(1000, 20000, 1000)}),
    (4, -30000.0, {11: 0, 20: 1, 21: 1, 22: 1, 23: 1, 24: 1}),  # in one part of the row, whatever the parts
    (8, -30000.0, {**{40 + t: 2 for t in range(7)}, 60: 1, 61: 1, 50: 0}),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("V", [20000, 128256])
def test_one_score_of_many_logits(cuda_lib, dtype, case, V):
    beams, score, places = CASES[case]
    if dtype == "bf16":
        score *= 2.0 ** 16  # whose last place is above a bf16 logit's here
    x = np.tile(background(V, dtype, case), (beams, 1))
    for token, steps in places.items():
        x[0, token] = above(np.float32(6.0), dtype, steps)
    want = order(x[0], score, beams)
    # the sizes are such that no rounding of lse decides
    assert all(order(x[0], score, beams, u) == want for u in (-4, -2, -1, 1, 2, 4))
    scores = np.full((1, beams), -np.inf, np.float32)
    scores[0, 0] = score
    got, _ = run(x, scores, dtype=dtype)
    assert got[0][0].tolist() == [0] * beams and got[1][0].tolist() == want


@pytest.mark.parametrize("seed", range(6))
def test_random_rows_under_a_large_score(cuda_lib, seed):
    """Logits in few distinct values and many last places, beside each other."""
    r = np.random.default_rng(seed)
    V, beams = 30011, 6
    x = background(V, "f32", seed)
    at = r.choice(V, 40, replace=False)
    for t in at:
        x[t] = above(np.float32(7.0), "f32", int(r.integers(0, 4)))
    score = -float(2 ** r.integers(13, 18)) - 0.5
    want = order(x, score, beams)
    assert all(order(x, score, beams, u) == want for u in (-4, -1, 1, 4))
    scores = np.full((1, beams), -np.inf, np.float32)
    scores[0, 2] = score
    got, _ = run(np.tile(x, (beams, 1)), scores)
    assert got[0][0].tolist() == [2] * beams and got[1][0].tolist() == want
