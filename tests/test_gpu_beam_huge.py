"""Beam selection of logits so large that fp32 cannot scale them: the lowest finite value as a mask, and beyond 2^30."""
import numpy as np
import pytest

from tests.test_gpu_beam import run
from tinygpt_b200 import workloads as W

pytestmark = pytest.mark.gpu

LOWEST = {"f32": np.finfo(np.float32).min, "bf16": W.bf16_bits_to_f32(np.array([0xff7f], np.uint16))[0]}


def defined(x, scores, allowed=None):
    """The definition: lse in 64 bits rounded to fp32, score = fl(score + fl(x - lse)); [B, K * V]."""
    B, K = scores.shape
    z = x if allowed is None else np.where(allowed, x, np.float32(-np.inf))
    top = z.max(1, keepdims=True).astype(np.float64)
    base = np.where(np.isfinite(top), top, 0.0)
    with np.errstate(divide="ignore"):
        lse = (base + np.log(np.exp(z.astype(np.float64) - base).sum(1, keepdims=True))).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        s = (z - lse).astype(np.float32) + scores.reshape(-1, 1)
    return np.where(z > -np.inf, s, np.float32(-np.inf)).reshape(B, -1)


def expect(x, scores, got, allowed=None):
    """Ids as the definition orders them; scores to fp32 rounding (no two of these candidates are closer than that
    but for equal logits of one beam, which keep their order)."""
    ref = defined(x, scores, allowed)
    V = x.shape[1]
    for b in range(len(scores)):
        want = np.lexsort((np.arange(ref.shape[1]), -ref[b]))[:scores.shape[1]]
        there = ref[b][want] > -np.inf
        assert got[0][b].tolist() == np.where(there, want // V, -1).tolist()
        assert got[1][b].tolist() == np.where(there, want % V, -1).tolist()
        np.testing.assert_allclose(got[2][b][there], ref[b][want][there], rtol=2.0 ** -21, atol=2.0 ** -18)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [7, 256, 1000, 5003])
def test_a_beam_of_the_lowest_value(cuda_lib, dtype, V):
    """Every logit of a beam is the lowest finite value: each token has its score (log V is below fp32's rounding
    of such an lse), and no more than that."""
    x = np.random.default_rng(V).standard_normal((3, V)).astype(np.float32)
    if dtype == "bf16":
        x = W.bf16_bits_to_f32(W.to_bf16_bits(x))
    x[1] = LOWEST[dtype]
    for scores in ([-1.0, -40.0, -2.0], [-1.0, -0.5, -2.0]):
        s = np.array([scores], np.float32)
        got, status = run(x, s, dtype=dtype)
        assert status == 0
        expect(x, s, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [256, 20000])
def test_the_lowest_value_under_a_mask(cuda_lib, dtype, V):
    """Five tokens allowed, all of them at the lowest finite value."""
    x = np.random.default_rng(1).standard_normal((2, V)).astype(np.float32)
    if dtype == "bf16":
        x = W.bf16_bits_to_f32(W.to_bf16_bits(x))
    bits = np.zeros((1, (V + 31) // 32 * 32), bool)
    five = np.array([3, 40, 41, 200, V - 1])
    bits[0, five] = True
    x[1, five] = LOWEST[dtype]
    s = np.array([[-9.0, -3.0]], np.float32)
    allowed = np.stack([np.ones(V, bool), bits[0, :V]])
    got, _ = run(x, s, dtype=dtype, table=W.pack_mask(bits).view(np.int32), state=np.array([-1, 0], np.int32))
    expect(x, s, got, allowed)
    assert got[0][0].tolist() == [1, 1] and got[1][0].tolist() == [3, 40] and got[2][0].tolist() == [-3.0, -3.0]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("low", ["lowest", -1e9, -1e10, -1e30])
def test_masked_by_a_large_negative_value(cuda_lib, dtype, low):
    """Most of a row at the mask's value, before, between and after ordinary logits: as if it were -inf there."""
    V, K = 40000, 4
    r = np.random.default_rng(2)
    x = r.standard_normal((K, V)).astype(np.float32) * 3
    fill = LOWEST[dtype] if low == "lowest" else np.float32(low)
    x[0, :20000] = fill
    x[1, r.random(V) < 0.5] = fill
    x[2, 100:] = fill
    x[3, :-3] = fill
    if dtype == "bf16":
        x = W.bf16_bits_to_f32(W.to_bf16_bits(x))
    s = np.array([[-1.0, -1.25, -8.5, -3.0]], np.float32)
    got, _ = run(x, s, dtype=dtype)
    ref = defined(x, s)[0]
    gap = np.abs(np.diff(np.sort(ref)[-5:]))
    if (gap > 1e-5).all():  # f32: no two of the best are within rounding
        expect(x, s, got)
    np.testing.assert_allclose(got[2][0], np.sort(ref)[::-1][:K], rtol=2.0 ** -21, atol=2.0 ** -18)


@pytest.mark.parametrize("size", [1e9, 3e10, 1e20, 2.3e38])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_rows(cuda_lib, size, sign):
    """All logits of a row of one large size: each of V has the score of its beam less log V, or, where fp32 cannot
    hold lse so finely, the definition's rounding of that."""
    V = 300
    x = np.full((2, V), np.float32(sign * size))
    x[1] = np.linspace(-2, 2, V, dtype=np.float32)
    x[0, 17] = np.nextafter(x[0, 17], np.float32(-np.inf))
    s = np.array([[-1.0, -30.0]], np.float32)
    got, _ = run(x, s)
    expect(x, s, got)
