"""Beam selection against its definition in 64 bits.

Two candidates of different beams whose scores are closer than fp32 rounding may come in
either order, so ids are checked through their scores: each chosen candidate has the
score it is given, the scores fall, and nothing left out is better by more than the
rounding.  A score is two fp32 additions of numbers up to |x|, |lse|, |score|, and lse
carries one rounding and a sum accurate to about 2^-21: the bound is 2^-21 of their
sizes.  Within a beam the order is exact, and so are all cases of one beam.
"""
import ctypes

import numpy as np
import pytest

from tests.decode_reference import beam_reference
from tinygpt_b200 import _lib
from tinygpt_b200 import workloads as W

pytestmark = pytest.mark.gpu


def run(x, scores, *, dtype="f32", finished=None, table=None, state=None, eos=-1, pad=0, history=None, length=None, offset=0, stride=None):
    """x: float32 logits [B * W, V] (already bf16 values for bf16); offset, stride: elements."""
    import torch
    from tinygpt_b200 import BeamSearch
    rows, V = x.shape
    B, K = scores.shape
    stride = stride or V
    buf = torch.full((rows * stride + offset,), float("nan"), device="cuda", dtype=torch.float32 if dtype == "f32" else torch.bfloat16)
    t = buf[offset:offset + rows * stride].view(rows, stride)
    t[:, :V] = torch.from_numpy(x).cuda().to(buf.dtype)
    h = BeamSearch(V, K, B)
    cu = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    r = h.select(t, cu(scores), finished=cu(finished), eos_id=eos, pad_id=pad, mask_table=cu(table), state_id=cu(state),
                 history=cu(history), history_len=cu(length))
    return [None if v is None else v.cpu().numpy() for v in r], h.device_status()


def check(x, scores, got, finished=None, allowed=None, pad=0):
    B, K = scores.shape
    V = x.shape[1]
    ref = beam_reference(x.astype(np.float64), scores, finished, allowed, pad)
    parents, tokens, best = got[:3]
    xr = x.reshape(B, K, V)
    for b in range(B):
        there = int((ref[b] > -np.inf).sum())
        n = min(K, there)
        assert (tokens[b, n:] == -1).all() and (parents[b, n:] == -1).all() and (best[b, n:] == -np.inf).all()
        at = parents[b, :n].astype(np.int64) * V + tokens[b, :n]
        assert len(set(at.tolist())) == n and (at >= 0).all() and (at < K * V).all()
        tol = 2.0 ** -21 * (np.abs(best[b, :n]).max(initial=0) + np.abs(scores[b][np.isfinite(scores[b])]).max(initial=0) + 2 * np.nanmax(np.abs(np.where(np.isfinite(xr[b]), xr[b], 0))) + 16)
        np.testing.assert_allclose(best[b, :n], ref[b][at], rtol=0, atol=tol)
        assert (np.diff(best[b, :n]) <= 0).all()
        rest = np.delete(ref[b], at)
        if n == K and rest.size:
            assert rest.max() <= best[b, n - 1] + tol
        # in a beam: a higher logit first, of equal ones the lower token
        for w in set(parents[b, :n].tolist()):
            if finished is not None and finished[b, w]:
                assert tokens[b, :n][parents[b, :n] == w].tolist() == [pad]
                continue
            mine = tokens[b, :n][parents[b, :n] == w]
            v = np.where(np.isnan(xr[b, w]), -np.inf, np.minimum(xr[b, w], np.finfo(np.float32).max))
            if allowed is not None:
                v = np.where(allowed.reshape(B, K, V)[b, w], v, -np.inf)
            want = np.lexsort((np.arange(V), -v))[:len(mine)]
            assert v[mine].tolist() == v[want].tolist()
            assert sorted(mine.tolist()) == sorted(want.tolist())


def inputs(B, K, V, dtype, seed=0, std=3.0):
    g = np.random.default_rng(seed)
    x = (g.standard_normal((B * K, V)) * std).astype(np.float32)
    if dtype == "bf16":
        x = W.bf16_bits_to_f32(W.to_bf16_bits(x))
    return x, -(g.random((B, K)) * 20).astype(np.float32), g


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 3), (2, 3, 7), (3, 5, 1000), (2, 32, 257), (5, 8, 4099), (1, 16, 50257),
                                   (9, 2, 32000), (2, 4, 128256), (40, 4, 5003)])
def test_shapes(cuda_lib, B, K, V, dtype):
    x, scores, _ = inputs(B, K, V, dtype, seed=B * 7 + K)
    got, status = run(x, scores, dtype=dtype)
    assert status == 0
    check(x, scores, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset,stride", [(0, 5008), (1, 5003), (3, 5010), (5, 5017)])
def test_rows_off_the_boundary(cuda_lib, dtype, offset, stride):
    x, scores, _ = inputs(3, 4, 5003, dtype, seed=11)
    got, _ = run(x, scores, dtype=dtype, offset=offset, stride=stride)
    check(x, scores, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [50, 5003, 128256])
def test_masks(cuda_lib, dtype, V):
    """Full, sparse, single-token and empty mask rows, unmasked rows, a state id past the table."""
    B, K = 3, 4
    x, scores, g = inputs(B, K, V, dtype, seed=V)
    words = (V + 31) // 32
    bits = np.zeros((5, words * 32), bool)
    bits[0, :V] = True
    bits[1, :V] = g.random(V) < 0.05
    bits[2, V // 2] = True
    bits[4, :V] = g.random(V) < 0.5
    table = W.pack_mask(bits)
    state = np.array([0, 1, 2, 3, -1, 4, 3, 1, 3, 3, 3, 3], np.int32)
    allowed = np.where((state < 0)[:, None], True, bits[np.maximum(state, 0), :V])
    got, status = run(x, scores, dtype=dtype, table=table.view(np.int32), state=state)
    assert status == 0
    check(x, scores, got, allowed=allowed)
    assert (got[0][2] == -1).all() and (got[3][2] == 1).all()  # the third row has nothing to choose from
    state[0] = 5
    _, status = run(x, scores, dtype=dtype, table=table.view(np.int32), state=state)
    assert status == 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_finished_and_dead_beams(cuda_lib, dtype):
    B, K, V = 4, 4, 1003
    x, scores, g = inputs(B, K, V, dtype, seed=3)
    finished = np.array([[0, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 1], [1, 0, 0, 0]], np.int32)
    scores[0, 1] = -0.5
    scores[2, :3] = -np.inf
    scores[3, 1:] = [-np.inf, np.nan, -np.inf]
    got, _ = run(x, scores, dtype=dtype, finished=finished, eos=7, pad=5)
    s = np.where(np.isnan(scores), -np.inf, scores)
    check(x, s, got, finished=finished, pad=5)
    assert got[0][0, 0] == 1 and got[1][0, 0] == 5 and got[2][0, 0] == np.float32(-0.5)
    assert sorted(got[0][1].tolist()) == [0, 1, 2, 3] and (got[3][1] == 1).all()
    assert got[0][2].tolist() == [3, -1, -1, -1] and (got[3][2] == 1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_eos(cuda_lib, dtype):
    """A beam that takes eos is finished; with eos_id -1 none is."""
    x, scores, _ = inputs(1, 4, 1003, dtype, seed=4)
    scores[0] = [-1.0, -9.0, -9.0, -9.0]
    x[0, 7] = 50.0
    got, _ = run(x, scores, dtype=dtype, eos=7)
    assert got[0][0, 0] == 0 and got[1][0, 0] == 7 and got[3][0].tolist() == (got[1][0] == 7).astype(int).tolist()
    got, _ = run(x, scores, dtype=dtype)
    assert got[1][0, 0] == 7 and not got[3].any()


def test_first_step(cuda_lib):
    """One live beam of four, as at the start of a search: all the next beams are its children."""
    x, _, _ = inputs(1, 4, 3001, "f32", seed=8)
    scores = np.array([[0, -np.inf, -np.inf, -np.inf]], np.float32)
    got, _ = run(x, scores)
    want = np.argsort(-x[0], kind="stable")[:4]
    assert got[0].tolist() == [[0] * 4] and got[1][0].tolist() == want.tolist()


@pytest.mark.parametrize("V", [40, 5003, 128256])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties(cuda_lib, V, dtype):
    """All logits equal; a rising row; few distinct values; equal beams: the lower index wins."""
    K = 8
    scores = np.zeros((1, K), np.float32)
    flat = np.zeros((K, V), np.float32)
    got, _ = run(flat, scores, dtype=dtype)
    assert got[0][0].tolist() == [0] * K and got[1][0].tolist() == list(range(K))
    scores = np.full((1, K), -np.inf, np.float32)
    scores[0, 3] = -1.0
    up = np.tile(np.arange(V, dtype=np.float32) / 64, (K, 1))
    if dtype == "bf16":
        up = W.bf16_bits_to_f32(W.to_bf16_bits(up))
    got, _ = run(up, scores, dtype=dtype)
    want = np.lexsort((np.arange(V), -up[3]))[:K]
    assert got[0][0].tolist() == [3] * K and got[1][0].tolist() == want.tolist()
    few = np.random.default_rng(1).integers(0, 3, (K, V)).astype(np.float32)
    got, _ = run(few, scores, dtype=dtype)
    assert got[1][0].tolist() == np.lexsort((np.arange(V), -few[3]))[:K].tolist()


def test_scores_that_rounding_makes_equal(cuda_lib):
    """Logits one ulp apart under a large negative beam score: their fp32 scores are equal, so the lower
    token comes first although its logit is the smaller one."""
    V, K = 20000, 4
    x = np.full((K, V), -10.0, np.float32)
    at = np.array([11, 500, 777, 4000, 9000, 15000, 19000])
    v = np.float32(3.0)
    for i, t in enumerate(at):  # rising with the token
        x[0, t] = v
        v = np.nextafter(v, np.float32(9))
    scores = np.array([[-30000.0, -np.inf, -np.inf, -np.inf]], np.float32)
    got, _ = run(x, scores)
    assert got[1][0].tolist() == at[:4].tolist()
    assert len(set(got[2][0].tolist())) == 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_and_nan(cuda_lib, dtype):
    """NaN counts as -inf, +inf as the largest finite value; huge finite logits; a row of nothing."""
    K, V = 2, 3000
    x, _, _ = inputs(1, K, V, dtype, seed=5)
    scores = np.array([[-1.0, -2.0]], np.float32)
    for place, what in ((5, np.nan), (2999, np.nan), (7, -np.inf)):
        y = x.copy()
        y[0, place] = what
        got, _ = run(y, scores, dtype=dtype)
        check(np.where(np.isnan(y), -np.inf, y), scores, got)
    y = x.copy()
    y[1, 40] = np.inf
    y[1, 30] = np.inf
    got, _ = run(y, scores, dtype=dtype)
    # both infinite tokens have log-probability 0 in fp32 (their lse rounds to the largest value)
    assert got[0][0].tolist() == [1, 1] and got[1][0].tolist() == [30, 40] and got[2][0].tolist() == [-2.0, -2.0]
    y = x.copy()
    y[0] = -3e38
    y[0, 9] = 3e38
    if dtype == "bf16":
        y = W.bf16_bits_to_f32(W.to_bf16_bits(y))
    got, _ = run(y, scores, dtype=dtype)
    assert got[0][0, 0] == 0 and got[1][0, 0] == 9 and got[2][0, 0] == -1.0
    y[0] = -3e38 if dtype == "f32" else W.bf16_bits_to_f32(W.to_bf16_bits(np.full(V, -3e38, np.float32)))
    got, _ = run(y, np.array([[0.0, -np.inf]], np.float32), dtype=dtype)
    assert got[1][0].tolist() == [0, 1] and np.allclose(got[2][0], -np.log(V), atol=1e-4) or got[2][0].tolist() == [0.0, 0.0]
    y[:] = -np.inf
    got, _ = run(y, scores, dtype=dtype)
    assert (got[0] == -1).all() and (got[1] == -1).all() and (got[2] == -np.inf).all() and (got[3] == 1).all()


@pytest.mark.parametrize("stride,full", [(1, 1), (17, 17), (1024, 1000)])
def test_histories(cuda_lib, stride, full):
    B, K, V = 3, 4, 501
    x, scores, g = inputs(B, K, V, "f32", seed=stride)
    finished = (g.random((B, K)) < 0.3).astype(np.int32)
    history = g.integers(0, V, (B * K, stride)).astype(np.int32)
    length = g.integers(0, full + 1, B * K).astype(np.int32)
    length[0], length[1] = 0, full
    scores[1] = [-1, -np.inf, -np.inf, -np.inf]
    finished[1] = [1, 0, 0, 0]
    got, status = run(x, scores, finished=finished, history=history, length=length, pad=2)
    assert status == 0
    parents, tokens, _, _, new, new_len = got
    for b in range(B):
        for w in range(K):
            r, p = b * K + w, parents[b, w]
            if p < 0:
                assert new_len[r] == 0 and (new[r] == -1).all()
                continue
            n = length[b * K + p]
            want = history[b * K + p, :n].tolist()
            if not finished[b, p] and n < stride:
                want.append(tokens[b, w])
            assert new_len[r] == len(want) and new[r].tolist() == want + [-1] * (stride - len(want))
    length[2] = stride + 5
    _, status = run(x, scores, history=history, length=length)
    assert status in (0, 2)  # told only where the beam is a parent
    length[:] = -1
    _, status = run(x, scores, history=history, length=length)
    assert status == 2


def test_same_twice_and_on_another_stream(cuda_lib):
    import torch
    from tinygpt_b200 import BeamSearch
    x, scores, _ = inputs(8, 8, 32000, "bf16", seed=2)
    h = BeamSearch(32000, 8, 8)
    t, s = torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(scores).cuda()
    a = h.select(t, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = h.select(t, s)
    torch.cuda.current_stream().wait_stream(side)
    c = h.select(t[:64], s[:8], stream=None)
    for u, v, w in zip(a[:4], b[:4], c[:4]):
        assert torch.equal(u, v) and torch.equal(u, w)


def test_refusals(cuda_lib):
    import torch
    from tinygpt_b200 import BeamSearch
    h = BeamSearch(100, 4, 2)
    x, s = torch.zeros((8, 100), device="cuda"), torch.zeros((2, 4), device="cuda")
    big = ctypes.c_void_p()
    assert cuda_lib.tg_beam_create(0, 0, 4, 1, ctypes.byref(big)) == _lib.TG_ERR_UNSUPPORTED
    assert cuda_lib.tg_beam_create(0, 100, 33, 1, ctypes.byref(big)) == _lib.TG_ERR_UNSUPPORTED
    assert cuda_lib.tg_beam_create(0, 100, 4, 0, ctypes.byref(big)) == _lib.TG_ERR_INVALID_ARG
    assert cuda_lib.tg_beam_create(55, 100, 4, 1, ctypes.byref(big)) == _lib.TG_ERR_NO_DEVICE
    for call in (lambda: h.select(x[:, :99], s), lambda: h.select(x[:4], s), lambda: h.select(x, s.double()),
                 lambda: h.select(x.t().contiguous().t(), s), lambda: h.select(x, s, finished=torch.zeros((2, 4), device="cuda")),
                 lambda: h.select(x, s, state_id=torch.zeros(8, dtype=torch.int32, device="cuda")),
                 lambda: h.select(x, s, history=torch.zeros((8, 4), dtype=torch.int32, device="cuda")),
                 lambda: h.select(x.cpu(), s)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        h.select(x.half(), s)
    for kw in (dict(eos_id=100), dict(eos_id=-2), dict(pad_id=100), dict(pad_id=-1)):
        with pytest.raises(_lib.TGError):
            h.select(x, s, **kw)
    with pytest.raises(_lib.TGError):
        BeamSearch(100, 4, 1).select(x, s)
    assert h.device_status() == 0
