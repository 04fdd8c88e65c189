"""Cache, tree attention, sampler and beam selection together (examples/decode.py), and the calls' repeated rows."""
import importlib.util
import pathlib

import pytest

pytestmark = pytest.mark.gpu

# What the example's model rounds to 8 significant bits, per layer: q, k, v, the softmax
# weights and the attention's output, each by 2^-9 of its value at most.  With unit-variance
# activations and 2 layers that is about sqrt(10) * 2^-9 = 0.6% of a logit's rms; the largest
# of 512 logits' errors is some 4 times that.  The bound is twice as wide.
TOLERANCE = 0.05


def example():
    at = pathlib.Path(__file__).resolve().parents[1] / "examples" / "decode.py"
    spec = importlib.util.spec_from_file_location("decode_example", at)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def wide(model):
    """The model with 64-bit weights."""
    import copy
    m = copy.copy(model)
    m.embed, m.place, m.head = model.embed.double(), model.place.double(), model.head.double()
    m.blocks = [tuple(w.double() for w in b) for b in model.blocks]
    return m


def logits_of(model, tokens):
    """Logits [len, vocab] after each token, in 64 bits and without a cache."""
    import torch
    t = torch.tensor([tokens], device="cuda")
    n = len(tokens)
    hidden = torch.full((n, n), float("-inf"), dtype=torch.float64, device="cuda").triu(1)

    def attend(layer, q, k, v):
        group = model.q_heads // model.kv_heads
        k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
        s = torch.einsum("bihd,bjhd->bhij", q, k) * model.head_dim ** -0.5 + hidden
        return torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v)

    return model.forward(t, torch.arange(n, device="cuda")[None], attend)[0]


def setup(lengths, seed=3):
    import torch
    d = example()
    model = d.ToyModel(seed=seed)
    g = torch.Generator().manual_seed(seed)
    return d, model, [torch.randint(model.vocab, (n,), generator=g).tolist() for n in lengths]


def test_tree_decode_follows_the_model():
    d, model, prompts = setup((1, 16, 17, 64, 65, 130))
    new = d.tree_decode(model, prompts, 12)
    ref = wide(model)
    assert any(len(t) > 12 for t in new)  # some drafted token was accepted
    for p, t in zip(prompts, new):
        assert 12 <= len(t) <= 12 * 5
        z = logits_of(ref, p + t)[len(p) - 1:-1]
        rms = z.square().mean().sqrt()
        for i, token in enumerate(t):
            assert z[i, token] >= z[i].max() - 2 * TOLERANCE * rms, (len(p), i)


def test_tree_decode_samples():
    d, model, prompts = setup((3, 40))
    new = d.tree_decode(model, prompts, 8, temperature=1.0)
    assert all(8 <= len(t) <= 40 and all(0 <= x < model.vocab for x in t) for t in new)


@pytest.mark.parametrize("beams", [1, 4])
def test_beam_decode_scores(beams):
    import torch
    d, model, prompts = setup((1, 33, 70))
    steps = 9
    ref = wide(model)
    for p, found in zip(prompts, d.beam_decode(model, prompts, steps, beams)):
        scores = [s for _, s in found]
        assert scores == sorted(scores, reverse=True)
        assert len({tuple(t) for t, _ in found}) == beams
        for tokens, score in found:
            assert len(tokens) == steps
            z = logits_of(ref, p + tokens)[len(p) - 1:-1]
            rms = z.square().mean().sqrt().item()
            want = z.log_softmax(-1)[torch.arange(steps), torch.tensor(tokens)].sum().item()
            # a log-probability moves by twice its logits' errors at most
            assert abs(score - want) <= steps * 2 * TOLERANCE * rms


def test_accept_serves_a_repeated_slot_once():
    """Rows 0 and 1 name one slot: one of them is served, the other is reported and does nothing."""
    import torch
    from tinygpt_b200 import PagedCache
    c = PagedCache(1, 1, 16, 8, 16, 3, 4)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    c.extend(i32([0, 1]), i32([20, 20]))
    parents, tokens, ids = i32([[-1, 0, 0, 2]] * 3), i32([[5, 6, 7, 8]] * 3), i32([[7, 0, 8, 9]] * 3)
    out, taken = c.accept(i32([0, 0, 1]), parents, tokens, ids)
    assert c.device_status() == 1
    assert sorted(taken[:2].tolist()) == [0, 3] and taken[2] == 3 and out[2].tolist() == [7, 8, 9, -1]
    assert c.lens.tolist() == [3, 3, 0] and c.counts.tolist() == [1, 1, 0]
    assert c.refs.sum() == 2
    # the slot is free for the next call
    c.extend(i32([0]), i32([4]))
    _, taken = c.accept(i32([0]), parents[:1], tokens[:1], ids[:1])
    assert taken.tolist() == [3] and c.lens.tolist() == [6, 3, 0] and c.device_status() == 0


def test_truncate_of_a_repeated_slot_takes_the_shorter():
    import torch
    from tinygpt_b200 import PagedCache
    c = PagedCache(1, 1, 16, 8, 16, 2, 8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    c.extend(i32([0]), i32([60]))
    c.commit(i32([0]), i32([60]))
    c.truncate(i32([0, 0]), i32([50, 9]))
    assert c.lens[0] == 9 and c.counts[0] == 2 and c.refs.sum() == 2


def forked(nodes):
    """Slot 0 with 11 tokens of value 1, forked to slot 1: both end in one page."""
    import torch
    from tinygpt_b200 import PagedCache
    c = PagedCache(1, 1, 16, 8, 16, 2, 8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    c.extend(i32([0]), i32([11 + nodes]))
    ones = torch.ones((1, 11, 1, 16), dtype=torch.bfloat16, device="cuda")
    c.append(0, i32([0]), ones, ones)
    c.commit(i32([0]), i32([11]))
    c.fork(i32([0]), i32([1]))
    c.k[c.k != 1], c.v[c.v != 1] = 0, 0
    assert c.device_status() == 0
    return c, i32, c.k.clone()


@pytest.mark.parametrize("call", ["append", "attention", "accept"])
def test_nothing_is_stored_into_a_shared_page(call):
    """Until one of a forked pair is extended, neither may store into the page that both end in."""
    import torch
    c, i32, before = forked(3)
    new = torch.full((1, 3, 1, 16), 2.0, dtype=torch.bfloat16, device="cuda")
    for slot in ([0], [1]):
        if call == "append":
            c.append(0, i32(slot), new, new)
        elif call == "attention":
            out = c.tree_attention(0, i32(slot), new, new, new)
            assert out.isfinite().all() and (out > 1).all()  # the nodes are attended to all the same
        else:
            _, taken = c.accept(i32(slot), i32([[-1, 0, 0]]), i32([[5, 6, 7]]), i32([[7, 0, 8]]))
            assert taken.tolist() == [0]
        assert c.device_status() == 8
    assert torch.equal(c.k, before) and c.lens.tolist() == [11, 11]
    # extended, slot 1 has a page of its own, and slot 0 has its page alone again
    c.extend(i32([1]), i32([3]))
    for slot in ([0], [1]):
        if call == "append":
            c.append(0, i32(slot), new, new)
        elif call == "attention":
            c.tree_attention(0, i32(slot), new, new, new)
        else:
            _, taken = c.accept(i32(slot), i32([[-1, 0, 0]]), i32([[5, 6, 7]]), i32([[7, 0, 8]]))
            assert taken.tolist() == [2]
        assert c.device_status() == 0
    if call != "accept":
        assert (c.k == 2).sum() == 2 * 3 * 16
