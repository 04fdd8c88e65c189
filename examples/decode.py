"""Decoding with the paged cache: drafted trees, and beam search, on a small random transformer.

    python examples/decode.py

`tree_decode` runs a speculative step per pass: a draft table proposes a tree of tokens for
every sequence, one forward pass scores all of its nodes (PagedCache.tree_attention), the
sampler chooses a token at each node, and PagedCache.accept keeps the path that the choices
follow, in the cache too.  `beam_decode` runs BeamSearch.select and lets PagedCache.fork give
the new beams their parents' pages.  Neither loop waits for the device: lengths, paths and
parents stay there, and the results are read once at the end.
"""
from __future__ import annotations

import pathlib
import sys

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from tinygpt_b200 import BeamSearch, PagedCache, Sampler, row_params, tree_masks  # noqa: E402
from tinygpt_b200.sampler import params_to_device  # noqa: E402

# A tree of 12 nodes: the last token, its 3 likeliest successors, and so on.  PARENTS[i] < i;
# RANKS[i] says which of its parent's drafted successors node i is.
PARENTS = [-1, 0, 0, 0, 1, 1, 2, 3, 4, 4, 6, 8]
RANKS = [0, 0, 1, 2, 0, 1, 0, 0, 0, 1, 0, 0]
DEPTHS = [0, 1, 1, 1, 2, 2, 2, 2, 3, 3, 3, 4]


class ToyModel:
    """Pre-norm transformer with grouped heads and learned positions; float32 but for what the cache holds."""

    def __init__(self, vocab=512, hidden=128, layers=2, q_heads=8, kv_heads=2, head_dim=32, positions=512, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        w = lambda *shape: (torch.randn(shape, generator=g) / shape[-2] ** 0.5).to(device)  # noqa: E731
        self.vocab, self.layers, self.q_heads, self.kv_heads, self.head_dim = vocab, layers, q_heads, kv_heads, head_dim
        self.embed = torch.randn((vocab, hidden), generator=g).to(device)
        self.place = torch.randn((positions, hidden), generator=g).to(device)
        wide = (q_heads + 2 * kv_heads) * head_dim
        self.blocks = [(w(hidden, wide), w(q_heads * head_dim, hidden), w(hidden, 4 * hidden), w(4 * hidden, hidden)) for _ in range(layers)]
        self.head = w(hidden, vocab)

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def forward(self, tokens, positions, attend):
        """Logits [n, nodes, vocab]; attend(layer, q, k, v) [n, nodes, q_heads, head_dim]."""
        n, nodes = tokens.shape
        x = self.embed[tokens.long()] + self.place[positions.long()]
        for layer, (qkv, out, up, down) in enumerate(self.blocks):
            heads = (self.norm(x) @ qkv).view(n, nodes, -1, self.head_dim)
            q, k, v = heads.split([self.q_heads, self.kv_heads, self.kv_heads], 2)
            x = x + attend(layer, q, k, v).reshape(n, nodes, -1).to(x.dtype) @ out
            x = x + torch.relu(self.norm(x) @ up) @ down
        return self.norm(x) @ self.head

    def draft(self, ranks):
        """[vocab, ranks] int32: the likeliest successors of each token when nothing but the token is looked at."""
        return (self.norm(self.embed) @ self.head).topk(ranks, -1).indices.to(torch.int32)


def cached(model, cache, seqs, tokens, depths, masks=None, n_nodes=None):
    """The model's logits for nodes at `depths` past the slots' lengths; their keys and values go to the cache."""
    positions = cache.lens[seqs.long()][:, None] + depths

    def attend(layer, q, k, v):
        q, k, v = (t.to(cache.dtype) for t in (q, k, v))
        return cache.tree_attention(layer, seqs, q, k, v, masks, n_nodes=n_nodes)

    return model.forward(tokens, positions, attend)


def make_cache(model, slots, length, page=16, dtype=torch.bfloat16):
    width = -(-length // page)
    return PagedCache(model.layers, model.kv_heads, model.head_dim, page, slots * (width + 1), slots, width, dtype=dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prefill(model, cache, seqs, prompts):
    """All prompts but their last tokens, 64 tokens of each at a time; returns the last tokens [n, 1]."""
    rest = [p[:-1] for p in prompts]
    for at in range(0, max(map(len, rest)), 64):
        part = [r[at:at + 64] for r in rest]
        counts, nodes = ints([len(p) for p in part]), max(map(len, part))
        tokens = ints([p + [0] * (nodes - len(p)) for p in part])
        cache.extend(seqs, counts)
        cached(model, cache, seqs, tokens, torch.arange(nodes, device="cuda"), n_nodes=counts)
        cache.commit(seqs, counts)
    return ints([[p[-1]] for p in prompts])


def tree_decode(model, prompts, steps, temperature=0.0):
    """Continues the prompts by `steps` passes; returns a list of new tokens for each, 1 to 5 a pass."""
    n, nodes = len(prompts), len(PARENTS)
    cache = make_cache(model, n, max(map(len, prompts)) + steps * (max(DEPTHS) + 1) + nodes)
    sampler = Sampler(model.vocab, n * nodes)
    params = params_to_device(row_params(n * nodes, temperature=temperature), "cuda")
    seqs, counts = ints(range(n)), ints([nodes] * n)
    root = prefill(model, cache, seqs, prompts)
    parents, depths, draft = ints([PARENTS] * n), ints(DEPTHS), model.draft(max(RANKS) + 1)
    masks = tree_masks(parents)
    results = []
    for _ in range(steps):
        columns = [root[:, 0]]
        for up, rank in zip(PARENTS[1:], RANKS[1:]):
            columns.append(draft[columns[up].long(), rank])
        tokens = torch.stack(columns, 1)
        cache.extend(seqs, counts)
        logits = cached(model, cache, seqs, tokens, depths, masks)
        uniforms = torch.rand(n * nodes, device="cuda") if temperature > 0 else None
        ids, _ = sampler.sample(logits.view(n * nodes, -1), params, uniforms=uniforms)
        path, taken = cache.accept(seqs, parents, tokens, ids.view(n, nodes))
        root = path.gather(1, taken.long()[:, None] - 1)
        results.append((path, taken))
    out = [[] for _ in prompts]
    for path, taken in results:
        for i, (p, t) in enumerate(zip(path.tolist(), taken.tolist())):
            out[i] += p[:t]
    if cache.device_status():
        raise RuntimeError("the cache reported an error")
    return out


def beam_decode(model, prompts, steps, beams=4, eos_id=-1):
    """The `beams` best continuations by `steps` tokens: for each prompt a list of (tokens, log-probability)."""
    n, rows = len(prompts), len(prompts) * beams
    cache = make_cache(model, rows, max(map(len, prompts)) + steps)
    search = BeamSearch(model.vocab, beams, n)
    slots, one = ints(range(rows)), ints([1] * rows)
    first = slots[::beams].contiguous()
    root = prefill(model, cache, first, prompts).repeat_interleave(beams, 0)
    cache.fork(first.repeat_interleave(beams), slots)
    scores = torch.full((n, beams), float("-inf"), device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros((n, beams), dtype=torch.int32, device="cuda")
    history, history_len = torch.full((rows, steps), -1, dtype=torch.int32, device="cuda"), torch.zeros_like(slots)
    depth, base = ints([0]), first[:, None]
    for _ in range(steps):
        cache.extend(slots, one)
        logits = cached(model, cache, slots, root, depth)[:, 0]
        cache.commit(slots, one)
        _, tokens, scores, finished, history, history_len = step = search.select(
            logits, scores, finished=finished, eos_id=eos_id, history=history, history_len=history_len)
        cache.fork(torch.where(step.parents < 0, -1, base + step.parents).to(torch.int32).view(rows), slots)
        root = tokens.clamp(min=0).view(rows, 1)
    if cache.device_status() or search.device_status():
        raise RuntimeError("the cache or the search reported an error")
    found, lens, best = history.view(n, beams, steps).tolist(), history_len.view(n, beams).tolist(), scores.tolist()
    return [[(found[i][w][:lens[i][w]], best[i][w]) for w in range(beams)] for i in range(n)]


def main():
    model = ToyModel()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(model.vocab, (length,), generator=g).tolist() for length in (5, 70, 131)]
    steps = 24
    for p, new in zip(prompts, tree_decode(model, prompts, steps)):
        print(f"prompt of {len(p)}: {len(new)} tokens in {steps} passes: {new[:12]} ...")
    for p, found in zip(prompts, beam_decode(model, prompts, steps)):
        print(f"prompt of {len(p)}: best beam {found[0][1]:.3f}: {found[0][0][:12]} ...")


if __name__ == "__main__":
    main()
