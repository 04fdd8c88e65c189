"""The decoding operators on a paged key/value cache and on beams, as cases to time and to check.

Four operators, each in a plain form of elementary torch operations in 32 bits
(`own` false) and through the package's public calls (`own` true):

  tree    attention of the drafted nodes of a tree (or of one token, or of a chain) over a
          paged cache, which also stores the nodes' keys and values in the cache
  fork    beams forked from their parents (pages shared) and given room for a token each:
          the partly filled last page is copied, in every layer
  accept  a step over a drafted tree settled: the tree walked with the sampled tokens, the
          accepted path's keys and values moved together in every layer, surplus pages freed
  beam    selection over beams and vocabulary with the history's reordering

The state of a cache is: pools k, v [layers, pages, kv_heads, page_size, head_dim]; for every
sequence slot its length, its number of pages and its row of page ids (-1 past that number);
for every page the number of rows that hold it.  A call that needs pages takes the
lowest-numbered free ones, row after row.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- the cases ------------------------------------------------------------------------------

def _tree(name, batch, nodes, heads, kv_heads, dim, ctx, page, dtype, ragged):
    return {"name": name, "op": "tree", "batch": batch, "nodes": nodes, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "ctx": ctx, "page": page, "dtype": dtype, "ragged": ragged}


def _fork(name, groups, beams, ctx, layers, kv_heads, dim, page, dtype):
    return {"name": name, "op": "fork", "groups": groups, "beams": beams, "ctx": ctx, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _accept(name, batch, nodes, ctx, layers, kv_heads, dim, page, dtype):
    return {"name": name, "op": "accept", "batch": batch, "nodes": nodes, "ctx": ctx, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _beam(name, batch, beams, vocab, dtype, history, masked):
    return {"name": name, "op": "beam", "batch": batch, "beams": beams, "vocab": vocab, "dtype": dtype,
            "history": history, "masked": masked}


def listed():
    return [
        # one user's next token after a short prompt, every head with its own keys: latency
        _tree("tree 1x1 short", 1, 1, 8, 8, 64, 200, 16, "bf16", False),
        # a serving batch decoding one token per sequence, lengths of all kinds
        _tree("tree 64x1 decode", 64, 1, 32, 8, 128, 4096, 64, "bf16", True),
        # speculative verification of 5 drafted tokens and their root, 128 sequences
        _tree("tree 128x6 chain f16", 128, 6, 32, 8, 128, 1500, 32, "f16", True),
        # one long document and a wide tree: few sequences, a long axis to split
        _tree("tree 1x64 long", 1, 64, 32, 8, 128, 65536, 128, "bf16", False),
        # a full serving batch with trees: the largest call
        _tree("tree 64x16 largest", 64, 16, 32, 8, 128, 8192, 64, "bf16", True),
        # the first beams of a small model: bookkeeping latency
        _fork("fork 2x4 small", 2, 4, 77, 2, 4, 64, 16, "bf16"),
        # a beam batch over a 32-layer model: the page copies fill the memory system
        _fork("fork 16x4 32 layers", 16, 4, 2043, 32, 8, 128, 64, "bf16"),
        # one sequence's tree settled: latency
        _accept("accept 1x16", 1, 16, 301, 4, 8, 64, 16, "f16"),
        # a batch of wide trees over a 32-layer model
        _accept("accept 64x64 32 layers", 64, 64, 1023, 32, 8, 128, 64, "bf16"),
        # one user's beam search over a byte-pair vocabulary, 32-bit logits: latency
        _beam("beam 1x4 50257 f32", 1, 4, 50257, "f32", 100, False),
        # constrained beams: a grammar's mask row for every beam
        _beam("beam 16x8 128256 masked", 16, 8, 128256, "bf16", 700, True),
        # a large batch of beams: the logits' bytes bound it
        _beam("beam 64x16 128256", 64, 16, 128256, "bf16", 1024, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "fork", "accept", "beam", "beam"])
    if op == "tree":
        batch, nodes = _log(rng, 1, 128), _log(rng, 1, 64)
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        dim, page = rng.choice([64, 80, 96, 128]), rng.choice([8, 16, 32, 64, 128, 256])
        ctx = _log(rng, 1, 65536)
        # no more keys, and no more scores, than the largest listed case has
        ctx = max(1, min(ctx, 64 * 8192 * 8 * 128 // (batch * kv_heads * dim), 64 * 32 * 16 * 8192 // (batch * kv_heads * group * nodes)))
        return {k: v for k, v in _tree("", batch, nodes, kv_heads * group, kv_heads, dim, ctx, page, rng.choice(["bf16", "f16"]), rng.random() < 0.7).items() if k != "name"}
    if op in ("fork", "accept"):
        layers, kv_heads = _log(rng, 1, 32), rng.choice([1, 2, 4, 8])
        dim, page = rng.choice([64, 80, 96, 128]), rng.choice([8, 16, 32, 64, 128])
        ctx = _log(rng, 2, 2043)
        if op == "fork":
            c = _fork("", _log(rng, 1, 16), rng.randint(1, 4), ctx, layers, kv_heads, dim, page, rng.choice(["bf16", "f16"]))
        else:
            c = _accept("", _log(rng, 1, 64), _log(rng, 2, 64), min(ctx, 1023), layers, kv_heads, dim, page, rng.choice(["bf16", "f16"]))
        return {k: v for k, v in c.items() if k != "name"}
    beams, dtype = _log(rng, 1, 16), rng.choice(["bf16", "f32"])
    vocab = _log(rng, 500, 131072)
    most = 64 * 16 * 128256 // (2 if dtype == "f32" else 1)
    batch = max(1, min(_log(rng, 1, 64), most // (beams * vocab)))
    return {k: v for k, v in _beam("", batch, beams, vocab, dtype, _log(rng, 1, 1024), rng.random() < 0.4).items() if k != "name"}


# ---- shapes that follow from a case alone -----------------------------------------------------

def _lens(case):
    """Tokens in the cache, by sequence."""
    n = case["batch"] if "batch" in case else case["groups"]
    i = np.arange(n, dtype=np.int64)
    if case["op"] == "tree" and not case["ragged"]:
        return np.full(n, case["ctx"], np.int64)
    # between a fifth of the context and all of it (the first has all), in no order
    low = case["ctx"] // 5
    return np.maximum(1, case["ctx"] - (i * 7919) % max(1, case["ctx"] - low))


def _nodes(case):
    """Nodes of each sequence's tree."""
    i = np.arange(case["batch"], dtype=np.int64)
    if case["op"] == "tree" and not case["ragged"]:
        return np.full(case["batch"], case["nodes"], np.int64)
    return case["nodes"] - (i * 5) % max(1, case["nodes"] // 2)


def _shape(case):
    """Each sequence's tree: parents [batch, nodes] (a parent comes before its child, -1 at the root and past the
    tree's end), and the path that will be accepted, as a truth value for each node."""
    r = random.Random(case["nodes"] * 1009 + case["batch"])
    n, N = _nodes(case), case["nodes"]
    parents = np.full((case["batch"], N), -1, np.int32)
    kept = np.zeros((case["batch"], N), bool)
    for b in range(case["batch"]):
        for i in range(1, int(n[b])):
            parents[b, i] = r.randint(max(0, i - 6), i - 1)
        at = 0
        kept[b, 0] = True
        for _ in range(r.randint(0, 8)):
            below = np.flatnonzero(parents[b] == at)
            if not len(below):
                break
            at = int(below[r.randrange(len(below))])
            kept[b, at] = True
    return parents, kept


def _ancestors(parents, n):
    """[batch, nodes] 64-bit sets: bit j of node i says that node i sees node j (its ancestors and itself)."""
    B, N = parents.shape
    bits = np.zeros((B, N), np.uint64)
    for i in range(N):
        p = parents[:, i]
        up = np.where(p >= 0, bits[np.arange(B), np.maximum(p, 0)], np.uint64(0))
        bits[:, i] = np.where(i < n, up | (np.uint64(1) << np.uint64(i)), np.uint64(0))
    return bits.view(np.int64)


def _up(a, b):
    return -(-a // b)


def work(case):
    op = case["op"]
    if op == "beam":
        rows, es = case["batch"] * case["beams"], 4 if case["dtype"] == "f32" else 2
        masks = rows * _up(case["vocab"], 32) * 4 if case["masked"] else 0
        return {"bytes": rows * (case["vocab"] * es + 8 * case["history"] + 40) + masks, "flops": 4 * rows * case["vocab"]}
    token = 2 * case["kv_heads"] * case["dim"] * 2  # a token's keys and values in one layer
    lens = _lens(case)
    if op == "tree":
        n, G = _nodes(case), case["heads"] // case["kv_heads"]
        seen = int((lens * n).sum() + (n * n).sum())
        io = int(n.sum()) * (2 * token + case["heads"] * (4 * case["dim"] + 4) + 8)
        return {"bytes": int(lens.sum()) * token + io + int(_up(lens, case["page"]).sum()) * 4, "flops": 4 * seen * G * case["kv_heads"] * case["dim"]}
    if op == "fork":
        part = int((lens % case["page"]).sum()) * case["beams"]
        rows = int(_up(lens, case["page"]).sum()) * case["beams"]
        return {"bytes": 2 * part * token * case["layers"] + 16 * rows, "flops": 0}
    parents, kept = _shape(case)
    moved = sum(int((np.flatnonzero(k) != np.arange(int(k.sum()))).sum()) for k in kept)
    return {"bytes": 2 * moved * token * case["layers"] + 16 * parents.size, "flops": 0}


# ---- inputs -------------------------------------------------------------------------------------

def _randn(g, shape, dtype, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


class _Plain:
    """A cache's state as torch tensors."""

    def __init__(self, case, layers, pages, slots, width):
        shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
        self.page = case["page"]
        self.k = torch.empty(shape, dtype=TYPES[case["dtype"]], device="cuda")
        self.v = torch.empty_like(self.k)
        self.lens = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.counts = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.tables = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")

    def extend(self, seqs, more):
        """Pages for `more` tokens past each row's length; a shared page that they would be written to is copied."""
        ps, pages, s = self.page, self.refs.numel(), seqs.long()
        rows = torch.arange(len(s), device="cuda")
        length, have = self.lens[s].long(), self.counts[s].long()
        need = ((length + more + ps - 1) // ps - have).clamp(min=0)
        at = (length // ps).clamp(max=self.tables.shape[1] - 1)
        last = self.tables[s, at].long()
        partly = (length % ps != 0) & (more > 0) & (last >= 0)
        last = torch.where(partly, last, torch.full_like(last, pages))  # one page more, for the rows without
        refs = torch.cat([self.refs.long(), self.refs.new_zeros(1).long()])
        calls = torch.zeros(pages + 1, dtype=torch.long, device="cuda").index_add_(0, last, torch.ones_like(last))
        first = torch.full((pages + 1,), len(s), dtype=torch.long, device="cuda").scatter_reduce_(0, last, rows, "amin")
        stays = (refs[last] == 1) | ((calls[last] == refs[last]) & (first[last] == rows))
        copy = partly & ~stays
        takes = need + copy
        start = takes.cumsum(0) - takes
        free = torch.sort((self.refs != 0).to(torch.int8), stable=True).indices
        # the copies, each to its row's first page; rows without one do the first copy once more
        fresh = free[start.clamp(max=pages - 1)]
        as_row = torch.where(copy, rows, copy.int().argmax())
        src, dst = torch.where(copy, last, fresh)[as_row], fresh[as_row]
        self.k[:, dst] = self._part(self.k, src, dst, copy[as_row], (length % ps)[as_row])
        self.v[:, dst] = self._part(self.v, src, dst, copy[as_row], (length % ps)[as_row])
        slot = torch.arange(self.tables.shape[1], device="cuda")[None]
        new = (slot >= have[:, None]) & (slot < (have + need)[:, None])
        which = (start + copy)[:, None] + slot - have[:, None]
        table = torch.where(new, free[which.clamp(0, pages - 1)], self.tables[s].long())
        table = torch.where(copy[:, None] & (slot == at[:, None]), fresh[:, None], table)
        gone = torch.where(copy, last, torch.full_like(last, pages))
        refs.index_add_(0, gone, -torch.ones_like(gone))
        got = torch.arange(pages, device="cuda") < takes.sum()
        refs.index_add_(0, free, got.long())
        self.refs.copy_(refs[:pages])
        self.tables[s] = table.int()
        self.counts[s] = (have + need).int()

    @staticmethod
    def _part(pool, src, dst, copy, n):
        """The pages as they are after the copy of the first n tokens."""
        t = torch.arange(pool.shape[3], device="cuda")
        some = (copy[:, None] & (t < n[:, None]))[None, :, None, :, None]
        return torch.where(some, pool[:, src], pool[:, dst])

    def fork(self, src, dst):
        """dst's rows become src's."""
        s, d, pages = src.long(), dst.long(), self.refs.numel()
        slot = torch.arange(self.tables.shape[1], device="cuda")[None]
        keep = (self.lens[s].long() + self.page - 1) // self.page
        new = torch.where(slot < keep[:, None], self.tables[s], torch.full_like(self.tables[s], -1))
        refs = torch.cat([self.refs, self.refs.new_zeros(1)])
        for_all = torch.where(new >= 0, new, torch.full_like(new, pages)).long().reshape(-1)
        old = self.tables[d]
        of_old = torch.where(old >= 0, old, torch.full_like(old, pages)).long().reshape(-1)
        refs.index_add_(0, for_all, torch.ones_like(for_all, dtype=torch.int32))
        refs.index_add_(0, of_old, -torch.ones_like(of_old, dtype=torch.int32))
        self.refs.copy_(refs[:pages])
        lens = self.lens[s]
        self.tables[d], self.counts[d], self.lens[d] = new, keep.int(), lens

    def cut(self, seqs, lens):
        """Lengths set back, pages past them released."""
        s, pages = seqs.long(), self.refs.numel()
        keep = (lens.long() + self.page - 1) // self.page
        slot = torch.arange(self.tables.shape[1], device="cuda")[None]
        table = self.tables[s]
        gone = torch.where((slot >= keep[:, None]) & (table >= 0), table, torch.full_like(table, pages)).long().reshape(-1)
        refs = torch.cat([self.refs, self.refs.new_zeros(1)]).index_add_(0, gone, -torch.ones_like(gone, dtype=torch.int32))
        self.refs.copy_(refs[:pages])
        self.tables[s] = torch.where(slot < keep[:, None], table, torch.full_like(table, -1))
        self.counts[s] = torch.minimum(self.counts[s], keep.int())
        self.lens[s] = lens


def _cache(case, layers, pages, slots, width, lens, g):
    """A cache that holds sequences 0.. of these lengths, their pages not in one piece: grown in two steps."""
    seqs = torch.arange(len(lens), device="cuda", dtype=torch.int32)
    first, rest = _i32(lens // 2), _i32(lens - lens // 2)
    if own:
        from tinygpt_b200 import PagedCache
        c = PagedCache(layers, case["kv_heads"], case["dim"], case["page"], pages, slots, width, dtype=TYPES[case["dtype"]])
        for n in (first, rest):
            c.extend(seqs, n)
            c.commit(seqs, n)
    else:
        c = _Plain(case, layers, pages, slots, width)
        for n in (first, rest):
            c.extend(seqs, n.long())
            c.lens[: len(lens)] += n
    # what the earlier steps stored: values as projections give them
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    return c


def _real(n, N):
    """The nodes that are there: their rows, and their places in them."""
    row, node = np.nonzero(np.arange(N)[None] < n[:, None])
    return {"row": torch.from_numpy(row).cuda(), "node": torch.from_numpy(node).cuda()}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _PREPARE[case["op"]](case, seed, g)


def _prepare_tree(case, seed, g):
    B, N, D, Hq, Hkv = case["batch"], case["nodes"], case["dim"], case["heads"], case["kv_heads"]
    lens, n = _lens(case), _nodes(case)
    width = int(_up(lens + N, case["page"]).max())
    pages = int(_up(lens + n, case["page"]).sum()) + 1
    c = _cache(case, 1, pages, B, width, lens, g)
    seqs, n_nodes = torch.arange(B, device="cuda", dtype=torch.int32), _i32(n)
    c.extend(seqs, n_nodes if own else n_nodes.long())
    # the projections' output, queries, keys and values of a node side by side
    qkv = _randn(g, (B, N, Hq + 2 * Hkv, D), TYPES[case["dtype"]])
    return {"op": "tree", "cache": c, "seqs": seqs, "n": n_nodes, "q": qkv[:, :, :Hq].mul_(1.5), "k": qkv[:, :, Hq:Hq + Hkv], "v": qkv[:, :, Hq + Hkv:],
            "masks": torch.from_numpy(_ancestors(_shape(case)[0], n)).cuda(), "pages": int(_up(lens, case["page"]).max()), **_real(n, N)}


def _prepare_fork(case, seed, g):
    lens = _lens(case)
    G, W = case["groups"], case["beams"]
    width = int(_up(lens + 1, case["page"]).max())
    pages = int(_up(lens, case["page"]).sum()) + 2 * G * W
    c = _cache(case, case["layers"], pages, G * (1 + W), width, lens, g)
    ids = torch.arange(G * W, device="cuda", dtype=torch.int32)
    return {"op": "fork", "cache": c, "src": ids // W, "dst": ids + G, "one": torch.ones(G * W, dtype=torch.int32, device="cuda")}


def _prepare_accept(case, seed, g):
    B, N = case["batch"], case["nodes"]
    lens, n = _lens(case), _nodes(case)
    width = int(_up(lens + N, case["page"]).max())
    pages = int(_up(lens + N, case["page"]).sum())
    c = _cache(case, case["layers"], pages, B, width, lens, g)
    parents, kept = _shape(case)
    r = np.random.default_rng(seed)
    tokens = r.integers(0, 32000, (B, N)).astype(np.int32)
    ids = (tokens[:, ::-1] + 40000).copy()  # tokens that no draft holds, but along the path that is accepted
    rows, at = np.nonzero(kept & (parents >= 0))
    ids[rows, parents[rows, at]] = tokens[rows, at]
    return {"op": "accept", "cache": c, "seqs": torch.arange(B, device="cuda", dtype=torch.int32), "lens": _i32(lens), "n": _i32(n), "parents": _i32(parents),
            "tokens": _i32(tokens), "ids": _i32(ids), **_real(n, N)}


def _prepare_beam(case, seed, g):
    B, W, V = case["batch"], case["beams"], case["vocab"]
    logits = torch.randn((B * W, V), generator=g, device="cuda").mul_(3.0).to(TYPES[case["dtype"]])
    scores = -torch.rand((B, W), generator=g, device="cuda") * 20
    finished = torch.rand((B, W), generator=g, device="cuda") < 0.1
    s = {"op": "beam", "logits": logits, "scores": scores, "finished": finished.int(), "eos": 2 % V, "pad": 0, "table": None, "state": None,
         "history": torch.randint(0, V, (B * W, case["history"] + 1), generator=g, device="cuda", dtype=torch.int32),
         "length": torch.full((B * W,), case["history"], dtype=torch.int32, device="cuda")}
    if case["masked"]:
        words = torch.randint(-2**31, 2**31, (64, _up(V, 32)), generator=g, device="cuda", dtype=torch.int64)
        s["table"] = (words & torch.randint(-2**31, 2**31, words.shape, generator=g, device="cuda", dtype=torch.int64)).int()
        s["state"] = torch.randint(-1, 64, (B * W,), generator=g, device="cuda", dtype=torch.int32)
    if own:
        from tinygpt_b200 import BeamSearch
        s["search"] = BeamSearch(V, W, B)
    return s


# ---- one pass -------------------------------------------------------------------------------------

def run(state):
    return (_OWN if own else _RUN)[state["op"]](state)


def _own_tree(s):
    c = s["cache"]
    out, lse = c.tree_attention(0, s["seqs"], s["q"], s["k"], s["v"], s["masks"], n_nodes=s["n"], want_lse=True)
    return {"out": out, "lse": lse, "k": c.k, "v": c.v}


def _own_fork(s):
    c = s["cache"]
    c.fork(s["src"], s["dst"])
    c.extend(s["dst"], s["one"])
    return {"lens": c.lens, "counts": c.counts, "tables": c.tables, "refs": c.refs, "k": c.k, "v": c.v}


def _own_accept(s):
    c = s["cache"]
    c.truncate(s["seqs"], s["lens"])  # the step starts from where the one before it ended
    c.extend(s["seqs"], s["n"])
    ids, count = c.accept(s["seqs"], s["parents"], s["tokens"], s["ids"], n_nodes=s["n"])
    return {"ids": ids, "count": count, "lens": c.lens, "counts": c.counts, "tables": c.tables, "refs": c.refs, "k": c.k, "v": c.v}


def _own_beam(s):
    r = s["search"].select(s["logits"], s["scores"], finished=s["finished"], eos_id=s["eos"], pad_id=s["pad"], mask_table=s["table"], state_id=s["state"],
                           history=s["history"], history_len=s["length"])
    return {"parents": r.parents, "tokens": r.tokens, "scores": r.scores, "finished": r.finished, "history": r.history, "length": r.history_len}


def _run_tree(s):
    c, n = s["cache"], s["n"].long()
    B, N, Hq, D = s["q"].shape
    Hkv, ps = s["k"].shape[2], c.page
    lens = c.lens[s["seqs"].long()].long()
    node = torch.arange(N, device="cuda")
    real = node[None] < n[:, None]
    # the nodes' keys and values go to their places in the cache
    place = lens[:, None] + node[None]
    page = c.tables[s["seqs"].long()].long().gather(1, (place // ps).clamp(max=c.tables.shape[1] - 1))
    b, i = s["row"], s["node"]
    c.k[0, page[b, i], :, place[b, i] % ps] = s["k"][b, i]
    c.v[0, page[b, i], :, place[b, i] % ps] = s["v"][b, i]
    table = c.tables[s["seqs"].long(), : s["pages"]].long().clamp(min=0)
    keys = c.k[0, table].transpose(2, 3).reshape(B, -1, Hkv, D).float()
    values = c.v[0, table].transpose(2, 3).reshape(B, -1, Hkv, D).float()
    q = s["q"].float().reshape(B, N, Hkv, Hq // Hkv, D)
    past = torch.arange(keys.shape[1], device="cuda")[None] < lens[:, None]
    sees = ((s["masks"][:, :, None] >> node) & 1).bool() & real[:, None, :] & real[:, :, None]
    low = float("-inf")
    sc = 1.0 / math.sqrt(D)
    a = torch.where((past[:, None] & real[:, :, None])[:, :, None, None, :], torch.einsum("bnkgd,btkd->bnkgt", q, keys) * sc, low)
    t = torch.where(sees[:, :, None, None, :], torch.einsum("bnkgd,btkd->bnkgt", q, s["k"].float()) * sc, low)
    top = torch.maximum(a.amax(-1), t.amax(-1))
    base = torch.where(top == low, torch.zeros_like(top), top)[..., None]
    a, t = torch.exp(a - base), torch.exp(t - base)
    total = a.sum(-1) + t.sum(-1)
    out = torch.einsum("bnkgt,btkd->bnkgd", a, values) + torch.einsum("bnkgt,btkd->bnkgd", t, torch.where(real[:, :, None, None], s["v"].float(), 0.0))
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    return {"out": out.reshape(B, N, Hq, D).to(s["q"].dtype), "lse": (base[..., 0] + torch.log(total)).reshape(B, N, Hq), "k": c.k, "v": c.v}


def _run_fork(s):
    c = s["cache"]
    c.fork(s["src"], s["dst"])
    c.extend(s["dst"], s["one"].long())
    return {"lens": c.lens, "counts": c.counts, "tables": c.tables, "refs": c.refs, "k": c.k, "v": c.v}


def _run_accept(s):
    c, q, ps = s["cache"], s["seqs"].long(), s["cache"].page
    c.cut(s["seqs"], s["lens"])
    c.extend(s["seqs"], s["n"].long())
    B, N = s["parents"].shape
    node = torch.arange(N, device="cuda")
    above = s["parents"].long().clamp(min=0)
    real = (node[None] < s["n"][:, None]) & (node[None] > 0) & (s["parents"] >= 0)
    hit = real & (s["tokens"] == s["ids"].gather(1, above))
    # of siblings with the same token the first counts
    twin = (above[:, :, None] == above[:, None, :]) & hit[:, :, None] & hit[:, None, :] & (node[None, :] < node[:, None])
    hit = hit & ~twin.any(-1)
    # a node is accepted when it and all its ancestors are hits: the ancestors by squaring "is i or its parent"
    up = ((above[:, :, None] == node) & real[:, :, None] | (node[:, None] == node)).float()
    up = (up @ up).clamp(max=1)
    up = (up @ up).clamp(max=1)
    up = (up @ up).clamp(max=1)
    up = (up @ up).clamp(max=1)
    up = (up @ up).clamp(max=1)
    up = (up @ up).clamp(max=1)
    good = hit | (node[None] == 0)
    taken = good & ~((up > 0) & ~good[:, None, :]).any(-1)
    count = taken.sum(1)
    path = torch.sort((~taken).to(torch.int8), dim=1, stable=True).indices
    kept = node[None] < count[:, None]
    out = torch.where(kept, s["ids"].gather(1, path), -1).int()
    # the path's keys and values move together; the other places stay
    frm = s["lens"].long()[:, None] + torch.where(kept, path, node[None])
    to = s["lens"].long()[:, None] + node[None]
    row, i = s["row"], s["node"]
    table = c.tables[q].long()
    frm, to = frm[row, i], to[row, i]
    p, r = table[row, frm // ps], table[row, to // ps]
    c.k[:, r, :, to % ps] = c.k[:, p, :, frm % ps]
    c.v[:, r, :, to % ps] = c.v[:, p, :, frm % ps]
    lens = s["lens"] + count.int()
    c.cut(s["seqs"], lens)
    return {"ids": out, "count": count.int(), "lens": c.lens, "counts": c.counts, "tables": c.tables, "refs": c.refs, "k": c.k, "v": c.v}


def _run_beam(s):
    B, W = s["scores"].shape
    x = s["logits"].float()
    V = x.shape[1]
    token = torch.arange(V, device="cuda")
    low = float("-inf")
    if s["table"] is not None:
        bit = (s["table"][s["state"].long().clamp(min=0)][:, token // 32] >> (token % 32).int()) & 1
        x = torch.where((bit == 1) | (s["state"] < 0)[:, None], x, low)
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = (x - lse).reshape(B, W, V) + s["scores"][:, :, None]
    # a finished beam goes on as it is, once
    stay = torch.where(token == s["pad"], s["scores"][:, :, None], low)
    score = torch.where((s["finished"] != 0)[:, :, None], stay, score).reshape(B, W * V)
    best, at = torch.sort(score, dim=1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    there = best > low
    parent, tok = torch.where(there, at // V, -1).int(), torch.where(there, at % V, -1).int()
    was = s["finished"].gather(1, parent.long().clamp(min=0)) != 0
    done = (was | (tok == s["eos"]) | ~there).int()
    row = (torch.arange(B, device="cuda")[:, None] * W + parent.long().clamp(min=0)).reshape(-1)
    grow = (there & ~was).reshape(-1) & (s["length"][row] < s["history"].shape[1])
    length = torch.where(there.reshape(-1), s["length"][row], 0)
    place = torch.arange(s["history"].shape[1], device="cuda", dtype=torch.int32)[None]
    history = torch.where(place < length[:, None], s["history"][row], -1)
    history = torch.where((place == length[:, None]) & grow[:, None], tok.reshape(-1, 1), history)
    return {"parents": parent, "tokens": tok, "scores": best, "finished": done, "history": history, "length": length + grow.int()}


# ---- the definition in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    """In 64 bits, sequence by sequence.  None: whole numbers, and bits that are only moved."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _EXACT[case["op"]](case, s)


def _exact_tree(case, s):
    c = s["cache"]
    B, N, Hq, D = s["q"].shape
    G = Hq // s["k"].shape[2]
    lens, n = _lens(case), _nodes(case)
    out = torch.zeros((B, N, Hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, N, Hq), float("-inf"), dtype=torch.float64, device="cuda")
    j = torch.arange(N, device="cuda")
    for b in range(B):
        L, m = int(lens[b]), int(n[b])
        t = torch.arange(L, device="cuda")
        page, slot = c.tables[b].long()[t // case["page"]], t % case["page"]
        k = torch.cat([c.k[0, page, :, slot], s["k"][b, :m]]).double().permute(1, 0, 2)
        v = torch.cat([c.v[0, page, :, slot], s["v"][b, :m]]).double().permute(1, 0, 2)
        q = s["q"][b, :m].double().permute(1, 0, 2)
        sees = torch.cat([torch.ones((m, L), dtype=torch.bool, device="cuda"), ((s["masks"][b, :m, None] >> j[:m]) & 1).bool()], 1)
        for h in range(Hq):
            z = (q[h] @ k[h // G].T / math.sqrt(D)).masked_fill(~sees, float("-inf"))
            lse[b, :m, h] = torch.logsumexp(z, 1)
            out[b, :m, h] = torch.softmax(z, 1) @ v[h // G]
    return {"out": out, "lse": lse, "k": None, "v": None}


def _exact_beam(case, s):
    B, W = s["scores"].shape
    V = s["logits"].shape[1]
    x = s["logits"].double()
    if s["table"] is not None:
        bits = np.unpackbits(s["table"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
        state = s["state"].cpu().numpy()
        allowed = torch.from_numpy(bits[np.maximum(state, 0)] | (state < 0)[:, None]).cuda()
        x = x.masked_fill(~allowed, float("-inf"))
    z = torch.log_softmax(x, 1).view(B, W, V) + s["scores"].double()[:, :, None]
    f = s["finished"].bool()
    z[f] = float("-inf")
    z[..., s["pad"]] = torch.where(f, s["scores"].double(), z[..., s["pad"]])
    return {"parents": None, "tokens": None, "scores": torch.topk(z.view(B, W * V), W, dim=1).values, "finished": None, "history": None, "length": None}


_PREPARE = {"tree": _prepare_tree, "fork": _prepare_fork, "accept": _prepare_accept, "beam": _prepare_beam}
_OWN = {"tree": _own_tree, "fork": _own_fork, "accept": _own_accept, "beam": _own_beam}
_RUN = {"tree": _run_tree, "fork": _run_fork, "accept": _run_accept, "beam": _run_beam}
_EXACT = {"tree": _exact_tree, "fork": lambda case, s: None, "accept": lambda case, s: None, "beam": _exact_beam}
