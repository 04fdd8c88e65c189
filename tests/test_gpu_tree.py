"""Tree attention over the paged cache against its definition in 64 bits.

Tolerance of an output element, from the arithmetic: the weights are rounded to the
cache's type for the product with the values (relative u = 2^-8 for bf16, 2^-11 for
f16: half a unit in the last of 8 and 11 significant bits), the output once more; a
score is a sum of head_dim products in fp32, off by at most (head_dim + 2) 2^-23 of the
sum of their sizes, which moves a weight by as much, relative, twice (numerator and
sum); exponentials and the running rescales add 2^-18.  An f16 weight below 2^-14 of
its row's largest is rounded to 2^-25 of it instead.
"""
import ctypes

import numpy as np
import pytest

from tests.decode_reference import tree_reference
from tinygpt_b200 import _lib

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def tree(r, n, nodes):
    """Random parents and the ancestor sets, as Python integers."""
    parents = np.array([[-1] + [int(r.integers(max(0, j - 4), j)) for j in range(1, nodes)] for _ in range(n)])
    masks = []
    for b in range(n):
        m = []
        for i in range(nodes):
            m.append((1 << i) | (m[parents[b, i]] if i else 0))
        masks.append(m)
    return masks


def as_tensor(masks):
    import torch
    return torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64).reshape(len(masks), -1)).cuda()


class Case:
    def __init__(self, lens, nodes, heads, kv_heads, dim, page, dtype="bf16", layers=1, layer=0, seed=0, spare=3, n_nodes=None, std=1.5):
        import torch
        from tinygpt_b200 import PagedCache
        self.r = np.random.default_rng(seed)
        torch.manual_seed(seed)
        dt = torch.bfloat16 if dtype == "bf16" else torch.float16
        lens = np.array(lens)
        n = len(lens)
        width = int((-(-(lens + nodes) // page)).max()) + 1
        pages = int((-(-(lens + nodes) // page)).sum()) + spare
        self.c = c = PagedCache(layers, kv_heads, dim, page, pages, n + 2, width, dtype=dt)
        c.k.fill_(float("nan"))  # what no token was stored in
        c.v.fill_(float("inf"))
        self.seqs = dev(self.r.permutation(n + 2)[:n])
        self.lens, self.layer, self.nodes = lens, layer, nodes
        # grown in pieces, so that a sequence's pages are scattered
        left = lens.copy()
        while left.any():
            step = np.minimum(left, self.r.integers(0, max(2, int(lens.max()) // 2 + 1), n))
            c.extend(self.seqs, dev(step))
            c.commit(self.seqs, dev(step))
            left -= step
        for b in range(n):
            L = int(lens[b])
            t = torch.arange(L)
            page_ids = c.tables[int(self.seqs[b])].cpu().long()[t // page].cuda()
            c.k[layer, page_ids, :, (t % page).cuda()] = torch.randn(L, kv_heads, dim, device="cuda").to(dt)
            c.v[layer, page_ids, :, (t % page).cuda()] = torch.randn(L, kv_heads, dim, device="cuda").to(dt)
        self.n_nodes = np.full(n, nodes) if n_nodes is None else np.array(n_nodes)
        c.extend(self.seqs, dev(self.n_nodes))
        assert c.device_status() == 0
        qkv = torch.randn(n, nodes, heads + 2 * kv_heads, dim, device="cuda")
        qkv[:, :, :heads] *= std
        qkv = qkv.to(dt)
        self.q, self.k, self.v = qkv[:, :, :heads], qkv[:, :, heads:heads + kv_heads], qkv[:, :, heads + kv_heads:]
        self.masks = tree(self.r, n, nodes)
        self.scale = dim ** -0.5

    def run(self, masks="own", scale=None, n_nodes="own", **kw):
        m = as_tensor(self.masks) if isinstance(masks, str) else masks
        nn = dev(self.n_nodes) if isinstance(n_nodes, str) else n_nodes
        return self.c.tree_attention(self.layer, self.seqs, self.q, self.k, self.v, m, n_nodes=nn, scale=scale, want_lse=True, **kw)

    def expect(self, out, lse, scale=None):
        import torch
        scale = self.scale if scale is None else scale
        want, want_lse, weight, spread, peak = tree_reference(self.c, self.layer, self.seqs.cpu(), self.lens, self.q, self.k, self.v,
                                                              self.masks, self.n_nodes, scale)
        f16 = self.c.dtype == torch.float16
        u = 2.0 ** -11 if f16 else 2.0 ** -8
        move = (self.c.head_dim + 2) * 2.0 ** -23 * spread + 2.0 ** -18
        tol = u * (want.abs() + 1.01 * weight) + 2 * move[..., None] * weight
        if f16:  # small weights, and a small output
            vmax = max(t.float().nan_to_num(0.0, 0.0, 0.0).abs().max().item() for t in (self.c.v[self.layer], self.v))
            tol += (int(self.lens.max()) + self.nodes) * 2.0 ** -25 * vmax * peak[..., None] + 2.0 ** -24
        got = out.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
        err = (got - want).abs()
        assert (err[fine] <= tol[fine]).all(), (err - tol)[fine].max()
        g = lse.double().cpu()
        f = torch.isfinite(want_lse)
        assert torch.equal(torch.isfinite(g), f)
        assert ((g - want_lse)[f].abs() <= (move + 2.0 ** -20 * want_lse.abs().clamp(min=1))[f]).all()
        return want

    def stored(self):
        """The nodes' keys and values are in the cache, and nothing else has changed."""
        import torch
        ps = self.c.page_size
        for b in range(len(self.lens)):
            m = int(self.n_nodes[b])
            t = torch.arange(int(self.lens[b]), int(self.lens[b]) + m)
            page = self.c.tables[int(self.seqs[b])].cpu().long()[t // ps].cuda()
            assert torch.equal(self.c.k[self.layer, page, :, (t % ps).cuda()], self.k[b, :m])
            assert torch.equal(self.c.v[self.layer, page, :, (t % ps).cuda()], self.v[b, :m])
        assert int((~torch.isnan(self.c.k)).sum()) == int((self.lens + self.n_nodes).sum()) * self.c.kv_heads * self.c.head_dim


def go(**kw):
    case = Case(**kw)
    out, lse = case.run()
    case.expect(out, lse)
    case.stored()
    assert case.c.device_status() == 0
    return case


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 72, 80, 96, 120, 128])
def test_head_dims(cuda_lib, dim, dtype):
    go(lens=[0, 1, 130, 300], nodes=5, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages(cuda_lib, page, dim):
    """Pages that end inside a tile, tiles that end inside a page, lengths around both."""
    go(lens=[0, 1, page - 1, page, page + 1, 127, 128, 129, 255, 256, 257, 384, 520], nodes=3, heads=2, kv_heads=1, dim=dim, page=page)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (3, 1), (10, 2), (32, 8), (16, 1), (20, 4), (71, 1)])
@pytest.mark.parametrize("nodes", [1, 7, 64])
def test_head_layouts(cuda_lib, heads, kv_heads, nodes):
    """From one row per key head to 71 heads x 64 nodes on one key head."""
    go(lens=[77, 200], nodes=nodes, heads=heads, kv_heads=kv_heads, dim=64, page=32, dtype="f16")


@pytest.mark.parametrize("nodes", [1, 2, 8, 16, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_node_counts(cuda_lib, nodes, dtype):
    go(lens=[5, 190], nodes=nodes, heads=8, kv_heads=2, dim=128, page=64, dtype=dtype)


@pytest.mark.parametrize("heads,nodes", [(4, 1), (4, 32), (8, 64)])
def test_long_context(cuda_lib, heads, nodes):
    """A long axis over many blocks, joined again; and beside it short rows."""
    go(lens=[20011, 3, 0, 9000], nodes=nodes, heads=heads, kv_heads=1, dim=128, page=128)


def test_many_short_rows(cuda_lib):
    r = np.random.default_rng(3)
    go(lens=r.integers(0, 60, 150), nodes=4, heads=4, kv_heads=2, dim=64, page=16, dtype="f16")


def test_ragged_trees(cuda_lib):
    """Rows of 0 nodes to all, and what lies past a row's nodes is never read."""
    import torch
    case = Case(lens=[9, 0, 150, 40, 33], nodes=20, heads=6, kv_heads=2, dim=80, page=16, n_nodes=[0, 20, 1, 13, 7])
    for b, m in enumerate(case.n_nodes):
        for t in (case.q, case.k, case.v):
            t[b, m:] = float("nan")
    out, lse = case.run()
    case.expect(out, lse)
    case.stored()
    for b, m in enumerate(case.n_nodes):
        assert (out[b, m:] == 0).all() and (lse[b, m:] == -float("inf")).all()
    assert torch.isfinite(out).all()


def test_chain_without_masks(cuda_lib):
    case = Case(lens=[50, 129], nodes=64, heads=4, kv_heads=2, dim=64, page=16)
    case.masks = [[(2 << i) - 1 for i in range(64)] for _ in range(2)]
    out, lse = case.run(masks=None)
    case.expect(out, lse)
    whole, _ = case.run()
    assert (whole == out).all()


def test_rows_that_see_nothing(cuda_lib):
    """An empty cache and an empty mask: output 0, lse -inf; bits past the nodes are ignored."""
    case = Case(lens=[0, 0, 140], nodes=6, heads=4, kv_heads=2, dim=64, page=16, n_nodes=[6, 4, 6])
    case.masks[0] = [0, 1, 0, 8, 63, 0]
    case.masks[1] = [0, 0, 3, 15, 0, 0]
    case.masks[2] = [0, 0, 0, 0, 0, 1]
    wide = [[x | (0xFFFF << 40) for x in m] for m in case.masks]
    out, lse = case.run(masks=as_tensor(wide))
    case.expect(out, lse)
    assert (out[0, 0] == 0).all() and (lse[0, 2] == -float("inf")).all()


def test_infinities_and_nan_where_unseen(cuda_lib):
    """A node's NaN or infinity reaches the nodes that see it, no others."""
    import torch
    case = Case(lens=[100, 0], nodes=8, heads=4, kv_heads=1, dim=64, page=16)
    case.masks = [[1, 3, 5, 9, 17, 35, 67, 131]] * 2  # 5, 6 and 7 hang on 1
    case.v[:, 2, 0, 5] = float("inf")
    case.v[:, 3, 0, 63] = float("nan")
    case.v[:, 4, 0, 0] = -float("inf")
    case.k[:, 2] = float("nan")  # node 2's own score is NaN: so is its whole output
    out, lse = case.run()
    for b in range(2):
        for i in (0, 1, 5, 6, 7):
            assert torch.isfinite(out[b, i]).all() and torch.isfinite(lse[b, i]).all()
        assert torch.isnan(out[b, 2]).all()
        bad = ~torch.isfinite(out[b, 3])
        assert bad[:, 63].all() and bad.sum() == 4 and torch.isnan(out[b, 3, :, 63]).all()
        assert (out[b, 4, :, 0] == -float("inf")).all() and torch.isfinite(out[b, 4, :, 1:]).all()
    case.k[:, 2] = 0.5
    case.v[:, 2, 0, 5] = case.v[:, 3, 0, 63] = case.v[:, 4, 0, 0] = 0.25
    out2, _ = case.run()
    for i in (0, 1, 5, 6, 7):
        assert torch.equal(out[:, i], out2[:, i])


def test_large_scores(cuda_lib):
    """Scores of hundreds: one weight takes all, maxima move in every tile."""
    case = Case(lens=[700, 1500], nodes=9, heads=4, kv_heads=2, dim=128, page=64, std=40.0)
    out, lse = case.run()
    case.expect(out, lse)
    case = Case(lens=[700], nodes=9, heads=4, kv_heads=2, dim=128, page=64, dtype="f16")
    for scale in (-0.7, 0.0, 3.0):
        out, lse = case.run(scale=scale)
        case.expect(out, lse, scale=scale)


def test_rising_scores(cuda_lib):
    """Keys that grow along the sequence: the running maximum rises by a little, or a lot, tile after tile."""
    import torch
    for rate in (0.002, 0.02):
        case = Case(lens=[2000], nodes=4, heads=4, kv_heads=1, dim=64, page=64)
        t = torch.arange(2000)
        page = case.c.tables[int(case.seqs[0])].cpu().long()[t // 64].cuda()
        ramp = (t.float() * rate).cuda().to(torch.bfloat16)
        case.c.k[0, page, :, (t % 64).cuda()] = ramp[:, None, None].expand(2000, 1, 64)
        case.q.abs_()
        out, lse = case.run()
        case.expect(out, lse)


@pytest.mark.parametrize("offset,pad", [(1, 0), (8, 3), (0, 1), (3, 5)])
def test_strides_off_the_boundary(cuda_lib, offset, pad):
    """Queries, keys and values at any element offset and stride."""
    import torch
    case = Case(lens=[30, 140], nodes=6, heads=4, kv_heads=2, dim=72, page=16)

    def off(t):
        n, N, H, D = t.shape
        buf = torch.full((n * N * (H * (D + pad) + 7) + offset,), float("nan"), dtype=t.dtype, device="cuda")
        v = buf[offset:].view(n, N, H * (D + pad) + 7)[:, :, :H * (D + pad)].unflatten(2, (H, D + pad))[..., :D]
        v.copy_(t)
        return v
    out, lse = case.run()
    case.q, case.k, case.v = off(case.q), off(case.k), off(case.v)
    out2, lse2 = case.run()
    case.expect(out2, lse2)
    case.stored()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    # heads before nodes
    case.q = case.q.transpose(1, 2).contiguous().transpose(1, 2)
    case.k = case.k.transpose(1, 2).contiguous().transpose(1, 2)
    out3, _ = case.run()
    assert torch.equal(out, out3)


def test_layers(cuda_lib):
    import torch
    case = Case(lens=[40, 200], nodes=5, heads=4, kv_heads=2, dim=64, page=32, layers=3, layer=2)
    out, lse = case.run()
    case.expect(out, lse)
    assert torch.isnan(case.c.k[:2]).all()


def test_pages_past_32_bit_offsets(cuda_lib):
    """A sequence whose pages lie past 2^32 elements of the pools."""
    import torch
    from tinygpt_b200 import PagedCache
    page, heads, dim = 64, 8, 128
    pages = 2 ** 32 // (page * heads * dim) + 40
    case = Case(lens=[500], nodes=5, heads=16, kv_heads=8, dim=dim, page=page)
    big = PagedCache(1, heads, dim, page, pages, 4, pages)
    big.extend(dev([0]), dev([(pages - 20) * page]))
    big.commit(dev([0]), dev([(pages - 20) * page]))
    big.extend(dev([1]), dev([500]))
    big.commit(dev([1]), dev([500]))
    big.extend(dev([1]), dev([5]))
    t = torch.arange(500)
    src = case.c.tables[int(case.seqs[0])].cpu().long()[t // page].cuda()
    dst = big.tables[1].cpu().long()[t // page].cuda()
    assert int(dst.min()) >= 2 ** 32 // (page * heads * dim)
    s = (t % page).cuda()
    big.k[0, dst, :, s] = case.c.k[0, src, :, s]
    big.v[0, dst, :, s] = case.c.v[0, src, :, s]
    out, lse = case.run()
    case.expect(out, lse)
    out2, lse2 = big.tree_attention(0, dev([1]), case.q, case.k, case.v, as_tensor(case.masks), want_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    t = torch.arange(500, 505)
    dst = big.tables[1].cpu().long()[t // page].cuda()
    assert torch.equal(big.k[0, dst, :, (t % page).cuda()], case.k[0])
    # forked: the copy of the partly filled page, past 2^32 elements too
    big.fork(dev([1, 1]), dev([2, 3]))
    big.extend(dev([2, 3]), dev([5, 5]))
    out3, lse3 = big.tree_attention(0, dev([3]), case.q, case.k, case.v, as_tensor(case.masks), want_lse=True)
    assert torch.equal(out, out3) and big.device_status() == 0


def test_same_twice_other_stream_and_graph(cuda_lib):
    """Bit-equal in every run; on another stream; captured in a graph whose lengths then move."""
    import torch
    case = Case(lens=[4000, 60, 900], nodes=6, heads=8, kv_heads=2, dim=128, page=64)
    out, lse = case.run()
    for _ in range(3):
        again, lse2 = case.run()
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    masks, n = as_tensor(case.masks), dev(case.n_nodes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, _ = case.run(masks=masks, n_nodes=n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, b)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        case.c.tree_attention(0, case.seqs, case.q, case.k, case.v, masks, n_nodes=n, out=o2, lse=l2)
    g.replay()
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    case.c.truncate(case.seqs, dev([130, 0, 899]))
    case.c.extend(case.seqs, n)
    case.lens = np.array([130, 0, 899])
    g.replay()
    case.expect(o2, l2)


def test_one_after_another_without_waiting(cuda_lib):
    """Calls of other shapes between: nothing of one call is left for the next."""
    import torch
    a = Case(lens=[3000, 20], nodes=16, heads=8, kv_heads=2, dim=128, page=64, seed=1)
    b = Case(lens=[700] * 9, nodes=3, heads=4, kv_heads=4, dim=64, page=16, seed=2, dtype="f16")
    first = [x.run()[0] for x in (a, b)]
    for _ in range(20):
        got = [x.run()[0] for x in (a, b, a)]
    assert torch.equal(first[0], got[0]) and torch.equal(first[1], got[1]) and torch.equal(first[0], got[2])


def test_unreserved_nodes_are_not_stored(cuda_lib):
    """Without pages for them the nodes attend all the same; their keys are dropped and a bit is set."""
    import torch
    case = Case(lens=[30, 16], nodes=5, heads=4, kv_heads=2, dim=64, page=16)
    out, lse = case.run()
    case.c.truncate(case.seqs, dev(case.lens))
    before = case.c.k.clone()
    out2, _ = case.run()
    assert torch.equal(out, out2)
    assert case.c.device_status() == 8
    assert torch.equal(before.nan_to_num(7.0), case.c.k.nan_to_num(7.0))  # row 0 has room for 2, as before


def test_bad_rows(cuda_lib):
    import torch
    case = Case(lens=[30, 16], nodes=5, heads=4, kv_heads=2, dim=64, page=16)
    good, _ = case.run()
    case.seqs[0] = 99
    out, lse = case.run()
    assert case.c.device_status() & 1
    assert (out[0] == 0).all() and torch.equal(out[1], good[1])
    case.seqs[0] = -1
    out, lse = case.run()
    assert case.c.device_status() & 1 and (out[0] == 0).all()
    out, _ = case.run(n_nodes=dev([5, 6]))
    assert case.c.device_status() & 32
    assert (out[1] == 0).all()
    out, _ = case.run(n_nodes=dev([5, -1]))
    assert case.c.device_status() & 32 and (out[1] == 0).all()


def test_refusals(cuda_lib):
    import torch
    case = Case(lens=[30], nodes=5, heads=4, kv_heads=2, dim=64, page=16)
    c, q, k, v, s = case.c, case.q, case.k, case.v, case.seqs
    for call in (lambda: c.tree_attention(0, s, q.half(), k, v), lambda: c.tree_attention(0, s, q, k[:, :4], v),
                 lambda: c.tree_attention(0, s, q, k[:, :, :1], v), lambda: c.tree_attention(0, s, q[..., :32], k, v),
                 lambda: c.tree_attention(0, s, q, k, v, as_tensor(case.masks).int()), lambda: c.tree_attention(0, s, q[0], k, v),
                 lambda: c.tree_attention(0, s, q, k, v, n_nodes=dev([5, 5])), lambda: c.tree_attention(0, s, q, k, v, out=q),
                 lambda: c.tree_attention(0, s.long(), q, k, v), lambda: c.tree_attention(0, s, q, k, v, lse=torch.empty(1, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    big = torch.zeros((1, 65, 4, 64), dtype=c.dtype, device="cuda")
    for call in (lambda: c.tree_attention(1, s, q, k, v), lambda: c.tree_attention(-1, s, q, k, v),
                 lambda: c.tree_attention(0, s, big, big[:, :, :2], big[:, :, :2]), lambda: c.tree_attention(0, s, q[:, :, :3], k, v),
                 lambda: c.tree_attention(0, s, q, k, v, scale=float("nan")), lambda: c.tree_attention(0, s, q, k, v, scale=float("inf"))):
        with pytest.raises(_lib.TGError):
            call()
    assert cuda_lib.tg_tree_attention(c.handle, 0, 1, None, 5, None, None, 4, None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, ctypes.c_float(1.0),
                                      None, None, None) == _lib.TG_ERR_INVALID_ARG
    assert c.device_status() == 0
