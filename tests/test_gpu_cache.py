"""The paged cache's bookkeeping and page copies against a model in Python lists."""
import ctypes

import numpy as np
import pytest

from tests.decode_reference import PagedModel
from tinygpt_b200 import _lib

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def make(layers=2, heads=3, dim=16, page=8, pages=40, seqs=12, width=6, dtype="bf16"):
    import torch
    from tinygpt_b200 import PagedCache
    c = PagedCache(layers, heads, dim, page, pages, seqs, width, dtype=torch.bfloat16 if dtype == "bf16" else torch.float16)
    c.k.fill_(float("nan"))
    c.v.fill_(float("nan"))
    return c, PagedModel(pages, seqs, page, width)


def value(c, x):
    """A stored token's keys and values [layers, heads, dim] from its number: exact in 16 bits."""
    import torch
    layer = torch.arange(c.layers, device="cuda")[:, None, None]
    head = torch.arange(c.kv_heads, device="cuda")[None, :, None]
    col = torch.arange(c.head_dim, device="cuda")[None, None, :]
    k = ((x * 7 + layer * 31 + head * 13 + col) % 251).to(c.dtype)
    return k, -k


def store(c, m, seqs, numbers):
    """Token numbers[i] (a list) stored past slot seqs[i]'s length in every layer."""
    import torch
    most = max(len(n) for n in numbers)
    if most == 0:
        return
    k = torch.zeros((c.layers, len(seqs), most, c.kv_heads, c.head_dim), dtype=c.dtype, device="cuda")
    v = torch.zeros_like(k)
    for i, n in enumerate(numbers):
        for t, x in enumerate(n):
            k[:, i, t], v[:, i, t] = value(c, x)
    for layer in range(c.layers):
        c.append(layer, dev(seqs), k[layer], v[layer], dev([len(n) for n in numbers]))
    for s, n in zip(seqs, numbers):
        m.store(s, n)


def served(m, s, n):
    """Slot s has n places past its length that it alone holds."""
    at = m.lens[s] // m.page
    return m.lens[s] + n <= len(m.rows[s]) * m.page and (m.lens[s] % m.page == 0 or m.refs[m.rows[s][at]] == 1)


def same(c, m):
    assert c.lens.tolist() == m.lens
    assert c.counts.tolist() == [len(r) for r in m.rows]
    assert c.tables.tolist() == [r + [-1] * (m.width - len(r)) for r in m.rows]
    assert c.refs.tolist() == m.refs
    for s, n in enumerate(m.lens):  # every committed token where the model has it
        for t in range(n):
            p, slot = m.place(s, t)
            x = m.text.get((p, slot))
            if x is not None:
                k, v = value(c, x)
                assert (c.k[:, p, :, slot] == k).all() and (c.v[:, p, :, slot] == v).all(), (s, t)


@pytest.mark.parametrize("seed,page,dtype", [(0, 8, "bf16"), (1, 8, "f16"), (2, 16, "bf16"), (3, 64, "f16")])
def test_random_calls(cuda_lib, seed, page, dtype):
    """Extends, stores, forks (in place, with repeats, to empty), cuts, trees settled, in random order."""
    r = np.random.default_rng(seed)
    c, m = make(page=page, dtype=dtype)
    number = 0
    for step in range(60):
        op = r.choice(["grow", "grow", "fork", "cut", "accept", "free"])
        n = int(r.integers(1, 9))
        seqs = r.permutation(12)[:n]
        if op == "grow":
            counts = r.integers(0, 2 * page, n)
            c.extend(dev(seqs), dev(counts))
            m.extend(seqs, counts)
            fits = [int(a) if served(m, s, a) else 0 for s, a in zip(seqs, counts)]
            numbers = [list(range(number + 100 * i, number + 100 * i + f)) for i, f in enumerate(fits)]
            number += 1000
            store(c, m, seqs, numbers)
            c.commit(dev(seqs), dev(fits))
            for s, f in zip(seqs, fits):
                m.commit(s, f)
        elif op == "fork":
            src = r.integers(-1, 12, n)
            c.fork(dev(src), dev(seqs))
            m.fork(src, seqs)
        elif op in ("cut", "free"):
            lens = np.array([int(r.integers(0, m.lens[s] + 1)) if op == "cut" else 0 for s in seqs])
            c.truncate(dev(seqs), dev(lens)) if op == "cut" else c.free(dev(seqs))
            for s, x in zip(seqs, lens):
                m.truncate(s, int(x))
        else:
            N = int(r.integers(1, 2 * page))
            N = min(N, 64)
            c.extend(dev(seqs), dev([N] * n))
            m.extend(seqs, [N] * n)
            seqs = np.array([s for s in seqs if served(m, s, N)], dtype=np.int64)
            n = len(seqs)
            if n == 0:
                continue
            store(c, m, seqs, [list(range(number + 100 * i, number + 100 * i + N)) for i in range(n)])
            number += 1000
            parents = np.array([[-1] + [int(r.integers(0, j)) for j in range(1, N)] for _ in range(n)])
            tokens, ids = r.integers(0, 3, (n, N)), r.integers(0, 3, (n, N))
            out, count = c.accept(dev(seqs), dev(parents), dev(tokens), dev(ids))
            for i, s in enumerate(seqs):
                want = m.accept(s, parents[i].tolist(), tokens[i].tolist(), ids[i].tolist())
                assert count[i].item() == len(want)
                assert out[i].tolist() == want + [-1] * (N - len(want))
        same(c, m)
        c.device_status()
    c.free(dev(np.arange(12)))
    for s in range(12):
        m.truncate(s, 0)
    same(c, m)
    assert sum(m.refs) == 0


def test_beams_share_and_copy(cuda_lib):
    """Four beams of one prompt: the prompt's full pages are shared, the partly filled one is copied for
    all but the first of its only holders."""
    c, m = make(pages=40, page=8, width=6)
    c.extend(dev([0]), dev([21]))
    m.extend([0], [21])
    store(c, m, [0], [list(range(21))])
    c.commit(dev([0]), dev([21]))
    m.commit(0, 21)
    c.fork(dev([0, 0, 0, 0]), dev([0, 1, 2, 3]))
    m.fork([0, 0, 0, 0], [0, 1, 2, 3])
    same(c, m)
    assert m.refs[:3] == [4, 4, 4]
    c.extend(dev([3, 1, 0, 2]), dev([1, 1, 1, 1]))
    m.extend([3, 1, 0, 2], [1, 1, 1, 1])
    same(c, m)
    assert m.refs[:3] == [4, 4, 1] and m.rows[3][2] == 2 and [m.rows[s][2] for s in (1, 0, 2)] == [3, 4, 5]
    store(c, m, [0, 1, 2, 3], [[100], [101], [102], [103]])
    c.commit(dev([0, 1, 2, 3]), dev([1, 1, 1, 1]))
    for s in range(4):
        m.commit(s, 1)
    same(c, m)
    c.fork(dev([3, 3, -1, 0]), dev([0, 1, 2, 3]))  # the beams replaced by their parents, one emptied
    m.fork([3, 3, -1, 0], [0, 1, 2, 3])
    same(c, m)
    assert c.device_status() == 0


def test_pages_run_out_in_row_order(cuda_lib):
    c, m = make(pages=5, page=8, width=6)
    c.extend(dev([4, 2, 7, 1]), dev([16, 8, 40, 1]))
    m.extend([4, 2, 7, 1], [16, 8, 40, 1])
    same(c, m)
    assert [len(m.rows[s]) for s in (4, 2, 7, 1)] == [2, 1, 0, 0]
    assert c.device_status() == 2 and c.device_status() == 0


def test_many_rows_and_pages(cuda_lib):
    """More rows than the block has threads, a bitmap of many words, a page count off the word."""
    r = np.random.default_rng(5)
    c, m = make(layers=1, heads=1, dim=8, page=8, pages=9001, seqs=2500, width=9)
    seqs = r.permutation(2500)
    for _ in range(2):
        counts = r.integers(0, 20, 2500)
        c.extend(dev(seqs), dev(counts))
        m.extend(seqs, counts)
        c.commit(dev(seqs), dev(counts))
        for s, n in zip(seqs, counts):
            m.commit(s, int(n))
    src = r.integers(-1, 2500, 2500)
    c.fork(dev(src), dev(seqs))
    m.fork(src, seqs)
    c.extend(dev(seqs), dev(np.ones(2500)))
    m.extend(seqs, [1] * 2500)
    assert c.lens.tolist() == m.lens
    assert c.tables.tolist() == [x + [-1] * (9 - len(x)) for x in m.rows]
    assert c.refs.tolist() == m.refs


def test_rows_that_cannot_be_served(cuda_lib):
    """Bad slots, repeated slots, bad lengths, unreserved positions: the row stays, a status bit tells."""
    c, m = make()
    c.extend(dev([0, 1]), dev([10, 10]))
    m.extend([0, 1], [10, 10])
    store(c, m, [0, 1], [list(range(10)), list(range(50, 60))])
    c.commit(dev([0, 1]), dev([10, 10]))
    m.commit(0, 10), m.commit(1, 10)
    assert c.device_status() == 0
    c.extend(dev([-1, 12, 2]), dev([1, 1, 9]))
    m.extend([2], [9])
    assert c.device_status() == 1
    same(c, m)
    c.extend(dev([3, 3]), dev([1, 1]))
    m.extend([3], [1])
    assert c.device_status() == 1
    same(c, m)
    c.extend(dev([0, 1]), dev([-3, 48]))
    assert c.device_status() == 4
    c.fork(dev([12, 0, 0, -2]), dev([4, -1, 99, 5]))
    assert c.device_status() == 1
    c.truncate(dev([0, 1]), dev([11, -1]))
    assert c.device_status() == 4
    c.commit(dev([0]), dev([7]))  # 2 pages hold 16
    assert c.device_status() == 8
    c.commit(dev([0]), dev([-1]))
    assert c.device_status() == 4
    same(c, m)
    k, v = value(c, 900)
    six = k[0].expand(1, 8, c.kv_heads, c.head_dim).contiguous()
    c.append(0, dev([0]), six, -six)  # 8 tokens, room for 6
    assert c.device_status() == 8
    c.append(0, dev([0]), six, -six, dev([9]))
    assert c.device_status() == 4
    out, n = c.accept(dev([0]), dev([[-1] + [0] * 7]), dev([[0] * 8]), dev([[1] * 8]))  # 8 nodes, room for 6
    assert c.device_status() == 8 and n.item() == 0 and (out == -1).all()
    out, n = c.accept(dev([1]), dev([[-1, 0]]), dev([[0, 1]]), dev([[1, 2]]), n_nodes=dev([3]))
    assert c.device_status() == 32 and n.item() == 0
    same(c, m)


@pytest.mark.parametrize("dim,offset", [(16, 0), (24, 0), (16, 1), (8, 3)])
def test_append_strides(cuda_lib, dim, offset):
    """Keys and values out of one projection's output, on and off 16-byte boundaries."""
    import torch
    c, _ = make(dim=dim, heads=2, layers=2, page=8, pages=9, width=4)
    c.extend(dev([3, 5]), dev([20, 11]))
    flat = torch.randn(2 * 20 * 5 * dim + offset, device="cuda").to(c.dtype)[offset:].view(2, 20, 5, dim)
    k, v = flat[:, :, :2], flat[:, :, 3:]
    c.append(1, dev([3, 5]), k, v, dev([20, 11]))
    t = torch.arange(20, device="cuda")
    for row, (s, n) in enumerate(((3, 20), (5, 11))):
        page = c.tables[s].long()[t[:n] // 8]
        assert torch.equal(c.k[1, page, :, t[:n] % 8], k[row, :n])
        assert torch.equal(c.v[1, page, :, t[:n] % 8], v[row, :n])
    assert c.k[0].isnan().all() and c.device_status() == 0
    assert int((~c.k.isnan()).sum()) == 31 * 2 * dim


def test_masks_from_parents(cuda_lib):
    import torch
    from tinygpt_b200 import tree_masks
    r = np.random.default_rng(7)
    for n, nodes in ((1, 1), (5, 64), (40, 33), (3, 2)):
        parents = np.array([[-1] + [int(r.integers(max(0, j - 3), j)) for j in range(1, nodes)] for _ in range(n)])
        count = r.integers(0, nodes + 1, n)
        got = tree_masks(dev(parents), dev(count)).cpu().numpy().view(np.uint64)
        for b in range(n):
            for i in range(nodes):
                bits, j = 0, i if i < count[b] else -1
                while j >= 0:
                    bits |= 1 << j
                    j = parents[b, j] if j else -1
                assert int(got[b, i]) == bits
    chain = np.arange(-1, 63)[None]
    assert int(tree_masks(dev(chain))[0, 63].item()) == -1  # all 64 bits
    torch.cuda.synchronize()


def test_accept_longest_path(cuda_lib):
    """64 nodes in a line, all accepted; and the same tree with twins: the lower sibling is taken."""
    c, m = make(page=8, pages=30, width=16)
    c.extend(dev([2]), dev([5 + 64]))
    m.extend([2], [69])
    store(c, m, [2], [list(range(69))])
    c.commit(dev([2]), dev([5]))
    m.commit(2, 5)
    line = np.arange(-1, 63)[None]
    out, n = c.accept(dev([2]), dev(line), dev(np.arange(64)[None]), dev(np.arange(1, 65)[None]))
    assert n.item() == 64 and out[0].tolist() == list(range(1, 65))
    m.accept(2, line[0].tolist(), list(range(64)), list(range(1, 65)))
    same(c, m)
    c.truncate(dev([2]), dev([5]))
    m.truncate(2, 5)
    c.extend(dev([2]), dev([5]))
    m.extend([2], [5])
    store(c, m, [2], [[200, 201, 202, 203, 204]])
    tree = [[-1, 0, 0, 2, 1]]
    out, n = c.accept(dev([2]), dev(tree), dev([[0, 9, 9, 4, 4]]), dev([[9, 4, 4, 5, 6]]))
    assert n.item() == 3 and out[0].tolist() == [9, 4, 6, -1, -1]
    assert m.accept(2, tree[0], [0, 9, 9, 4, 4], [9, 4, 4, 5, 6]) == [9, 4, 6]
    same(c, m)


def test_step_in_a_graph(cuda_lib):
    """Extend, accept and fork captured once and replayed: lengths advance on the device alone."""
    import torch
    c, m = make(page=8, pages=60, width=10, layers=1)
    c.extend(dev([0, 1]), dev([3, 9]))
    m.extend([0, 1], [3, 9])
    c.commit(dev([0, 1]), dev([3, 9]))
    m.commit(0, 3), m.commit(1, 9)
    seqs, four = dev([0, 1]), dev([4, 4])
    parents, tokens, ids = dev([[-1, 0, 1, 0]] * 2), dev([[0, 5, 6, 7]] * 2), dev([[7, 0, 0, 1], [5, 6, 2, 0]])
    out, n = torch.empty((2, 4), dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    two, five = dev([0, 1]), dev([4, 5])
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            c.extend(seqs, four)
            c.accept(seqs, parents, tokens, ids, out_ids=out, out_n=n)
            c.fork(two, five)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(5):
        g.replay()
        m.extend([0, 1], [4, 4])
        for i in range(2):
            m.accept(i, parents[i].tolist(), tokens[i].tolist(), ids[i].tolist())
        m.fork([0, 1], [4, 5])
        assert c.lens.tolist() == m.lens and c.refs.tolist() == m.refs
        assert n.tolist() == [2, 3]
    assert c.device_status() == 0


def test_calls_allocate_nothing(cuda_lib):
    import torch
    c, _ = make()
    seqs, one = dev([0, 1, 2]), dev([3, 3, 3])

    def calls():
        c.extend(seqs, one)
        c.fork(seqs, dev([4, 5, 6]))
        c.free(seqs)
        torch.cuda.synchronize()

    calls()
    free0, _ = torch.cuda.mem_get_info()
    for _ in range(3):
        calls()
    assert torch.cuda.mem_get_info()[0] == free0


def test_a_dropped_cache_frees_its_memory(cuda_lib):
    """The views of the state keep the handle, not the pools; the handle goes with the last of them."""
    import gc
    import torch
    c, _ = make(pages=4000, dim=128, heads=8, page=64)
    lens = c.lens
    held = torch.cuda.memory_allocated()
    del c
    gc.collect()
    assert torch.cuda.memory_allocated() < held - 2 * 4000 * 8 * 64 * 128 * 2
    assert lens.sum().item() == 0


def test_refusals(cuda_lib):
    import torch
    from tinygpt_b200 import PagedCache
    P = ctypes.c_void_p
    c, _ = make()
    ok = (2, 3, 16, 8, 40, 12, 6)
    for bad, code in (((0, 3, 16, 8, 40, 12, 6), _lib.TG_ERR_INVALID_ARG), ((2, 3, 12, 8, 40, 12, 6), _lib.TG_ERR_UNSUPPORTED),
                      ((2, 3, 136, 8, 40, 12, 6), _lib.TG_ERR_UNSUPPORTED), ((2, 3, 16, 12, 40, 12, 6), _lib.TG_ERR_UNSUPPORTED),
                      ((2, 3, 16, 4, 40, 12, 6), _lib.TG_ERR_UNSUPPORTED), ((2, 3, 16, 512, 40, 12, 6), _lib.TG_ERR_UNSUPPORTED),
                      ((2, 3, 16, 8, 40, 70000, 6), _lib.TG_ERR_UNSUPPORTED)):
        cfg, h = _lib.CacheConfig(*bad, _lib.TG_DTYPE_BF16), ctypes.c_void_p()
        assert cuda_lib.tg_cache_create(0, ctypes.byref(cfg), P(c.k.data_ptr()), P(c.v.data_ptr()), ctypes.byref(h)) == code, bad
    for dtype in (_lib.TG_DTYPE_F32, 9):
        cfg, h = _lib.CacheConfig(*ok, dtype), ctypes.c_void_p()
        assert cuda_lib.tg_cache_create(0, ctypes.byref(cfg), P(c.k.data_ptr()), P(c.v.data_ptr()), ctypes.byref(h)) == _lib.TG_ERR_UNSUPPORTED
    cfg = _lib.CacheConfig(*ok, _lib.TG_DTYPE_BF16)
    assert cuda_lib.tg_cache_create(0, ctypes.byref(cfg), P(c.k.data_ptr() + 2), P(c.v.data_ptr()), ctypes.byref(h)) == _lib.TG_ERR_INVALID_ARG
    assert cuda_lib.tg_cache_create(77, ctypes.byref(cfg), P(c.k.data_ptr()), P(c.v.data_ptr()), ctypes.byref(h)) == _lib.TG_ERR_NO_DEVICE
    s, n = dev([0]), dev([1])
    a, b = P(s.data_ptr()), P(n.data_ptr())
    assert cuda_lib.tg_cache_extend(c.handle, 13, a, b, None) == _lib.TG_ERR_INVALID_ARG
    assert cuda_lib.tg_cache_extend(c.handle, -1, a, b, None) == _lib.TG_ERR_INVALID_ARG
    assert cuda_lib.tg_cache_extend(c.handle, 1, a, None, None) == _lib.TG_ERR_INVALID_ARG
    assert cuda_lib.tg_cache_extend(c.handle, 0, None, None, None) == _lib.TG_OK
    assert cuda_lib.tg_cache_accept(c.handle, 1, a, 65, None, a, a, a, a, a, None) == _lib.TG_ERR_UNSUPPORTED
    assert cuda_lib.tg_cache_append(c.handle, 2, 1, a, b, 1, a, 0, 0, 0, a, 0, 0, 0, None) == _lib.TG_ERR_INVALID_ARG
    x = torch.zeros((1, 1, 3, 16), dtype=c.dtype, device="cuda")
    for call in (lambda: c.extend(s.long(), n), lambda: c.extend(s, dev([1, 2])), lambda: c.extend(s.cpu(), n),
                 lambda: c.fork(s, dev([1, 2])), lambda: c.append(0, s, x.half(), x), lambda: c.append(0, s, x[..., :8], x),
                 lambda: c.append(0, s, x.transpose(2, 3).contiguous().transpose(2, 3), x),
                 lambda: c.accept(s, dev([[0, 1]]), dev([[0]]), dev([[0, 1]]))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        PagedCache(*ok, dtype=torch.float32)
    with pytest.raises(ValueError):
        PagedCache(*ok, k=c.k[:1], v=c.v)
    assert c.device_status() == 0
