"""A tree that accept cannot settle leaves its row as it was: the reserved pages, and what is stored in them."""
import numpy as np
import pytest

from tests.test_gpu_cache import dev, make, value

pytestmark = pytest.mark.gpu


def state(c):
    return c.lens.tolist(), c.counts.tolist(), c.tables.tolist(), c.refs.tolist()


def filled(pages=12):
    """Slot 1 with 11 tokens and 10 nodes stored past them: 3 pages of 8, the last of them reserved only."""
    c, _ = make(layers=2, heads=1, page=8, pages=pages, seqs=6, width=6)
    c.extend(dev([1]), dev([11]))
    c.commit(dev([1]), dev([11]))
    c.extend(dev([1]), dev([10]))
    for layer in range(2):
        k = np.arange(10)
        t = value(c, 0)[0][layer].repeat(10, 1, 1)[None] + dev(k)[None, :, None, None].to(c.dtype)
        c.append(layer, dev([1]), t, -t)
    assert c.device_status() == 0 and c.counts[1] == 3
    return c


TREE = [[-1] + list(range(9))]
TOKENS, IDS = [list(range(10))], [list(range(1, 11))]


def accept(c, slot, n_nodes=None):
    out, n = c.accept(dev([slot]), dev(TREE), dev(TOKENS), dev(IDS), n_nodes=None if n_nodes is None else dev([n_nodes]))
    return out[0].tolist(), n.item()


@pytest.mark.parametrize("n_nodes", [-1, 11, 2 ** 31 - 1])
def test_bad_node_count(cuda_lib, n_nodes):
    import torch
    c = filled()
    before, k = state(c), c.k.clone()
    assert accept(c, 1, n_nodes) == ([-1] * 10, 0)
    assert c.device_status() == 32
    assert state(c) == before and torch.equal(c.k.nan_to_num(7.0), k.nan_to_num(7.0))
    # put right, the same tree is settled
    assert accept(c, 1, 10) == (list(range(1, 11)), 10)
    assert c.device_status() == 0 and c.lens[1] == 21 and c.counts[1] == 3
    assert torch.equal(c.k.nan_to_num(7.0), k.nan_to_num(7.0))


def test_tree_past_the_reserved_pages(cuda_lib):
    c = filled()
    c.commit(dev([1]), dev([4]))  # 15 tokens: 9 places are left of 24
    before = state(c)
    assert accept(c, 1) == ([-1] * 10, 0)
    assert c.device_status() == 8 and state(c) == before
    c.extend(dev([1]), dev([10]))
    assert accept(c, 1)[1] == 10 and c.device_status() == 0


def test_shared_last_page(cuda_lib):
    """A fork holds the page that the row ends in: the row keeps what it reserved behind it."""
    c = filled()
    c.fork(dev([1]), dev([2]))
    before = state(c)
    assert before[1] == [0, 3, 2, 0, 0, 0]
    for slot in (1, 2):
        assert accept(c, slot, 3) == ([-1] * 10, 0)
        assert c.device_status() == 8 and state(c) == before
    c.free(dev([2]))
    assert accept(c, 1)[1] == 10 and c.device_status() == 0


def test_beside_rows_that_are_served(cuda_lib):
    """A slot named twice, a slot that is none and a bad count, between rows that are settled."""
    c = filled()
    c.extend(dev([0, 3]), dev([10, 10]))
    seqs, n = dev([0, 9, 1, 3, 3]), dev([10, 10, 11, 10, 10])
    rows = lambda x: dev(np.repeat(np.array(x), 5, 0))  # noqa: E731
    tables = c.tables.tolist()
    out, taken = c.accept(seqs, rows(TREE), rows(TOKENS), rows(IDS), n_nodes=n)
    taken = taken.tolist()
    assert c.device_status() == 33
    assert taken[:3] == [10, 0, 0] and sorted(taken[3:]) == [0, 10]
    assert c.lens.tolist() == [10, 11, 0, 10, 0, 0] and c.counts.tolist() == [2, 3, 0, 2, 0, 0] and c.tables.tolist() == tables
