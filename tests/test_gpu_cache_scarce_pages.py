"""Extend with too few pages for the copies of a shared page: no row counts as served that may not store."""
import pytest

from tests.test_gpu_cache import dev, make, value

pytestmark = pytest.mark.gpu


def shared(pages, prompts):
    """Slots 2i and 2i + 1 hold one prompt of prompts[i] tokens together, and nobody else does."""
    c, _ = make(layers=1, heads=1, page=8, pages=pages, seqs=8, width=4)
    for i, n in enumerate(prompts):
        c.extend(dev([2 * i]), dev([n]))
        c.commit(dev([2 * i]), dev([n]))
        c.fork(dev([2 * i]), dev([2 * i + 1]))
    assert c.device_status() == 0
    return c


def state(c):
    return c.lens.tolist(), c.counts.tolist(), c.tables.tolist(), c.refs.tolist()


def may_store(c, slot, n):
    k = value(c, slot)[0][0].expand(1, n, 1, c.head_dim).contiguous()
    c.append(0, dev([slot]), k, -k)
    return c.device_status() == 0


def test_no_page_for_the_other_holder(cuda_lib):
    """The pool is full: neither of the two may store, both are as they were."""
    c = shared(2, [11])
    before = state(c)
    c.extend(dev([0, 1]), dev([1, 1]))
    assert c.device_status() == 2 and state(c) == before
    assert not may_store(c, 0, 1) and not may_store(c, 1, 1)
    c.free(dev([1]))
    c.extend(dev([0]), dev([1]))
    assert c.device_status() == 0 and may_store(c, 0, 1)


def test_the_first_holder_wants_more_pages(cuda_lib):
    """One free page, for the first row's tokens past its length: of no use while the second holds its last page."""
    c = shared(3, [11])
    before = state(c)
    c.extend(dev([0, 1]), dev([6, 1]))
    assert c.device_status() == 2 and state(c) == before


def test_a_row_between(cuda_lib):
    """The one free page goes to a row between the two holders."""
    c = shared(3, [11])
    c.extend(dev([0, 4, 1]), dev([2, 5, 1]))
    assert c.device_status() == 2
    assert c.counts.tolist() == [2, 2, 0, 0, 1, 0, 0, 0] and c.tables[4, 0] == 2
    assert c.tables[:2, :2].tolist() == [[0, 1], [0, 1]] and c.refs.tolist() == [2, 2, 1]
    assert may_store(c, 4, 5) and not may_store(c, 0, 1)


def test_one_page_for_two_pairs(cuda_lib):
    """A pair inside another: the inner is served, the outer's last row does not fit, so its first is not served."""
    c = shared(5, [11, 12])
    assert c.tables[:4, :2].tolist() == [[0, 1], [0, 1], [2, 3], [2, 3]]
    c.extend(dev([0, 2, 3, 1]), dev([1, 1, 1, 1]))
    assert c.device_status() == 2
    assert c.tables[:4, :2].tolist() == [[0, 1], [0, 1], [2, 3], [2, 4]] and c.refs.tolist() == [2, 2, 2, 1, 1]
    assert may_store(c, 2, 1) and may_store(c, 3, 1) and not may_store(c, 0, 1) and not may_store(c, 1, 1)


def test_three_holders(cuda_lib):
    """The second copies, the third does not fit: the page has two holders left, the first may not store."""
    c = shared(3, [11])
    c.fork(dev([0]), dev([4]))
    c.extend(dev([0, 1, 4]), dev([1, 1, 1]))
    assert c.device_status() == 2
    assert [c.tables[s, 1].item() for s in (0, 1, 4)] == [1, 2, 1] and c.refs.tolist() == [3, 2, 1]
    assert may_store(c, 1, 1) and not may_store(c, 0, 1) and not may_store(c, 4, 1)


def test_enough_pages(cuda_lib):
    """With a page for each copy the first of each pair keeps the page, as ever."""
    c = shared(6, [11, 12])
    c.extend(dev([0, 2, 3, 1]), dev([1, 1, 1, 1]))
    assert c.device_status() == 0
    assert c.tables[:4, :2].tolist() == [[0, 1], [0, 5], [2, 3], [2, 4]]
    assert all(may_store(c, s, 1) for s in range(4))


def test_many_pairs(cuda_lib):
    """1,500 pairs, more rows than the block has threads, and pages for 700 copies: 700 pairs are served, the
    others are as they were; freed of their forks, their firsts are served too."""
    import torch
    c, _ = make(layers=1, heads=1, dim=8, page=8, pages=1500 + 700, seqs=3000, width=2)
    first = torch.arange(1500, device="cuda", dtype=torch.int32)
    three = torch.full_like(first, 3)
    c.extend(first, three)
    c.commit(first, three)
    c.fork(first, first + 1500)
    seqs = torch.cat([first, first + 1500])
    c.extend(seqs, torch.ones_like(seqs))
    assert c.device_status() == 2
    last = c.tables[:, 0].tolist()
    assert last == list(range(1500)) + list(range(1500, 2200)) + list(range(700, 1500))
    assert c.refs.tolist() == [1] * 700 + [2] * 800 + [1] * 700
    assert (c.counts == 1).all() and (c.lens == 3).all()
    c.free(first[700:] + 1500)
    c.extend(first, torch.ones_like(first))
    assert c.device_status() == 0 and c.tables[:1500, 0].tolist() == list(range(1500))
