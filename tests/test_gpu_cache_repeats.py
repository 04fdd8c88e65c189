"""Commit with a slot given more than once: the length never passes the reserved pages."""
import pytest

from tests.test_gpu_cache import dev, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("times", [2, 12])
def test_each_commit_counts_while_there_is_room(cuda_lib, times):
    c, _ = make(page=8, pages=40, seqs=12, width=6)
    c.extend(dev([0, 1]), dev([20, 44]))  # 24 and 48 places
    c.commit(dev([1] * times), dev([4] * times))
    assert c.lens.tolist()[:2] == [0, 4 * times] and c.device_status() == 0
    # of rows that together pass the pages, as many as fit
    c.commit(dev([0] * 12), dev([7] * 12))
    assert c.lens.tolist()[:2] == [21, 4 * times] and c.device_status() == 8
    c.commit(dev([0, 0, 0]), dev([3, 0, -1]))
    assert c.lens[0] == 24 and c.device_status() == 4


def test_rows_of_many_blocks(cuda_lib):
    """A call's rows lie in several blocks."""
    c, _ = make(layers=1, heads=1, dim=8, page=8, pages=300, seqs=1000, width=250)
    c.extend(dev([5]), dev([999]))
    c.commit(dev([5] * 1000), dev([1] * 1000))
    assert c.lens[5] == 1000 and c.device_status() == 0  # 125 pages
    c.commit(dev([5] * 1000), dev([1] * 1000))
    assert c.lens[5] == 1000 and c.device_status() == 8
