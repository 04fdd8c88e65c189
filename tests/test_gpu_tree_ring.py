"""Tree attention where queries and nodes leave the ring of keys and values the fewest slots.

At head dimensions above 64, 128 rows and 64 nodes take the most shared memory that a
block of 128 rows can; the last tile of a context that is no multiple of 16 tokens has
rows cleared behind the sequence's end while other tiles are on their way.  Against the
64-bit definition, with the tolerances of test_gpu_tree.py.
"""
import numpy as np
import pytest

from tests.test_gpu_tree import Case, go

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nodes,dim", [(61, 128), (62, 96), (63, 80), (64, 72), (64, 128)])
def test_short_last_tiles(cuda_lib, nodes, dim, dtype):
    """Two heads to a key head, many sequences of 2 to 4 tiles, none a multiple of 16 tokens."""
    r = np.random.default_rng(nodes + dim)
    lens = r.integers(129, 400, 24)
    lens += lens % 16 == 0
    go(lens=lens, nodes=nodes, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, seed=nodes)


@pytest.mark.parametrize("nodes,group", [(64, 2), (64, 1), (48, 2), (40, 3), (32, 4), (42, 3)])
def test_long_contexts(cuda_lib, nodes, group):
    """The smallest rings over many tiles, items cut over blocks, and short rows beside them."""
    go(lens=[9001, 3, 2050, 0, 131, 4099], nodes=nodes, heads=group, kv_heads=1, dim=128, page=64, seed=group)


def test_the_same_bits_every_time(cuda_lib):
    """However the loads of many sequences fall, the result is one."""
    import torch
    r = np.random.default_rng(9)
    case = Case(lens=r.integers(129, 700, 40), nodes=64, heads=4, kv_heads=2, dim=128, page=32, seed=9)
    out, lse = case.run()
    for _ in range(20):
        again, lse2 = case.run()
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    case.expect(out, lse)
