"""Tree attention in f16: the many small weights of a long context.

The weights are rounded to f16 for the product with the values.  They are scaled so that
the largest of a row lies between 2^7 and 2^15, so a weight is rounded to 2^-11 of itself
or, below 2^-21 of the largest, to 2^-32 of the largest at worst (half of f16's step of
2^-24, over 2^7).  The other parts of the tolerance are those of test_gpu_tree.py.
"""
import numpy as np
import pytest

from tests.decode_reference import tree_reference
from tests.test_gpu_tree import Case, dev

pytestmark = pytest.mark.gpu


def some_large(tokens, weight_log2, large, nodes=1, heads=1):
    """A row whose tokens `large` have weight 1 and value 0, all others 2^weight_log2 and value 1; the node itself is unseen."""
    import torch
    from tinygpt_b200 import PagedCache
    page = 256
    width = -(-(tokens + nodes) // page)
    c = PagedCache(1, 1, 64, page, width, 1, width, dtype=torch.float16)
    c.k.zero_(), c.v.fill_(1.0)
    c.extend(dev([0]), dev([tokens]))
    c.commit(dev([0]), dev([tokens]))
    c.extend(dev([0]), dev([nodes]))
    t = torch.tensor(large, device="cuda")
    p = c.tables[0].long()[t // page]
    c.k[0, p, 0, t % page, 0] = 1.0
    c.v[0, p, 0, t % page] = 0.0
    q = torch.zeros((1, nodes, heads, 64), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    kv = torch.zeros((1, nodes, 1, 64), dtype=torch.float16, device="cuda")
    masks = torch.zeros((1, nodes), dtype=torch.int64, device="cuda")
    out, lse = c.tree_attention(0, dev([0]), q, kv, kv, masks, scale=-weight_log2 * float(np.log(2.0)), want_lse=True)
    assert c.device_status() == 0
    return out.double().cpu(), lse.double().cpu()


@pytest.mark.parametrize("nodes,heads", [(1, 1), (3, 4), (64, 4)])
@pytest.mark.parametrize("tokens,weight_log2", [(1 << 20, -25.25), (1 << 20, -22.5), (1 << 18, -24.75), (70001, -19.3), (5000, -13.0), (5000, -3.0)])
def test_mass_of_small_weights(cuda_lib, tokens, weight_log2, nodes, heads):
    """One weight takes the row, and a million others have a part of it that f16 can show."""
    for at in (0, 127, tokens - 1):
        out, _ = some_large(tokens, weight_log2, [at], nodes, heads)
        small = (tokens - 1) * 2.0 ** weight_log2
        want, total = small / (1 + small), 1 + small
        # a score of 18 at most, in fp32: 2^-23 of it and the scale's own rounding; the exponentials
        move = 3 * 2.0 ** -23 * 18 + 2.0 ** -18
        tol = 2.0 ** -11 * (want + 1.01 * want) + 2 * move * want + tokens * 2.0 ** -32 / total + 2.0 ** -24
        assert (out - want).abs().max() <= tol, (at, out.min().item(), out.max().item(), want, tol)


@pytest.mark.parametrize("nodes,heads", [(1, 1), (3, 4), (64, 4)])
@pytest.mark.parametrize("tokens,weight_log2,every", [(1 << 20, -25.25, 1024), (1 << 20, -24.0, 512), (1 << 18, -27.5, 2048), (70001, -19.3, 128)])
def test_small_weights_beside_many_large(cuda_lib, tokens, weight_log2, every, nodes, heads):
    """Large weights in every part of the row that a block may take: none of the small ones is measured by itself."""
    large = list(range(every // 2, tokens, every))
    out, _ = some_large(tokens, weight_log2, large, nodes, heads)
    small = (tokens - len(large)) * 2.0 ** weight_log2
    total = len(large) + small
    want = small / total
    move = 3 * 2.0 ** -23 * 20 + 2.0 ** -18
    tol = 2.0 ** -11 * 2.01 * want + 2 * move * want + tokens * 2.0 ** -32 / total + 2.0 ** -24
    assert want > 4 * tol
    assert (out - want).abs().max() <= tol, (out.min().item(), out.max().item(), want, tol)


@pytest.mark.parametrize("dim,std,seed", [(64, 4.0, 0), (128, 2.5, 1), (64, 8.0, 2)])
def test_peaked_rows(cuda_lib, dim, std, seed):
    """Random scores of a wide range over a long context."""
    case = Case(lens=[16001, 3000], nodes=5, heads=4, kv_heads=2, dim=dim, page=64, dtype="f16", std=std, seed=seed)
    out, lse = case.run()
    want, want_lse, weight, spread, peak = tree_reference(case.c, 0, case.seqs.cpu(), case.lens, case.q, case.k, case.v, case.masks, case.n_nodes, case.scale)
    move = (dim + 2) * 2.0 ** -23 * spread + 2.0 ** -18
    vmax = max(t.float().nan_to_num(0.0, 0.0, 0.0).abs().max().item() for t in (case.c.v, case.v))
    tol = 2.0 ** -11 * (want.abs() + 1.01 * weight) + 2 * move[..., None] * weight + (16001 + 5) * 2.0 ** -32 * vmax * peak[..., None] + 2.0 ** -24
    assert ((out.double().cpu() - want).abs() <= tol).all()
    assert ((lse.double().cpu() - want_lse).abs() <= move + 2.0 ** -20 * want_lse.abs().clamp(min=1)).all()


def test_values_at_the_ends_of_the_range(cuda_lib):
    """Values of 65,504 under weights of 2^7 to 2^15 times what they stand for: sums in 32 bits hold them."""
    import torch
    case = Case(lens=[4000, 130], nodes=6, heads=4, kv_heads=2, dim=64, page=64, dtype="f16", std=6.0)
    case.c.v[torch.isfinite(case.c.v)] = 65504.0
    case.v[:] = 65504.0
    out, _ = case.run()
    # the weights' sum and the sum of their rounded ones differ by 2^-11 at most
    assert (out.double() - 65504.0).abs().max() <= 65504.0 * 2.0 ** -10 and torch.isfinite(out).all()


@pytest.mark.parametrize("nodes,heads", [(1, 1), (3, 4), (64, 4)])
@pytest.mark.parametrize("tokens,weight_log2", [(1 << 20, -25.25), (1 << 20, -22.5), (1 << 18, -24.75), (70001, -19.3), (5000, -13.0), (5000, -3.0)])
def test_sum_of_small_weights(cuda_lib, tokens, weight_log2, nodes, heads):
    """The logarithm of a row's sum counts the small weights beside a large one: 64 of them meet it at a time."""
    for at in (0, 127, tokens - 1):
        _, lse = some_large(tokens, weight_log2, [at], nodes, heads)
        total = 1 + (tokens - 1) * 2.0 ** weight_log2
        move = 3 * 2.0 ** -23 * 18 + 2.0 ** -18
        assert (lse - (-weight_log2 * np.log(2.0) + np.log(total))).abs().max() <= move + 2.0 ** -20 * 24
