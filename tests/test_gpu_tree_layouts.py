"""Tree attention's two ways to bring queries and pages: the same numbers whatever the layout."""
import pytest

pytestmark = pytest.mark.gpu


def filled(dim, kv_heads, page, lens, dtype, room=64):
    """A cache whose slots hold `lens` tokens of fixed pseudo-random keys and values."""
    import torch
    from tinygpt_b200 import PagedCache
    width = max(-(-(n + room) // page) for n in lens)
    c = PagedCache(1, kv_heads, dim, page, width * len(lens), len(lens), width, dtype=dtype)
    c.k.fill_(float("nan"))
    c.v.fill_(float("nan"))
    seqs = torch.arange(len(lens), dtype=torch.int32, device="cuda")
    c.extend(seqs, torch.tensor([n + room for n in lens], dtype=torch.int32, device="cuda"))
    g = torch.Generator("cuda").manual_seed(dim + page)
    kv = torch.randn((2, len(lens), max(lens), kv_heads, dim), generator=g, device="cuda").to(dtype)
    counts = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.append(0, seqs, kv[0], kv[1], counts)
    c.commit(seqs, counts)
    return c, seqs


def shifted(t):
    """The same values one element off the 16-byte boundary."""
    import torch
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.copy_(t.reshape(-1)).view(t.shape)


@pytest.mark.parametrize("nodes,group,dim,dtype", [
    (1, 1, 128, "bf16"), (1, 8, 64, "f16"), (5, 3, 80, "bf16"), (16, 8, 128, "bf16"), (17, 8, 96, "f16"),
    (50, 8, 72, "bf16"), (64, 4, 128, "f16"), (64, 2, 8, "bf16"), (3, 128, 128, "bf16"), (2, 256, 64, "bf16"), (64, 1, 64, "f16")])
def test_queries_by_boxes_and_by_copies(nodes, group, dim, dtype):
    """Aligned queries may come in boxes, others come by copies; the arithmetic after is one."""
    import torch
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float16
    c, seqs = filled(dim, 2, 16, [0, 7, 130, 300], dtype)
    g = torch.Generator("cuda").manual_seed(nodes * group)
    q = torch.randn((4, nodes, 2 * group, dim), generator=g, device="cuda").to(dtype)
    k, v = torch.randn((2, 4, nodes, 2, dim), generator=g, device="cuda").to(dtype)
    n_nodes = torch.tensor([nodes, max(nodes - 1, 1), nodes, 0], dtype=torch.int32, device="cuda")
    want, lse = c.tree_attention(0, seqs, q, k, v, n_nodes=n_nodes, want_lse=True)
    assert want.isfinite().all() and (want[3] == 0).all()
    for other in (shifted(q), q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([q, q], -1)[..., :dim]):
        out, l2 = c.tree_attention(0, seqs, other, k, v, n_nodes=n_nodes, want_lse=True)
        assert torch.equal(out, want) and torch.equal(l2, lse)
    # a negative scale is the queries' sign turned
    out = c.tree_attention(0, seqs, -q, k, v, n_nodes=n_nodes, scale=-(dim ** -0.5))
    assert torch.equal(out, want)
    assert c.device_status() == 0


@pytest.mark.parametrize("nodes,group", [(1, 4), (20, 4), (40, 8)])
def test_broadcast_queries(nodes, group):
    """Strides of 0: one query for all heads, for all nodes."""
    import torch
    c, seqs = filled(64, 2, 32, [5, 90], torch.bfloat16)
    g = torch.Generator("cuda").manual_seed(nodes)
    k, v = torch.randn((2, 2, nodes, 2, 64), generator=g, device="cuda").to(torch.bfloat16)
    for shape in ((2, nodes, 1, 64), (2, 1, 2 * group, 64), (1, nodes, 2 * group, 64)):
        q = torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16).expand(2, nodes, 2 * group, 64)
        assert torch.equal(c.tree_attention(0, seqs, q, k, v), c.tree_attention(0, seqs, q.contiguous(), k, v))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 64, 128, 256])
def test_page_sizes_agree(dim, page):
    """A page's box is joined or not, part of a tile or more than one: the result is that of pages of 32."""
    import torch
    lens = [1, 31, 129, 511, 700]
    g = torch.Generator("cuda").manual_seed(dim)
    q = torch.randn((5, 9, 8, dim), generator=g, device="cuda").to(torch.bfloat16)
    k, v = torch.randn((2, 5, 9, 2, dim), generator=g, device="cuda").to(torch.bfloat16)
    kv = torch.randn((2, 5, 700, 2, dim), generator=g, device="cuda").to(torch.bfloat16)

    def run(size):
        c, seqs = filled(dim, 2, size, lens, torch.bfloat16)
        c.truncate(seqs, torch.zeros(5, dtype=torch.int32, device="cuda"))
        counts = torch.tensor(lens, dtype=torch.int32, device="cuda")
        c.extend(seqs, counts + 9)
        c.append(0, seqs, kv[0], kv[1], counts)
        c.commit(seqs, counts)
        out = c.tree_attention(0, seqs, q, k, v, want_lse=True)
        assert c.device_status() == 0
        return out

    want, got = run(32), run(page)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
