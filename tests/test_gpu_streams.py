"""Results of calls that name a stream: no other stream's pending work may reach their memory."""
import pytest

pytestmark = pytest.mark.gpu


def busy(shapes_dtypes):
    """Work queued on the current stream that will write to memory given back already: blocks of these shapes are
    free for the current stream's next allocations, and are still to be written to."""
    import torch
    held = [torch.empty(s, dtype=d, device="cuda") for s, d in shapes_dtypes]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)  # about 0.1 s
    for t in held:
        t.fill_(77)


def both(call, outputs):
    """call(stream) on a side stream, as a torch stream and as an address, beside pending work of the current one."""
    import torch
    want = [t.clone() for t in call(None)]
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        torch.cuda.synchronize()
        busy(outputs * 3)
        got = call(stream)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_tree_attention(cuda_lib):
    import torch
    from tinygpt_b200 import PagedCache
    n, nodes = 64, 4
    c = PagedCache(1, 2, 64, 16, 2 * n, n, 2)
    c.k.normal_(), c.v.normal_()
    seqs, twelve = ints(range(n)), ints([12] * n)
    c.extend(seqs, ints([16] * n))
    c.commit(seqs, twelve)
    q = torch.randn((n, nodes, 8, 64), device="cuda").bfloat16()
    k, v = torch.randn((2, n, nodes, 2, 64), device="cuda").bfloat16()
    both(lambda s: c.tree_attention(0, seqs, q, k, v, want_lse=True, stream=s), [((n, nodes, 8, 64), torch.bfloat16), ((n, nodes, 8), torch.float32)])


def test_accept_and_masks(cuda_lib):
    import torch
    from tinygpt_b200 import PagedCache, tree_masks
    n, nodes = 2048, 8
    c = PagedCache(1, 1, 16, 8, n, n, 1)
    c.k.zero_(), c.v.zero_()
    seqs, eight, none = ints(range(n)), ints([8] * n), ints([0] * n)
    parents, tokens, ids = ints([[-1, 0, 0, 1, 2, 3, 3, 5]] * n), ints([[0, 1, 2, 3, 4, 5, 6, 7]] * n), ints([[1, 3, 0, 6, 0, 0, 9, 0]] * n)

    def call(s):
        torch.cuda.synchronize() if s is None else None
        c.truncate(seqs, none, stream=s)
        c.extend(seqs, eight, stream=s)
        return c.accept(seqs, parents, tokens, ids, stream=s)

    both(call, [((n, nodes), torch.int32), ((n,), torch.int32)])
    both(lambda s: [tree_masks(parents, stream=s)], [((n, nodes), torch.int64)])


def test_beam_select(cuda_lib):
    import torch
    from tinygpt_b200 import BeamSearch
    B, W, V = 256, 4, 2000
    h = BeamSearch(V, W, B)
    x, scores = torch.randn((B * W, V), device="cuda"), -torch.rand((B, W), device="cuda")
    history, length = torch.randint(0, V, (B * W, 16), device="cuda", dtype=torch.int32), ints([5] * (B * W))
    both(lambda s: h.select(x, scores, history=history, history_len=length, stream=s),
         [((B, W), torch.int32)] * 3 + [((B, W), torch.float32), ((B * W, 16), torch.int32), ((B * W,), torch.int32)])
