"""The sampler's calls that name a stream: no other stream's pending work may reach their results."""
import pytest

from tests.test_gpu_streams import both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["device", "host"])
def test_sample(cuda_lib, where):
    import torch
    from tinygpt_b200 import Sampler, row_params
    from tinygpt_b200.sampler import params_to_device
    B, V = 1024, 3001
    s = Sampler(V, B)
    x = torch.randn((B, V), device="cuda")
    params = row_params(B, temperature=0.0)
    if where == "device":
        params = params_to_device(params, "cuda")
    both(lambda st: [s.sample(x, params, stream=st)[0]], [((B,), torch.int32)])


def test_spec_verify(cuda_lib):
    import torch
    from tinygpt_b200 import Sampler
    B, K, V = 64, 4, 1000
    s = Sampler(V, B)
    target, draft = torch.randn((B, K + 1, V), device="cuda"), torch.randn((B, K, V), device="cuda")
    ids = torch.randint(0, V, (B, K), dtype=torch.int32, device="cuda")
    temperature = torch.ones(B, device="cuda")
    u, w = torch.rand((B, K), device="cuda"), torch.rand(B, device="cuda")
    both(lambda st: s.spec_verify(target, draft, ids, temperature, u, w, stream=st), [((B, K + 1), torch.int32), ((B,), torch.int32)])
