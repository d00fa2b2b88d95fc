"""Steps through layers that 8 bits do not take, loaded where feed-forwards are wanted in 8 bits: what they give otherwise."""
import pytest
import torch

from test_fp8_loading_cpu import layer, load
from test_gpu_parts import DEV, _ctx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,identity", [(1024, 0), (6, 2)])
@pytest.mark.parametrize("hidden,inter,shared", [(128, 128, 128), (64, 32, 32), (128, 128, 64)])
def test_layers_give_what_they_do_otherwise(experts, identity, hidden, inter, shared):
    (a, source), (b, _) = (layer(experts, identity, hidden, inter, shared, DEV) for _ in range(2))
    load(a, source, True)
    load(b, source, False)
    for T in (1, 9, 40, 200):
        x = torch.randn(T, hidden, generator=torch.Generator().manual_seed(T)).bfloat16().to(DEV)
        y, z = (p.forward(x, _ctx([(0, T)], dtype=torch.bfloat16)[0]).tensor() for p in (a, b))
        assert y.isfinite().all() and torch.equal(y, z)
