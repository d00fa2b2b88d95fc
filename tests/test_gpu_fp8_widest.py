"""Products of the widest rows that 8-bit floating point takes."""
import pytest
import torch

from test_gpu_fp8 import DEV, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile", [None, (192, 2, 1), (64, 2, 3)])
def test_products_of_the_widest_rows(monkeypatch, tile):
    """Whole numbers -1, 0, 1: every sum is exact."""
    from sharpinference_amd import ops
    from sharpinference_amd.ops import fp8
    M, N, K = 256, 3, fp8.FP8_MOST_K
    g = _gen(M, N)
    x = torch.randint(-1, 2, (M, K), generator=g, device=DEV, dtype=torch.int8).bfloat16()
    w = torch.randint(-1, 2, (N, K), generator=g, device=DEV, dtype=torch.int8).bfloat16()
    want = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    for k in range(0, K, 1 << 20):
        want += x[:, k:k + (1 << 20)].double() @ w[:, k:k + (1 << 20)].double().T
    p = ops.quantize_weight(w)
    if tile is not None:
        monkeypatch.setattr(fp8, "tile_fp8", lambda *a: tile)
    assert torch.equal(ops.linear_fp8(x, p), want.to(torch.bfloat16))
    if tile is None:
        with pytest.raises(ops.KernelError):
            monkeypatch.setattr(fp8, "tile_fp8", lambda *a: (256, 2, 1))
            ops.linear_fp8(x, p)
