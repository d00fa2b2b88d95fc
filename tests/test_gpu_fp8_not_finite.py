"""Rows with an infinity or a NaN through feed-forwards and layers of experts: NaN in their results, whatever the unit, and nothing in the others'."""
import pytest
import torch

import plain_fp8 as plain
from test_gpu_fp8 import DEV, _gen, _normal, _picks, _weight

pytestmark = pytest.mark.gpu
ACTS = ["silu", "gelu_tanh", ("swish_clamp", 7.0)]


def _spoiled(x):
    """x with values that are not finite in its first, middle and last row, and which rows those are."""
    M, K = x.shape
    y, at = x.clone(), sorted({0, M // 2, M - 1})
    for row, (k, v) in zip(at, ((3, float("inf")), (K - 1, float("nan")), (K // 2, float("-inf")))):
        y[row, k] = v
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[at] = False
    return y, keep


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 2, 8, 40, 64, 65, 200])
def test_feed_forwards(M, act):
    from sharpinference_amd import ops
    g = _gen(M)
    x = _normal(g, M, 300).bfloat16()
    (_, p1), (_, p2) = _weight(g, 2 * 130, 300, gated=True), _weight(g, 50, 130)
    clean = ops.feed_forward_fp8(x, p1, p2, plain.code(act))
    bad, keep = _spoiled(x)
    for rows in (bad, ops.quantize_rows(bad)):
        y = ops.feed_forward_fp8(rows, p1, p2, plain.code(act))
        assert torch.equal(y[keep], clean[keep]) and y[~keep].isnan().all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("on_input", [False, True])
@pytest.mark.parametrize("T", [1, 2, 16, 17, 300])
def test_layers_of_experts(T, on_input, act):
    from sharpinference_amd import ops
    g = _gen(T)
    E = 4
    x = _normal(g, T, 256).bfloat16()
    p1, p2 = ops.quantize_weight(_normal(g, E + 1, 2 * 100, 256, scale=0.05), True), ops.quantize_weight(_normal(g, E + 1, 50, 100))
    ids, wts = _picks(g, T, E, 2)
    call = lambda v: ops.experts_fp8(v, ids, wts, p1, p2, plain.code(act), on_input, True)
    clean = call(x)
    bad, keep = _spoiled(x)
    y = call(bad)
    assert torch.equal(y[keep], clean[keep]) and y[~keep].isnan().all()
