"""Weights whose scales lie at the ends of the format's range, beside rows whose scales make up for it: few rows and many give the numbers that the products are."""
import pytest
import torch

import plain_fp8 as plain
from test_gpu_fp8 import DEV, F8, _gen, _whole

pytestmark = pytest.mark.gpu
# a block's weight byte, and the power of two of its codes (whole numbers up to 4 times that): ordinary ones and both ends
BLOCKS = [(127, 0), (247, 0), (241, 6), (180, 3), (8, -7), (1, -4), (60, -7)]
K = 128 * len(BLOCKS)


def _operands(g, M, N):
    """x [M, K] bfloat16 and weights (values in 64 bits, codes, bytes) whose products are whole numbers times 2^-6: the rows' powers undo the weights'."""
    x, codes = _whole(g, M, K), _whole(g, N, K)
    scales = torch.empty(N, len(BLOCKS), dtype=torch.uint8, device=DEV)
    for b, (byte, power) in enumerate(BLOCKS):
        at = slice(128 * b, 128 * b + 128)
        codes[:, at] *= 2.0 ** power
        scales[:, b] = byte
        x[:, at] = (x[:, at].double() * 2.0 ** (127 - byte - power - 6)).float()
    codes = codes.to(F8)
    w = (codes.double().view(N, -1, 128) * plain.power(scales.int() - 127)[..., None]).view(N, K)
    assert x.isfinite().all() and (x.abs()[x != 0] >= 2.0 ** -126).all()
    return x.bfloat16(), w, codes, scales


@pytest.mark.parametrize("M", [1, 2, 5, 16, 40, 64, 65, 200, 300])
def test_products(M):
    from sharpinference_amd import ops
    x, w, codes, scales = _operands(_gen(M), M, 70)
    want = x.double() @ w.T
    assert (plain.rows(x) == x.double()).all() and want.abs().max() < 2 ** 12
    y = ops.linear_fp8(x, ops.fp8_weight(codes, scales))
    assert torch.equal(y, want.to(torch.bfloat16))
    assert torch.equal(ops.linear_fp8(ops.quantize_rows(x), ops.fp8_weight(codes, scales)), y)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", ("swish_clamp", 7.0)])
@pytest.mark.parametrize("M", [1, 2, 5, 16, 40, 64, 65, 200, 300])
def test_feed_forwards(M, act):
    from sharpinference_amd import ops
    g = _gen(M, 2)
    I = 200
    x, w1, codes, scales = _operands(g, M, 2 * I)
    p1 = ops.fp8_weight(codes, scales, gated=True)
    w2 = torch.randn(40, I, generator=g, device=DEV) * 0.02
    want, bound = plain.feed_forward(x.double(), w1, plain.rows(w2), act)
    for rows in (x, ops.quantize_rows(x)):
        y = ops.feed_forward_fp8(rows, p1, ops.quantize_weight(w2), plain.code(act))
        assert ((y.double() - want).abs() <= bound + plain.stored(want)).all()


@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 100])
def test_layers_of_experts(T):
    from sharpinference_amd import ops
    g = _gen(T, 3)
    E, I = 3, 96
    x, w1, codes, scales = _operands(g, T, (E + 1) * 2 * I)
    p1 = ops.fp8_weight(codes.view(E + 1, 2 * I, K), scales.view(E + 1, 2 * I, -1), gated=True)
    w2 = torch.randn(E + 1, 40, I, generator=g, device=DEV) * 0.02
    ids = torch.randint(0, E, (T, 1), generator=g, device=DEV).int()
    wts = torch.full((T, 1), 0.5, device=DEV)
    y = ops.experts_fp8(x, ids, wts, p1, ops.quantize_weight(w2), shared=True)
    w1 = w1.view(E + 1, 2 * I, K)
    for t in range(T):
        e = int(ids[t])
        a, da = plain.feed_forward(x[t:t + 1].double(), w1[e], plain.rows(w2[e]), "silu")
        b, db = plain.feed_forward(x[t:t + 1].double(), w1[E], plain.rows(w2[E]), "silu")
        want = 0.5 * a + b
        # (two sums in float: half a step of each)
        assert ((y[t:t + 1].double() - want).abs() <= 0.5 * da + db + 2.0 ** -23 * (a.abs() + b.abs()) + plain.stored(want)).all()
