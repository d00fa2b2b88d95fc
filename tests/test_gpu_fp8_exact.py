"""8-bit products where every value counts: whole numbers, whose products and sums are exact, in every kind of tile and over every kind of k; and how far
random values are off on the whole, beside the bound of each."""
import pytest
import torch

import plain_fp8 as plain
from test_gpu_fp8 import DEV, FEED, LINEAR, _gen, _layer, _normal, _picks, _weight, _whole

pytestmark = pytest.mark.gpu
TILES = [(64, 2, 1), (64, 2, 3), (128, 2, 1), (128, 2, 2), (192, 1, 1), (192, 1, 4), (192, 2, 1), (192, 2, 2), (256, 1, 1), (256, 1, 3), (256, 2, 1), (256, 2, 4)]


def _product(M, N, K):
    """Whole numbers up to 4, blocks of 128 of k in scales of their own: sums below 2^24 of equal steps."""
    from sharpinference_amd import ops
    g = _gen(M, N, K)
    x, w = _whole(g, M, K), _whole(g, N, K)
    for b in range(-(-K // 128)):
        at, p = slice(128 * b, 128 * b + 128), 2.0 ** (7 * b % 11)
        x[:, at] *= p
        w[:, at] /= p
    # every k has a value somewhere, and the last one in every row
    x[:, -1], w[:, -1] = x[:, -1].sign() + 3 * (x[:, -1] == 0), 1.0
    return x, ops.quantize_weight(w), (plain.rows(x) @ plain.rows(w).T)


@pytest.mark.parametrize("M,N,K", [(70, 513, 2048), (100, 96, 1153), (300, 259, 895), (257, 128, 5121), (193, 40, 129)])
@pytest.mark.parametrize("tile", TILES)
def test_whole_numbers_in_every_kind_of_tile(monkeypatch, M, N, K, tile):
    from sharpinference_amd import ops
    from sharpinference_amd.ops import fp8
    x, p, want = _product(M, N, K)
    monkeypatch.setattr(fp8, "tile_fp8", lambda *a: (*tile[:2], min(tile[2], -(-K // 128))))
    assert torch.equal(ops.linear_fp8(x, p), want.to(torch.bfloat16))


@pytest.mark.parametrize("M", [1, 2, 3, 16, 17, 33, 64, 65, 129])
@pytest.mark.parametrize("N,K", [(5, 1), (33, 127), (100, 129), (40, 1023), (4700, 1025), (70, 2175)])
def test_whole_numbers_of_few_rows_and_more(M, N, K):
    from sharpinference_amd import ops
    x, p, want = _product(M, N, K)
    assert torch.equal(ops.linear_fp8(x, p), want.to(torch.bfloat16))
    assert torch.equal(ops.linear_fp8(x.bfloat16(), p), want.to(torch.bfloat16))


def _off(y, want):
    return float((y.double() - want).norm() / want.norm())


# bfloat16's rounding alone: evenly spread over half a step, which is 2^-8 of a value at most.  What the matrix instruction cuts: of eight products on end seven lose up to 2^-13 of the
# largest, some three times their rms, without a sign in common: sqrt(7) 3 / sqrt(3) 2^-13 beside a sum of sqrt(8), below 2^-12.
STORED, CUT = 2.0 ** -8 / 3 ** 0.5, 2.0 ** -12


@pytest.mark.parametrize("M,N,K", [c for c in LINEAR if c[0] * c[1] >= 2000])
def test_products_are_off_by_their_rounding(M, N, K):
    from sharpinference_amd import ops
    g = _gen(M, N, K)
    x = (_normal(g, M, K) * torch.exp(_normal(g, M, 1))).bfloat16()
    w, p = _weight(g, N, K)
    assert _off(ops.linear_fp8(x, p), plain.rows(x) @ plain.rows(w).T) <= STORED + CUT


@pytest.mark.parametrize("M,K,I", [c for c in FEED if c[0] * c[1] >= 2000])
def test_feed_forwards_are_off_by_their_rounding(M, K, I):
    """The first product is exact; a value of h that float steps move across a border moves by a code's step, 2^-3 of it at most.  The chance for a border of
    bfloat16, with |g| about 1: 2 (1 + |g|) 2^-19 / 2^-8 = 2^-9, and one in 2^4 of these is a code's border too: 2^-3 sqrt(2^-9) = 0.0055, a quarter of it."""
    from sharpinference_amd import ops
    g = _gen(M, K, I)
    x = _whole(g, M, K).bfloat16()
    w1 = _whole(g, 2 * I, K) / 64
    w2, p2 = _weight(g, K + 3, I)
    want, _ = plain.feed_forward(x.double(), w1.double(), plain.rows(w2), "silu")
    assert _off(ops.feed_forward_fp8(x, ops.quantize_weight(w1, True), p2), want) <= STORED + CUT + 0.0055 / 4


@pytest.mark.parametrize("T,E,k,K,I,N,shared", [(5, 100, 6, 300, 70, 257, False), (16, 16, 1, 256, 200, 128, True), (64, 8, 2, 300, 70, 96, True), (300, 8, 2, 300, 260, 140, False),
                                                (700, 3, 1, 256, 390, 300, True)])
def test_layers_are_off_by_their_rounding(T, E, k, K, I, N, shared):
    from sharpinference_amd import ops
    g = _gen(T, E, k, K, I, N)
    x = _whole(g, T, K).bfloat16()
    w1, w2, p1, p2 = _layer(g, E, K, I, N, shared)
    ids, wts = _picks(g, T, E, k)
    want = torch.zeros(T, N, dtype=torch.float64, device=DEV)
    for e in range(E + (1 if shared else 0)):
        at, pick = torch.nonzero(ids == e, as_tuple=True) if e < E else (torch.arange(T, device=DEV), None)
        if at.numel():
            y, _ = plain.feed_forward(x[at].double(), w1[e].double(), plain.rows(w2[e]), "silu")
            want.index_add_(0, at, y if pick is None else y * wts[at, pick, None].double())
    assert _off(ops.experts_fp8(x, ids, wts, p1, p2, shared=shared), want) <= STORED + CUT + 0.0055 / 4
