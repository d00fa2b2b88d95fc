"""Gated values near a border of two codes, which tiles compute again in float: how many of them a tile holds, and which rows lie beside, changes nothing."""
import functools
import math

import pytest
import torch

import plain_fp8 as plain
from test_gpu_fp8 import DEV, _gen, _layer, _normal, _picks

pytestmark = pytest.mark.gpu
ROWS, K, I = 32, 640, 65536


def _codes(q, rows, p, width, k, height, act=(1, 0.0)):
    """Codes (as bytes) and scale bytes of the gated first product of these rows of q, in tiles of so many rows."""
    from sharpinference_amd import ops
    U, M = -(-width // 128), len(rows)
    x, s = q.codes.view(torch.uint8)[rows].contiguous(), q.scales[rows].contiguous()
    codes, scales = torch.empty(M, U * 128, dtype=torch.uint8, device=DEV), torch.empty(M, -(-U // 4) * 4, dtype=torch.uint8, device=DEV)
    ops._run("sharpi_fp8_tiles_gated", x.data_ptr(), s.data_ptr(), M, p.codes.data_ptr(), p.scales.data_ptr(), p.stored_rows, codes.data_ptr(), scales.data_ptr(),
             M, width, k, None, None, 1, 0, None, *act, height, ops._stream())
    return codes, scales[:, :U]


@functools.lru_cache(maxsize=1)
def _case():
    """Rows of unlike channels through a wide matrix, and the codes of each row in a call of its own."""
    from sharpinference_amd import ops
    g = _gen(K, I)
    x = (_normal(g, ROWS, K) * torch.exp(0.7 * _normal(g, K))).bfloat16()
    w = _normal(g, 2 * I, K, scale=0.05)
    p, q = ops.quantize_weight(w, True), ops.quantize_rows(x)
    alone = [_codes(q, [i], p, I, K, 64) for i in range(ROWS)]
    return x, w, p, q, torch.cat([c for c, _ in alone]), torch.cat([s for _, s in alone])


@pytest.mark.parametrize("height,times", [(256, 256), (128, 128), (192, 160), (64, 64), (256, 2)])
def test_a_row_has_its_codes_wherever_it_stands(height, times):
    """Alone, again and again (a column near a border is so in each of a tile's rows: hundreds of values), and beside others: the same codes."""
    x, w, p, q, alone, alone_scales = _case()
    codes, scales = _codes(q, list(range(ROWS)), p, I, K, height)
    assert torch.equal(codes, alone) and torch.equal(scales, alone_scales)
    many = torch.arange(ROWS, device=DEV).repeat_interleave(times)
    codes, scales = _codes(q, many, p, I, K, height)
    assert torch.equal(codes.view(ROWS, times, -1), alone[:, None].expand(-1, times, -1))
    assert torch.equal(scales.reshape(ROWS, times, -1), alone_scales[:, None].expand(-1, times, -1))


@pytest.mark.parametrize("times", [1, 256])
def test_large_values_have_the_definitions_codes_however_often_a_row_comes(times):
    """As for rows that differ: of values of half of their block's largest and more, of which there are one in 50, 2e-4 lie on a border's wrong side before they are
    computed again (8 of the 2 million here), and 1.4 % of these stay: 0.1, and more than 2 do not happen."""
    x, w, p, q, _, _ = _case()
    codes, scales = _codes(q, torch.arange(ROWS, device=DEV).repeat_interleave(times), p, I, K, 256)
    codes, scales = codes.view(ROWS, times, -1)[:, times // 2], scales.reshape(ROWS, times, -1)[:, times // 2]
    y = plain.rows(x) @ plain.rows(w).T
    h = plain.unit("silu", y[:, :I], y[:, I:]).to(torch.bfloat16)
    want, e = plain.quantised(h)
    same = (scales.int() - 127 == e.int()).repeat_interleave(128, 1)
    size = h.double().abs().view(ROWS, -1, 128)
    large = (size >= size.amax(2, keepdim=True) / 2).view(ROWS, -1) & (want != 0)
    assert int(large.sum()) > ROWS * I // 200
    assert int(((codes.view(torch.float8_e4m3fn).double() != want) & large & same).sum()) <= 2


def _limit(h):
    """The limit at which a unit whose gate and up columns both lie beyond it gives h."""
    low, high = 1.0, 20.0
    for _ in range(80):
        mid = (low + high) / 2
        low, high = (mid, high) if mid / (1 + math.exp(-1.702 * mid)) * (mid + 1) < h else (low, mid)
    return low


@pytest.mark.parametrize("height,rows", [(64, 64), (128, 128), (192, 192), (256, 256), (256, 300), (128, 70)])
@pytest.mark.parametrize("border", [11.53125, 11.46875])
@pytest.mark.parametrize("side", [1 - 5e-5, 1 + 5e-5])
def test_a_tile_of_nothing_but_one_value_near_a_border(border, side, height, rows):
    """Every gate and every up column at the unit's limit: all of a tile's values are one number, 5e-5 of it from where bfloat16 rounds to the tie of two codes, in
    every row and column.  (The unit is within 2^-19 (1 + |g|) = 1e-5 of the number, so both round alike.)"""
    from sharpinference_amd import ops
    width, limit = 300, _limit(border * side)
    p, q = ops.quantize_weight(torch.ones(2 * width, 128, device=DEV), True), ops.quantize_rows(torch.ones(rows, 128, device=DEV))
    codes, scales = _codes(q, list(range(rows)), p, width, 128, height, (ops.ACT_SWISH_CLAMP, limit))
    both = torch.full((1, width), 128.0, dtype=torch.float64, device=DEV)
    want, e = plain.quantised(plain.unit(("swish_clamp", limit), both, both).to(torch.bfloat16))
    assert (codes.view(torch.float8_e4m3fn).double() == want).all() and (scales.int() - 127 == e).all()


@pytest.mark.parametrize("T,E,k", [(700, 3, 2), (400, 8, 2)])
def test_equal_tokens_of_a_layer_have_equal_results(T, E, k):
    """Five tokens again and again, sorted by expert in whatever order."""
    from sharpinference_amd import ops
    g = _gen(T, E, k)
    _, w2, _, p2 = _layer(g, E, 384, 2000, 140, True)
    p1 = ops.quantize_weight(_normal(g, E + 1, 4000, 384, scale=0.05), True)
    five, (ids, wts) = _normal(g, 5, 384).bfloat16(), _picks(g, 5, E, k)
    which = torch.randint(0, 5, (T,), generator=g, device=DEV)
    y = ops.experts_fp8(five[which], ids[which], wts[which], p1, p2, shared=True)
    for i in range(5):
        mine = y[which == i]
        assert (mine == mine[0]).all()
    for _ in range(5):
        assert torch.equal(ops.experts_fp8(five[which], ids[which], wts[which], p1, p2, shared=True), y)
