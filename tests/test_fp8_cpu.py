"""8-bit operators without a GPU: the stored order, what is refused before anything is launched, and the rules that choose tiles."""
import pytest
import torch

from sharpinference_amd import ops
from sharpinference_amd.ops import fp8

F8 = torch.float8_e4m3fn


def _stored(N, K, gated=False, lead=()):
    g = torch.Generator().manual_seed(N * 7 + K)
    codes = (torch.randn(*lead, N, K, generator=g) * 100).clamp(-448, 448).to(F8)
    scales = torch.randint(100, 140, (*lead, N, -(-K // 128)), generator=g).to(torch.uint8)
    return codes, scales, ops.fp8_weight(codes, scales, gated)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K,lead", [(2, 1, ()), (32, 128, ()), (34, 129, ()), (70, 1000, ()), (66, 300, (3,)), (128, 640, (2,))])
def test_stored_matrices_give_their_values_back(N, K, lead, gated):
    codes, scales, w = _stored(N, K, gated, lead)
    blocks = scales.shape[-1]
    powers = (scales.int() << 23).view(torch.float32).repeat_interleave(128, -1)[..., :K]
    assert w.shape == (*lead, N, K) and torch.equal(w.values(), codes.float() * powers)
    assert w.codes.shape[-2:] == (blocks, 4096) and w.codes.shape[-3] * 32 == w.stored_rows and w.stored_rows % (64 if gated else 32) == 0
    if lead:
        assert torch.equal(w.select(1).values(), w.values()[1])


def test_a_tile_lies_in_the_operands_order():
    """Byte k of row r of a tile's block is at [k / 64][k / 16 % 2][k / 32 % 2][r][k % 16]."""
    codes, _, w = _stored(64, 256)
    raw = codes.view(torch.uint8)
    for row, k in [(0, 0), (5, 17), (33, 200), (63, 255), (31, 96)]:
        at = (k % 128 // 64) * 2048 + (k // 16 % 2) * 1024 + (k // 32 % 2) * 512 + (row % 32) * 16 + k % 16
        assert w.codes[row // 32, k // 128, at] == raw[row, k]


def _refused(what, f, *a, **kw):
    with pytest.raises(ops.KernelError, match=what):
        f(*a, **kw)


def test_matrices_that_are_refused():
    codes, scales, w = _stored(4, 130)
    _refused("float8_e4m3fn", ops.fp8_weight, codes.float(), scales)
    _refused("float8_e4m3fn", ops.fp8_weight, codes[0], scales[0])
    _refused("scales must be uint8", ops.fp8_weight, codes, scales[:, :1])
    _refused("scales must be uint8", ops.fp8_weight, codes, scales.int())
    _refused("as many up rows", ops.fp8_weight, codes[:3], scales[:3], True)
    _refused("on the GPU", ops.quantize_weight, torch.zeros(4, 4))
    _refused("at most 1024", ops.empty_fp8_weight, (1025, 4, 4), False, "cpu")
    _refused(r"must be \[N, K\]", ops.empty_fp8_weight, (4,), False, "cpu")
    _refused("destination", ops.quantize_into, w, torch.zeros(4, 131))


def test_rows_that_are_refused():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    _refused("live on the GPU", ops.quantize_rows, x)
    _refused("whole blocks", ops.Fp8Rows, torch.zeros(2, 100).to(F8), torch.zeros(2, 4, dtype=torch.uint8), 100)
    _refused("multiple of 4", ops.Fp8Rows, torch.zeros(2, 128).to(F8), torch.zeros(2, 1, dtype=torch.uint8), 100)


def test_calls_that_are_refused():
    _, _, plain = _stored(4, 128)
    _, _, gated = _stored(8, 128, True)
    _, _, down = _stored(128, 4)
    stack = _stored(8, 128, True, (3,))[2]
    downs = _stored(128, 4, False, (3,))[2]
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    ids, wts = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1)
    _refused("not gated", ops.linear_fp8, x, gated)
    _refused("Fp8Weight", ops.linear_fp8, x, torch.zeros(4, 128))
    _refused("live on the GPU", ops.linear_fp8, x, plain)
    _refused("gated Fp8Weight", ops.feed_forward_fp8, x, plain, down)
    _refused("gated Fp8Weight", ops.feed_forward_fp8, x, stack, downs)
    _refused("do not fit", ops.feed_forward_fp8, x, gated, _stored(128, 5)[2])
    _refused("live on the GPU", ops.feed_forward_fp8, x, gated, down)
    _refused("gated Fp8Weight", ops.experts_fp8, x, ids, wts, gated, down)
    _refused("do not fit", ops.experts_fp8, x, ids, wts, stack, _stored(128, 4, False, (2,))[2])
    _refused("live on the GPU", ops.experts_fp8, x, ids, wts, stack, downs)


def test_an_engine_of_unknown_or_contradicting_kind():
    from sharpinference_amd.engine import Engine
    with pytest.raises(ValueError, match="not known"):
        Engine("nowhere", feed_forward="int4")
    with pytest.raises(ValueError, match="bfloat16 engine"):
        Engine("nowhere", dtype="float32", feed_forward="fp8")


def test_the_switch_is_read_where_weights_are_loaded():
    assert not ops.feed_forwards_are_8_bits()
    ops.feed_forwards_in_8_bits(True)
    try:
        assert ops.feed_forwards_are_8_bits()
    finally:
        ops.feed_forwards_in_8_bits(False)


@pytest.mark.parametrize("M", [1, 17, 65, 128, 300, 1000, 2048, 8192, 100000])
@pytest.mark.parametrize("N,K", [(1, 1), (249, 8154), (1024, 2048), (7168, 5120), (28672, 5120), (4096, 14336)])
def test_tiles_are_of_the_compiled_kinds(M, N, K):
    for gated in (False, True):
        height, nt, shares = fp8.tile_fp8(M, N, K, gated, 256)
        assert height in (64, 128, 192, 256) and nt in (1, 2) and (nt == 2 or (height > 128 and not gated))
        assert 1 <= shares <= max(1, -(-K // 128)) and (shares == 1 or not gated)


def test_which_rows_stream_the_weights():
    assert fp8.few_rows_fp8(16, 1 << 20) and fp8.few_rows_fp8(64, 12288) and not fp8.few_rows_fp8(17, 65536) and not fp8.few_rows_fp8(65, 8)


def test_shares_of_the_sum():
    for tiles in (1, 3, 64, 160, 2000):
        for blocks in (1, 7, 8, 100, 10000):
            s = fp8.sum_shares(tiles, blocks, 256)
            assert 1 <= s <= max(1, blocks // 8) and (s == 1 or s * tiles <= 512)
