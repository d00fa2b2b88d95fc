"""8-bit operands that are refused before anything is allocated or launched: sizes beyond the format's, matrices whose parts do not fit."""
import pytest
import torch

from sharpinference_amd import ops
from sharpinference_amd.ops import fp8


def test_matrices_beyond_the_largest():
    for shape in ((2, 1 << 24), (1 << 31, 128), (4, 2, 1 << 24)):
        with pytest.raises(ops.KernelError, match="columns|too large"):
            ops.empty_fp8_weight(shape, False, "cpu")


def test_matrices_of_the_host_are_not_quantised():
    with pytest.raises(ops.KernelError, match="live on the GPU"):
        ops.quantize_into(ops.empty_fp8_weight((4, 128), False, "cpu"), torch.zeros(4, 128))


@pytest.mark.parametrize("gated", [False, True])
def test_a_matrix_of_parts_that_do_not_fit(gated):
    w = ops.empty_fp8_weight((3, 66, 300), gated, "cpu")
    again = ops.Fp8Weight(w.codes, w.scales, w.shape, gated)
    assert again.stored_rows == (128 if gated else 96) and again.select(2).shape == (66, 300)
    for codes, scales, shape in ((w.codes[:2], w.scales, w.shape), (w.codes, w.scales[:, :1], w.shape), (w.codes, w.scales, (3, 200, 300)), (w.codes, w.scales, (3, 66, 400)),
                                 (w.codes.int(), w.scales, w.shape), (w.codes[..., ::2], w.scales, w.shape), (w.codes, w.scales, (66, 300))):
        with pytest.raises(ops.KernelError, match="not those of"):
            ops.Fp8Weight(codes, scales, shape, gated)


def test_limits_are_those_of_the_kernels():
    import pathlib
    import re
    csrc = pathlib.Path(fp8.__file__).parents[1] / "csrc"
    found = dict(re.findall(r"constexpr int (\w+) = ([\d <*]+);", (csrc / "fp8_few.hip").read_text() + (csrc / "fp8.h").read_text()))
    value = {k: eval(v) for k, v in found.items()}
    assert value["kFewRows"] == fp8.FP8_FEW_ROWS and value["kFewPairs"] == fp8.FP8_FEW_PAIRS and value["kFewExperts"] >= fp8.FP8_MAX_EXPERTS + 1
    assert value["kStagedRows"] == fp8.FP8_STAGED_ROWS and value["kStagedMost"] == fp8.FP8_STAGED_BYTES
    assert 16 * value["kLayerTiles"] == fp8.FP8_LAYER_COLUMNS and value["kF8MostK"] - 1 == fp8.FP8_MOST_K
