"""Layers of gated experts that 8 bits do not take, loaded where feed-forwards are wanted in 8 bits: all of the layer stays as it is."""
import pytest
import torch

from sharpinference_amd import ops
from sharpinference_amd.parts.feedforward import MoESwiGLU


class Source:
    def __init__(self, tensors):
        self.tensors = tensors

    def get(self, name):
        return self.tensors[name].clone()


def layer(experts, identity, hidden, inter, shared, device="cpu"):
    """(layer to be loaded, its tensors)"""
    part = MoESwiGLU(hidden, experts, 2, inter, shared_intermediate=shared, gate="softmax", score_on_input=False, identity=identity)
    g = torch.Generator().manual_seed(experts)
    specs = part.param_specs("m.")
    return part, Source({n: (torch.randn(s.shape, generator=g) * 0.2).bfloat16().to(device) for n, s in specs.items()})


def load(part, source, in_8_bits):
    ops.feed_forwards_in_8_bits(in_8_bits)
    try:
        part.load("m.", source)
    finally:
        ops.feed_forwards_in_8_bits(False)
    return part


def matrices(part):
    return [ops.unpack_weight(w) if isinstance(w, ops.PackedWeight) else w
            for w in (part.w_gate_up, part.w_down, part.shared.w_gate_up, part.shared.w_down)]


@pytest.mark.parametrize("experts,identity", [(1024, 0), (6, 2), (1022, 2)])
@pytest.mark.parametrize("hidden,inter,shared", [(16, 8, 8), (16, 8, 24), (128, 128, 128)])
def test_the_shared_expert_stays_with_its_layer(experts, identity, hidden, inter, shared):
    if experts > 100 and hidden == 128:
        experts, identity = 5, 1
    (a, source), (b, _) = (layer(experts, identity, hidden, inter, shared) for _ in range(2))
    load(a, source, True)
    load(b, source, False)
    assert a.merged == b.merged == (shared == inter)
    for x, y in zip(matrices(a), matrices(b)):
        assert x.dtype == torch.bfloat16 and torch.equal(x, y)


def test_experts_in_32_bits_keep_their_shared_expert():
    part, source = layer(4, 0, 16, 8, 8)
    source.tensors = {n: t if "shared" in n else t.float() for n, t in source.tensors.items()}
    load(part, source, True)
    assert part.w_gate_up.dtype == torch.float32 and part.shared.w_gate_up.dtype == torch.bfloat16 and not part.merged
