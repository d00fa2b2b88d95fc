"""Engines that two threads load side by side: each has the feed-forwards it asked for."""
import threading

import torch

from sharpinference_amd import ops
from sharpinference_amd.parts.feedforward import DenseSwiGLU
from test_fp8_loading_cpu import Source


def test_threads_have_a_switch_each(monkeypatch):
    """One loads in 8 bits, the other sets and clears its own switch in the middle of it."""
    monkeypatch.setattr(ops, "quantize_weight", lambda w, gated=False: ("8 bits", tuple(w.shape)))
    began, changed = threading.Event(), threading.Event()
    tensors = {"gate_proj.weight": torch.zeros(8, 16, dtype=torch.bfloat16), "up_proj.weight": torch.zeros(8, 16, dtype=torch.bfloat16),
               "down_proj.weight": torch.zeros(16, 8, dtype=torch.bfloat16)}

    class Slow(Source):
        def get(self, name):
            began.set()
            assert changed.wait(20)
            return super().get(name)

    def other():
        assert began.wait(20)
        seen.append(ops.feed_forwards_are_8_bits())
        ops.feed_forwards_in_8_bits(True)
        seen.append(ops.feed_forwards_are_8_bits())
        ops.feed_forwards_in_8_bits(False)
        changed.set()
    seen, part = [], DenseSwiGLU(16, 8)
    thread = threading.Thread(target=other)
    thread.start()
    ops.feed_forwards_in_8_bits(True)
    try:
        part.load("", Slow(tensors))
        assert ops.feed_forwards_are_8_bits()
    finally:
        ops.feed_forwards_in_8_bits(False)
        changed.set()
        thread.join()
    assert seen == [False, True] and part.w_gate_up == ("8 bits", (16, 16)) and part.w_down == ("8 bits", (16, 8))
