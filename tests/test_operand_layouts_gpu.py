"""Operands of the row operators and the quantised products in layouts other than contiguous ones, on the GPU: taken
for what they are, or refused."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew

pytestmark = pytest.mark.gpu
DEV = "cuda"


def announce(*what) -> None:
    print("\n[case]", *what, flush=True)


@pytest.mark.parametrize("operand", ["x_bias", "local"])
@pytest.mark.parametrize("op", ["gated_residual", "residual_rms", "residual_rms_q8"])
def test_channel_vectors_of_other_strides_are_refused(op, operand):
    announce("channel vectors", op, operand)
    h = torch.zeros(1, 2, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    wide = torch.arange(64 * 8, device=DEV, dtype=torch.float32).reshape(64, 8)
    column = wide[:, :1]

    def call(v):
        if op == "gated_residual":
            return ew.gated_residual(h, h, **{operand: v})
        return getattr(ew, op)(h, h, w, 1e-5, **{operand: v})[0]
    for bad in (column, wide[:, 0], torch.ones((), device=DEV), torch.ones(64)):
        with pytest.raises(ValueError, match=operand):
            call(bad)
    for good in (column.contiguous(), column[:, 0].contiguous(), column[:, 0].contiguous()[None]):
        assert torch.equal(call(good)[0, 1], wide[:, 0])


@pytest.mark.parametrize("op", ["gated_residual", "residual_rms", "residual_rms_q8"])
def test_memory_past_32_bits_is_past_the_end(op):
    announce("memory past 32 bits", op)
    h = torch.zeros(2, 4, 64, device=DEV)
    ones = torch.ones(64, device=DEV)

    def call(memory):
        if op == "gated_residual":
            return ew.gated_residual(h, h, local=ones, memory=memory)
        return getattr(ew, op)(h, h, ones, 1e-5, local=ones, memory=memory)[0]
    for memory in (4, 5, 1 << 31, 1 << 32, (1 << 32) + 2):
        assert (call(memory) == 0).all(), memory
    assert torch.equal(call(3)[:, :, 0], torch.tensor([[0.0, 0, 0, 1]] * 2, device=DEV))
    with pytest.raises(ValueError):
        call(-(1 << 32))
