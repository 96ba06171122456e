"""Operands of the row operators and the quantised products in layouts other than contiguous ones, on the GPU: taken
for what they are, or refused."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew
from hummingbird_amd import projection as pr

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


def test_one_token_of_each_sequence():
    """(B, 1, C) slices through every row operator and both products: as their contiguous copies."""
    announce("one token of each sequence")
    gen = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn(3, 5, 256, device=DEV, generator=gen).to(torch.bfloat16)
    w = torch.rand(128, device=DEV, generator=gen)
    x, h = wide[:, -1:, :128], wide[:, 1:2, 128:]
    xc, hc = x.contiguous(), h.contiguous()
    codes, scales = pr.quantize_q4(torch.randn(48, 128, device=DEV, generator=gen))
    weight, ws = ew.quantize_rows(torch.randn(48, 128, device=DEV, generator=gen))
    q, _ = ew.quantize_rows(wide)

    def equal(got, ref):
        for a, b in zip(got, ref):
            assert a.shape == b.shape and torch.equal(a.float(), b.float())
    equal(ew.quantize_rows(x), ew.quantize_rows(xc))
    equal(ew.rms_modulate_q8(x, w, 1e-5), ew.rms_modulate_q8(xc, w, 1e-5))
    equal(ew.residual_rms_q8(h, x, w, 1e-5), ew.residual_rms_q8(hc, xc, w, 1e-5))
    equal(ew.glu_q8(wide[:, 3:4]), ew.glu_q8(wide[:, 3:4].contiguous()))
    equal([pr.linear_q4(x, codes, scales)], [pr.linear_q4(xc, codes, scales)])
    token = q[:, -1:, :128]
    sx = torch.rand(3, 1, device=DEV, generator=gen)
    equal([pr.linear_q8(token, sx, weight, ws)], [pr.linear_q8(token.contiguous(), sx, weight, ws)])
    equal([ew.rms_modulate(x, w, 1e-5), ew.gated_residual(h, x)], [ew.rms_modulate(xc, w, 1e-5), ew.gated_residual(hc, xc)])


def test_operands_on_the_host_are_refused():
    """A host tensor's address means nothing to a kernel: every operand that goes to it as it is has to be on the rows'
    device. (Parameters that the wrappers convert, such as norm weights, are moved.)"""
    announce("host operands")
    h = torch.zeros(2, 3, 256, device=DEV, dtype=torch.bfloat16)
    w, host = torch.ones(256, device=DEV), torch.zeros(2, 256, dtype=torch.bfloat16)
    for call in (lambda: ew.rms_modulate(h, w, 1e-5, host, host), lambda: ew.gated_residual(h, h, gate=host),
                 lambda: ew.gated_residual(h, h.cpu()), lambda: ew.residual_rms(h, h.cpu(), w, 1e-5),
                 lambda: ew.residual_rms(h, h, w, 1e-5, gate=host), lambda: ew.residual_dyt(h, h.cpu()),
                 lambda: ew.residual_rms(h, h, w, 1e-5, scale=host, shift=host),
                 lambda: ew.rms_modulate_q8(h, w, 1e-5, host, host), lambda: ew.residual_rms_q8(h, h, w, 1e-5, gate=host),
                 lambda: ew.residual_rms_q8(h, h.cpu(), w, 1e-5), lambda: ew.residual_rms_q8(h, h, w, 1e-5, local=host[0]),
                 lambda: pr.residual_linear(h, torch.zeros(256, 256, dtype=torch.bfloat16, device=DEV), None, h.cpu())):
        with pytest.raises(ValueError):
            call()


def test_linear_q8_takes_the_scales_of_a_slice():
    """The rows, their scales and the features of slices: (B, L) scales' last tokens lie L apart."""
    announce("scales of slices")
    gen = torch.Generator(device=DEV).manual_seed(2)
    q, s = ew.quantize_rows(torch.randn(3, 5, 64, device=DEV, generator=gen))
    w, ws = ew.quantize_rows(torch.randn(40, 64, device=DEV, generator=gen))
    whole = pr.linear_q8(q, s, w, ws)
    assert torch.equal(pr.linear_q8(q[:, -1:], s[:, -1:], w, ws), whole[:, -1:])
    assert torch.equal(pr.linear_q8(q[:, 2], s[:, 2], w, ws), whole[:, 2])
    assert torch.equal(pr.linear_q8(q, s, w[::2], ws[::2]), whole[..., ::2])
    assert torch.equal(pr.linear_q8(q[:1], s[:1, 0, None].expand(1, 5) * 0 + s[:1], w, ws), whole[:1])
    for bad in (s[:, :, None], s[:, 1:], s[0]):
        with pytest.raises(ValueError, match="x_scale"):
            pr.linear_q8(q, bad, w, ws)
