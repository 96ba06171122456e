"""What the wrappers of the row operators make of their operands' shapes and strides, on the CPU (no kernel runs)."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import elementwise as ew


def test_channel_vectors_are_values_next_to_each_other():
    """A (C, 1) slice of a wider tensor has C values and a last stride of 1, and its values lie apart."""
    x = torch.zeros(2, 3, 16)
    wide = torch.arange(16 * 8, dtype=torch.float32).reshape(16, 8)
    for good in (torch.ones(16), torch.ones(1, 16), torch.ones(1, 1, 16), torch.ones(16, 1), wide[2:4].reshape(16)):
        assert ew._channel_vector(good, 16, x, "x_bias") == good.data_ptr()
    assert ew._channel_vector(None, 16, x, "x_bias") == 0
    for bad in (wide[:, :1], wide[:, 3], torch.ones(32)[::2], torch.ones(()), torch.ones(8), torch.ones(16).double(),
                torch.ones(16, device="meta")):
        with pytest.raises(ValueError, match="x_bias"):
            ew._channel_vector(bad, 16, x, "x_bias")


def test_memory_tokens_keep_their_meaning_past_32_bits():
    """Cut to the sequence's length, not to the low 32 bits of a C int."""
    for memory, held in ((0, 0), (3, 3), (4, 4), (5, 4), (1 << 31, 4), (1 << 32, 4), ((1 << 32) + 1, 4), (1 << 70, 4)):
        assert ew._memory_tokens(memory, 4) == held
    for memory in (-1, -(1 << 32), -(1 << 31) - 5):
        with pytest.raises(ValueError, match="memory"):
            ew._memory_tokens(memory, 4)


@pytest.mark.parametrize("rows,refused", [((1 << 31) - 1, False), (1 << 31, True), ((1 << 32) + 5, True)])
def test_row_counts_past_a_c_int_are_refused(rows, refused):
    """The features of a product go to the library as a C int: 2^32 + 5 of them would be taken for 5."""
    class Rows:
        is_cuda, shape = True, torch.Size((rows, 16))

        def dim(self):
            return 2

        def is_contiguous(self):
            return True

        def numel(self):
            return 16 * rows
    if refused:
        with pytest.raises(ValueError, match="2\\^31 rows"):
            ew._layout(Rows(), "weight")
    else:
        assert ew._layout(Rows(), "weight") == (rows, 16, 16)


def test_rows_of_one_token_per_sequence():
    """(B, 1, C) slices are B rows of the sequence's stride; the stride of an axis of one element says nothing."""
    x = torch.zeros(4, 5, 32)
    wide = torch.zeros(4, 5, 96)
    for t, rows, stride in ((x, 20, 32), (x[:, -1:], 4, 160), (x[:, 2], 4, 160), (wide[:, 1:2, 32:64], 4, 480),
                            (wide[..., 32:64], 20, 96), (wide[1:2, 2:3, :32], 1, 32), (x[0, 0], 1, 32),
                            (wide[2:3, :, 64:], 5, 96), (x.transpose(0, 1)[:, 1:2], 5, 32),
                            (torch.zeros(32, 1, 1).permute(1, 2, 0), 1, 32)):
        got = ew._rows(t, "x")
        assert got == (rows, stride), (tuple(t.shape), t.stride(), got)
        flat = torch.as_strided(t, (rows, 32), (stride, 1)) if rows > 1 else t.reshape(1, 32)
        assert flat.data_ptr() == t.data_ptr() and flat.shape[0] * 32 == t.numel()
    for t in (x.transpose(0, 1), x[:, ::2], wide[:, :3, :32], x.transpose(1, 2)):
        with pytest.raises(ValueError, match="x"):
            ew._rows(t, "x")


def test_batch_rows_of_another_device_are_refused():
    x = torch.zeros(2, 3, 16)
    rows = torch.zeros(2, 96)
    assert ew._per_batch(rows[:, 16:32], 2, 16, x, "gate") == (rows.data_ptr() + 64, 96)
    assert ew._per_batch(None, 2, 16, x, "gate") == (0, 0)
    with pytest.raises(ValueError, match="gate must be on"):
        ew._per_batch(torch.zeros(2, 16, device="meta"), 2, 16, x, "gate")
    with pytest.raises(TypeError):
        ew._per_batch(torch.zeros(2, 16).double(), 2, 16, x, "gate")
