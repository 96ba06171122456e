"""The limits of `hb_packed_attention`'s sizes on the CPU: at each one a call gets as far as its misaligned q, past it the sizes
are refused (no kernel is launched)."""
from __future__ import annotations

import pytest

from tests.test_packed import BF16, SHAPE, STRIDE, addr, attend, lib  # noqa: F401


@pytest.mark.parametrize("at,past", [
    (dict(T=1, N=1, H=65535, G=65535), dict(T=1, N=1, H=65536, G=65536)),
    (dict(T=1, N=1 << 20, H=2, G=2), dict(T=1, N=(1 << 20) + 1, H=2, G=2)),
    (dict(T=1 << 28, N=1, H=4, G=1), dict(T=(1 << 28) + 1, N=1, H=4, G=1)),
    (dict(T=1, N=1, Tk=1 << 30, H=2, G=2), dict(T=1, N=1, Tk=(1 << 30) + 1, H=2, G=2)),
    # (ceil(T gs / 128) + N) G below 2^24: by tokens, and by sequences
    (dict(T=((1 << 23) - 2) * 128, N=1, H=2, G=2), dict(T=((1 << 23) - 2) * 128 + 1, N=1, H=2, G=2)),
    (dict(T=128, N=(1 << 20) - 2, H=16, G=16), dict(T=128, N=(1 << 20) - 1, H=16, G=16)),
])
def test_sizes(lib, at, past):  # noqa: F811
    strides = dict(qt=128, qh=64, kt=128, kh=64, vt=128, vh=64, ot=128, oh=64, q=addr(0) + 2, dtype=BF16)
    assert attend(lib, **{**strides, **at}) == STRIDE
    assert attend(lib, **{**strides, **past}) == SHAPE
