"""The plain model's attentions against a `static` or offsets of other sizes than their input: refused, as the differential
model refuses another mask."""
from __future__ import annotations

import pytest
import torch

from hummingbird_amd import dit
from hummingbird_amd.dtypes import BF16
from tests.test_plain_denoiser_gpu import DEV, PLAIN, announce
from tests.test_sampler_gpu import case

pytestmark = pytest.mark.gpu


def test_static_of_another_batch_or_length_is_refused():
    announce("plain model, static of another batch or length")
    params, cond, mask, x = case(PLAIN, BF16, 1, 20)
    static = dit.prepare_static(params, cond, mask, PLAIN, BF16)
    block, length = params["transformer"]["blocks"][0], 20 + PLAIN.num_memory_tokens
    h = torch.randn(1, length, PLAIN.embed_dim, device=DEV, dtype=torch.bfloat16)
    want = dit.self_attention(h, block, static, PLAIN)
    assert want.shape == h.shape
    with pytest.raises(ValueError, match="static"):  # the second entry would be zeros
        dit.self_attention(h.expand(2, -1, -1), block, static, PLAIN)
    with pytest.raises(ValueError, match="static"):
        dit.self_attention(h[:, :-1], block, static, PLAIN)


def test_offsets_of_another_batch_are_refused():
    announce("plain model, offsets of another batch")
    params, cond, mask, x = case(PLAIN, BF16, 2, 20)
    static = dit.prepare_static(params, cond, mask, PLAIN, BF16)
    block = params["transformer"]["blocks"][0]
    h = torch.randn(2, 20 + PLAIN.num_memory_tokens, PLAIN.embed_dim, device=DEV, dtype=torch.bfloat16)
    want = dit.cross_attention(h, block, static["cross"][0], PLAIN)
    got = dit.cross_attention(h, block, static["cross"][0], PLAIN, offsets=static["offsets"])
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="offsets"):
        dit.cross_attention(h, block, static["cross"][0], PLAIN, offsets=static["offsets"][:2])
