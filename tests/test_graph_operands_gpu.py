"""A captured sampler loop whose caller lets go of the weights and the per-clip state, on the GPU."""
from __future__ import annotations

import gc
import weakref

import pytest
import torch

from hummingbird_amd import dit, sampling
from hummingbird_amd.dtypes import BF16
from tests.test_sampler_gpu import MEDIUM2, case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tensors(tree):
    if torch.is_tensor(tree):
        yield tree
    elif isinstance(tree, dict):
        for v in tree.values():
            yield from tensors(v)
    elif isinstance(tree, (list, tuple)):
        for v in tree:
            yield from tensors(v)


@pytest.mark.parametrize("projections", ["torch", "q8"])
def test_graph_holds_what_it_reads(projections):
    """Every tensor of `params` and `static` lives as long as the graph; its replays give the eager loop's result after
    the caller's references are gone and their memory could have been given back."""
    print("\n[case] PingpongGraph holds its operands", projections, flush=True)
    params, cond, mask, x = case(MEDIUM2, BF16, 1, 100, seed=31, ctx_tokens=257)
    if projections == "q8":
        params = dit.quantize_params(params)
    static = dit.prepare_static(params, cond, mask, MEDIUM2, BF16)
    noise = torch.randn((2, 1, MEDIUM2.io_channels, 100), device=DEV)
    schedule = sampling.build_schedule(2, device=DEV)
    ref, _ = sampling.pingpong(params, x, schedule, noise, static, MEDIUM2, BF16, trajectory=False, projections=projections)
    ref = ref.clone()
    graph = sampling.PingpongGraph(params, static, MEDIUM2, BF16, x, noise, projections=projections)
    refs = [weakref.ref(t) for t in (*tensors(params), *tensors(static))]
    contexts = [weakref.ref(c.workspace) for c in static["cross"]]
    assert len(refs) > 20 and len(contexts) == MEDIUM2.depth
    static.clear()
    del params, static
    gc.collect()
    assert all(r() is not None for r in refs + contexts)  # (before any replay)
    torch.cuda.empty_cache()
    for rep in range(3):
        got = graph(x, noise)
        torch.cuda.synchronize()
        assert torch.equal(got, ref), f"replay {rep}"
        torch.cuda.empty_cache()
    del graph, got
    gc.collect()
    assert all(r() is None for r in refs + contexts)
