"""What a captured sampler loop holds on to, on the CPU."""
from __future__ import annotations

import gc
import weakref

import torch

from hummingbird_amd import sampling


def test_held_keeps_every_tensor_of_a_tree():
    """A graph reads its weights and its per-clip state where they lie. The tensors stay when the caller's dictionaries
    change or go, and none is copied."""
    tree = {"blocks": [{"w": torch.ones(2), "pair": (torch.ones(3), None)}], "other": object(), "n": 3}
    held = sampling._held(tree)
    assert held["blocks"][0]["w"] is tree["blocks"][0]["w"] and held["other"] is tree["other"] and held["n"] == 3
    assert isinstance(held["blocks"], list) and isinstance(held["blocks"][0]["pair"], tuple)
    refs = [weakref.ref(tree["blocks"][0]["w"]), weakref.ref(tree["blocks"][0]["pair"][0])]
    tree["blocks"][0]["w"] = None
    tree["blocks"].clear()
    del tree
    gc.collect()
    assert all(r() is not None for r in refs)
    del held
    gc.collect()
    assert all(r() is None for r in refs)
