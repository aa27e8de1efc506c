"""The example network trains and serves (GPU)."""
from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_graph_layers_example(gpu):
    spec = importlib.util.spec_from_file_location(
        "graph_layers", os.path.join(ROOT, "examples", "graph_layers.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, y, y8 = mod.train(nodes=1024, steps=40, say=lambda s: print(s, flush=True))
    assert np.isfinite(losses).all() and losses[-1] < 0.3 * losses[0], losses
    # Two layers of e4m3 operands (4 significant bits): 2^-4 of each layer's update.
    assert np.linalg.norm(y8 - y) <= 2.0 ** -3 * np.linalg.norm(y)
