"""Attention with dot products at the ends of its scores: -infinity, and scores so large that their rounding shows."""
import math

import numpy as np
import pytest
import torch

import layers_ref as ref
from neutronbench_amd import layers
from test_gpu_layers import BF16, F16, F32, TYPES, graph, layer_of, rows

pytestmark = pytest.mark.gpu

NOWHERE = 0xFFFFFFFF


def gradients(device, co, ri, q, k, v, g, H, drop=None, bound=0):
    op = layers.DotAttentionOp(layer_of(co, ri, k.shape[0], device, bound), H, H, 0.25, layers.Dropout(*drop) if drop else None)
    return op.forward(q, k, v), op.lse, op.backward(g), *op.get_additional_grad()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [16, 20, 3])
@pytest.mark.parametrize("form", ["spans", "rows", "cut"])
@pytest.mark.parametrize("where", ["key", "query"])
def test_no_gradient_from_scores_of_minus_infinity(device, dtype, D, form, where):
    """A source whose key, or destinations whose query makes scores of -infinity: everything is as if those edges had no source, at destinations that
    keep others and at those that keep none."""
    rng = np.random.default_rng(D)
    Vs, H, drop = 45, 2, (0.3, 21, 4)
    co, ri = graph(rng, 60, Vs, 9, hub=5000 if form == "cut" else 0)
    dst = np.repeat(np.arange(60), np.diff(co.astype(np.int64)))
    (q, q64), (k, k64), (v, v64), (g, g64) = (rows(n, H * D, 30 + i, dtype, device) for i, n in enumerate((60, Vs, Vs, 60)))
    if where == "key":
        ri[dst == 5] = 3
        ri[dst == 30] = 3  # the hub, where there is one
        gone = ri == 3
        for t, p in ((q, q64), (k, k64)):  # every query has something positive there
            t[:, ::D] = t[:, ::D].abs() + 0.5
            p[:, ::D] = t[:, ::D].double().cpu().numpy()
        k[3, ::D] = -math.inf
    else:
        gone = np.isin(dst, [5, 30])
        k[:, ::D] = k[:, ::D].abs() + 0.5
        k64[:, ::D] = k[:, ::D].double().cpu().numpy()
        q[5, ::D] = q[30, ::D] = -math.inf
    left = np.where(gone, np.uint32(NOWHERE), ri)
    want = ref.attention(q64, k64, v64, g64, co, left, H, H, 0.25, drop, dtype)
    bound = int(np.diff(co.astype(np.int64)).max()) if form == "rows" else 0
    got = gradients(device, co, ri, q, k, v, g, H, drop, bound)
    assert np.isneginf(want["lse"][0][5]).all()
    for name, t in zip(("out", "lse", "q", "k", "v"), got):
        ref.check(t, want[name], name)
