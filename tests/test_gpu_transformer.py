"""The epoch's graph transformer: its layer against the same in 64 bits, and whole epochs whatever the number of batches in flight."""
import math

import numpy as np
import pytest
import torch

import layers_ref as ref
from gpu_util import dev
from neutronbench_amd import epoch
from neutronbench_amd.layout import SampledLayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(40, 90), (90, 40), (130, 40), (1, 1)])
@pytest.mark.parametrize("p", [0.0, 0.4])
def test_layer_and_its_gradients(device, m, n, p):
    """Fewer destinations than sources, and more: then rows of x stand in for several."""
    H, D, step = 4, 32, 9
    W = H * D
    rng = np.random.default_rng(m)
    degrees = rng.integers(0, 9, m)  # some destinations have no edges
    degrees[0] = 5
    co = torch.from_numpy(np.concatenate([[0], np.cumsum(degrees)]))
    ri = torch.from_numpy(rng.integers(0, n, int(co[-1])))
    sg = SampledLayer.from_host_csc(co, ri, torch.arange(n), torch.arange(m), device)
    gen = torch.Generator(device=device).manual_seed(m)
    weights = [(w, torch.randn(b.shape, device=device, generator=gen) * 0.1) for w, b in epoch.DotLayer.make(W, 70, device)]
    block = epoch.DotLayer(weights, H, p, 32)
    x, g = torch.randn(n, W, device=device, generator=gen), torch.randn(m, W, device=device, generator=gen)
    stages = []
    y = block.forward(sg, x, step, stages.append)
    gx = block.backward(g, stages.append)
    assert stages == ["dense_fwd", "aggregate_fwd", "dense_fwd", "dense_bwd", "aggregate_bwd", "dense_bwd"]
    # the same in 64 bits
    xs = x.double().cpu().requires_grad_()
    ws, bs = [[w[i].double().cpu().requires_grad_() for w in weights] for i in (0, 1)]
    t = xs[torch.arange(m) % n]
    q, k, v = t @ ws[0].T + bs[0], xs @ ws[1].T + bs[1], xs @ ws[2].T + bs[2]
    d = torch.repeat_interleave(torch.arange(m), co[1:] - co[:-1])
    e = torch.exp((q.view(m, H, D)[d] * k.view(n, H, D)[ri]).sum(2) / math.sqrt(D))
    pr = e / torch.zeros(m, H, dtype=torch.float64).index_add(0, d, e)[d]
    f = torch.from_numpy(ref.edge_factors(ri.numpy(), d.numpy(), H, p, 32, step))
    a = torch.zeros(m, H, D, dtype=torch.float64).index_add(0, d, (pr * f)[:, :, None] * v.view(n, H, D)[ri]).view(m, W)
    h = t + (a @ ws[3].T + bs[3]) * torch.from_numpy(ref.row_factors(m, W, p, 33, step))
    u = torch.nn.functional.gelu(h @ ws[4].T + bs[4]) * torch.from_numpy(ref.row_factors(m, 2 * W, p, 34, step))
    want = h + u @ ws[5].T + bs[5]
    want.backward(g.double().cpu())
    # six products and a softmax deep, each 32-bit sums of up to 256 terms: some thousand roundings, of which most cancel
    pairs = [(y, want.detach()), (gx, xs.grad)]
    for i, (gw, gb) in enumerate(block.grads):
        if i == 1 or (i == 0 and n == 1):  # the softmax does not see the keys' bias, nor anything where all sources are one: sums that cancel to 0
            continue
        pairs += [(gw, ws[i].grad), (gb, bs[i].grad)]
    if n > 1:
        pairs.append((block.grads[1][0], ws[1].grad))
    for got, exact in pairs:
        assert float((got.double().cpu() - exact).norm() / exact.norm()) < 200 * ref.U


@pytest.mark.parametrize("features,dropout", [("f32", 0.0), ("f32", 0.5), ("mxfp4", 0.3)])
def test_epochs_match_whatever_is_in_flight(features, dropout):
    runs = [epoch.run("gat", scale=0.02, max_batches=5, warmup_batches=1, pipeline=p, quiet=True, checksum=True, features=features,
                      attention="dot", dropout=dropout) for p in (1, 2, 4)]
    first = runs[0]
    assert first["sampled_edges"] > 0 and first["attention"] == "dot" and math.isfinite(first["checksum"]) and first["checksum"] != 0.0
    assert {"dense_fwd", "dense_bwd", "aggregate_fwd", "aggregate_bwd"} <= set(first["stage_s"])
    for r in runs[1:]:
        for key in ("batches", "sampled_edges", "gathered_rows", "cache_hit_rate", "checksum"):
            assert r[key] == first[key], key


def test_epoch_of_hops_sampled_one_by_one():
    runs = [epoch.run("gat", scale=0.02, max_batches=3, warmup_batches=0, sampler=s, quiet=True, checksum=True, attention="dot", dropout=0.2)
            for s in ("builder", "library")]
    assert runs[0]["sampled_edges"] == runs[1]["sampled_edges"]
    # the samplers bound destinations' edges or not, which takes other orders of sums
    assert runs[0]["checksum"] == pytest.approx(runs[1]["checksum"], rel=1e-3)
