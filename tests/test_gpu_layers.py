"""Layers in training (dropout, dense layers, attention with dot products) against plain implementations in 64 bits; the bounds are
derived in layers_ref."""
import math

import numpy as np
import pytest
import torch

import layers_ref as ref
from gpu_util import dev, host_u32
from neutronbench_amd import layers, synth
from neutronbench_amd.batch import BatchBuilder
from neutronbench_amd.layout import FullGraphChunk, SampledLayer, as_u32, u32_to_i64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def rows(n, F, seed, dtype, device, scale=1.0, shift=0):
    """Values that `dtype` holds, on the device (`shift` values behind an aligned address) and as doubles."""
    rng = np.random.default_rng(seed)
    t = torch.from_numpy((rng.standard_normal((n, F)) * scale).astype(np.float32)).to(dtype)
    flat = torch.zeros(n * F + shift, dtype=dtype, device=device)
    flat[shift:] = t.to(device).reshape(-1)
    return flat[shift:].view(n, F), t.double().numpy()


# ---- dropout ----------------------------------------------------------------------------------------


def test_numbers_of_the_generator():
    """Known answers of Philox-4x32 with ten rounds."""
    assert [int(w) for w in ref.words((0, 0, 0, 0), 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(w) for w in ref.words((0xFFFFFFFF,) * 4, 2**64 - 1)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def dropped(x, p, seed, step):
    """float32 values as the definition gives them (one product, rounded to the type afterwards)."""
    kept = ref.row_factors(*x.shape, p, seed, step) != 0
    with np.errstate(invalid="ignore", over="ignore"):
        return np.where(kept, x.astype(np.float32) * ref.factor(p), np.float32(0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,F,p", [(1, 1, 0.5), (1, 7, 0.1), (3, 8, 0.5), (5, 9, 0.3), (300, 41, 0.1), (1000, 128, 0.5), (257, 100, 0.75),
                                   (70, 1433, 0.5), (64, 64, 0.0), (64, 64, 1.0), (33, 16, 1e-7), (4000, 1, 0.5)])
def test_dropout(device, dtype, n, F, p):
    for seed, step, shift in ((0, 0, 0), (2**64 - 1, 2**32 - 1, 1), (0x123456789ABCDEF, 77, 3)):
        x, _ = rows(n, F, 5, dtype, device, shift=shift)
        g, _ = rows(n, F, 6, dtype, device, shift=shift)
        op = layers.DropoutOp(layers.Dropout(p, seed, step))
        for got, t in ((op.forward(x), x), (op.backward(g), g)):
            want = torch.from_numpy(dropped(t.float().cpu().numpy(), p, seed, step)).to(dtype)
            assert torch.equal(got.cpu(), want)


def test_dropout_of_infinities_and_nan(device):
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1.0] * 64] * 8, device=device)
    got = layers.DropoutOp(layers.Dropout(0.5, 3, 1)).forward(x).cpu().numpy()
    kept = ref.row_factors(8, 256, 0.5, 3, 1) != 0
    assert (got[~kept] == 0).all() and not np.isfinite(got[kept & ~np.isfinite(x.cpu().numpy())]).any()
    assert (got[kept & (x.cpu().numpy() == 1)] == 2).all()


def test_dropout_in_place_and_rows_behind(device):
    whole = torch.full((40, 33), 3.0, device=device)
    x = whole[:30]
    want = layers.DropoutOp(layers.Dropout(0.5, 9)).forward(x.clone())
    desc = layers._Drawn(layers.Dropout(0.5, 9), device).desc
    layers.call("nts_dropout", x.data_ptr(), x.data_ptr(), 0, 30, 33, layers._ref(desc), layers._stream(x.device))
    assert torch.equal(x, want) and (whole[30:] == 3.0).all()


def test_dropout_keeps_the_share_it_says(device):
    """4 M values: the share kept is within five standard deviations of 1 - p, and rows, columns and steps do not repeat each other."""
    x = torch.ones(4096, 1024, device=device)
    kept = []
    for step in (0, 1):
        y = layers.DropoutOp(layers.Dropout(0.3, 11, step)).forward(x)
        kept.append(y != 0)
        t = ref.threshold(0.3) / 65536
        assert abs(float(kept[-1].double().mean()) - (1 - t)) < 5 * math.sqrt(t * (1 - t) / x.numel())
    same = float((kept[0] == kept[1]).double().mean())
    assert abs(same - (0.7**2 + 0.3**2)) < 5 * math.sqrt(0.25 / x.numel())
    assert not torch.equal(kept[0][:, :512], kept[0][:, 512:]) and not torch.equal(kept[0][:2048], kept[0][2048:])


def test_dropout_of_a_large_table(device):
    """More than 2^31 values: rows far behind are those that their numbers say."""
    n, F = 70_000_000, 33
    x = torch.ones(n, F, dtype=torch.bfloat16, device=device)
    y = layers.DropoutOp(layers.Dropout(0.5, 21, 4)).forward(x)
    del x
    for first in (0, 32_537_631, 65_075_262, n - 50):
        groups = ref.numbers((np.arange(5)[None, :], np.arange(first, first + 50)[:, None], 4, 0), 21).reshape(50, -1)[:, :F]
        assert np.array_equal(y[first:first + 50].float().cpu().numpy(), np.where(groups >= 32768, 2.0, 0.0))


def test_step_on_the_device_in_a_captured_graph(device):
    """Replays draw what the step says that the word holds then; the backward pass uses its forward pass's step."""
    n, F = 300, 50
    step = torch.zeros(1, dtype=torch.int32, device=device)
    x, g = torch.randn(n, F, device=device), torch.randn(n, F, device=device)
    drop = layers.DropoutOp(layers.Dropout(0.4, 5, step))
    dense = layers.DenseOp("gelu", layers.Dropout(0.4, 6, step))
    w, b = torch.randn(24, F, device=device), torch.randn(24, device=device)

    def both():
        y = drop.forward(x)
        z = dense.forward(y, w, b)
        gy = dense.backward(z)
        return y, z, gy, *dense.get_additional_grad(), drop.backward(g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
        step.add_(1)
    for value in (0, 1, 7, -1):  # -1: the bit pattern of 2^32 - 1
        step.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        again = layers.DropoutOp(layers.Dropout(0.4, 5, value % 2**32))
        same = layers.DenseOp("gelu", layers.Dropout(0.4, 6, value % 2**32))
        y = again.forward(x)
        z = same.forward(y, w, b)
        gy = same.backward(z)
        for a, e in zip(got, (y, z, gy, *same.get_additional_grad(), again.backward(g))):
            assert torch.equal(a, e)


def test_step_may_advance_between_the_passes(device):
    x = torch.ones(100, 40, device=device)
    step = torch.full((1,), 3, dtype=torch.int32, device=device)
    op = layers.DropoutOp(layers.Dropout(0.5, 1, step))
    y = op.forward(x)
    step.add_(1)
    assert torch.equal(op.backward(x), y) and not torch.equal(op.forward(x), y)


# ---- dense ------------------------------------------------------------------------------------------


def dense_case(device, n, F, N, dtype, act, bias, residual, p, seed=0, shift=0, scale=1.0):
    x, x64 = rows(n, F, seed + 1, dtype, device, scale, shift)
    w, w64 = rows(N, F, seed + 2, dtype, device, 1 / math.sqrt(F), shift)
    b, b64 = rows(1, N, seed + 3, dtype, device, 0.5, shift) if bias else (None, None)
    r, r64 = rows(n, N, seed + 4, dtype, device, 1.0, shift) if residual else (None, None)
    g, g64 = rows(n, N, seed + 5, dtype, device, 1.0, shift)
    factors = ref.row_factors(n, N, p, 1234567 + seed, 8) if p else np.ones((n, N))
    if bias:
        b, b64 = b[0], b64[0]
    return (x, w, b, r, g), (x64, w64, b64, r64, g64), factors, layers.Dropout(p, 1234567 + seed, 8) if p else None


def check_dense(device, n, F, N, dtype, act, bias=True, residual=False, p=0.0, **kw):
    (x, w, b, r, g), plain, factors, dropout = dense_case(device, n, F, N, dtype, act, bias, residual, p, **kw)
    want = ref.dense(*plain, act, factors, dtype)
    op = layers.DenseOp(act, dropout)
    ref.check(op.forward(x, w, b, r), want["y"], "y")
    ref.check(op.backward(g), want["x"], "gradient of x")
    gw, gb = op.get_additional_grad()
    ref.check(gw, want["w"], "gradient of w")
    if bias:
        ref.check(gb, want["b"], "gradient of bias")
    else:
        assert gb is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,F,N", [(1, 1, 1), (1, 602, 256), (3, 17, 5), (8, 100, 130), (9, 33, 129), (64, 8, 8), (130, 64, 47), (129, 31, 128),
                                   (300, 128, 128), (257, 96, 260), (513, 47, 3), (1000, 100, 36), (40, 1433, 16), (700, 40, 200)])
def test_dense(device, dtype, n, F, N):
    for i, (act, bias, residual, p) in enumerate((("none", False, False, 0.0), ("relu", True, False, 0.5), ("gelu", True, True, 0.1),
                                                  ("silu", False, True, 0.0), ("none", True, True, 0.3), ("relu", True, True, 0.0))):
        check_dense(device, n, F, N, dtype, act, bias, residual, p, seed=10 * i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 3, 5])
def test_dense_at_any_alignment(device, dtype, shift):
    check_dense(device, 150, 64, 72, dtype, "gelu", True, True, 0.2, shift=shift)
    check_dense(device, 4, 64, 72, dtype, "gelu", True, True, 0.2, shift=shift)


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_of_many_rows(device, dtype):
    """Parts of the weight's gradient, tiles on every chiplet."""
    check_dense(device, 20000, 65, 130, dtype, "silu", True, False, 0.5)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("F,N,act", [(520, 3900, "gelu"), (3900, 520, "silu"), (1000, 4090, "none")])
@pytest.mark.parametrize("shift", [0, 1])
def test_dense_of_wide_layers(device, dtype, F, N, act, shift):
    """Large tiles: of the layer, of its gradient, and none where operands lie between aligned addresses."""
    check_dense(device, 4099, F, N, dtype, act, True, act == "gelu", 0.1 if act == "silu" else 0.0, shift=shift)


def test_dense_of_large_and_small_values(device):
    """Rows whose parts in 16 bits reach the ends of the exponents' range."""
    n, F, N = 40, 64, 32
    x, x64 = rows(n, F, 1, F32, device)
    w, w64 = rows(N, F, 2, F32, device)
    for up in (2.0 ** 126, 2.0 ** -100):
        a = x * up
        y = layers.DenseOp().forward(a, w / up)
        size = np.abs(x64) @ np.abs(w64).T
        # Parts below 2^-126 may count as 0.  The first such part is below 2^-126, so are the later ones by 2^-8 and 2^-16 of it: a value
        # stands for another one that is off by less than 2^-126 (1 + 2^-7).  With up = 2^126 every weight is such a value.
        lost = 2.0 ** -126 * (1 + 2.0 ** -7)
        size = (F + 4) * ref.U * size + lost * (up * np.abs(x64).sum(1)[:, None] + np.abs(w64).sum(1)[None, :] / up)
        assert (np.abs(y.double().cpu().numpy() - x64 @ w64.T) <= size).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 150])
def test_dense_of_infinities_and_nan(device, dtype, n):
    """They stay in their rows (columns, for those of the weight), with their signs."""
    F, N = 40, 24
    x = torch.ones(n, F, dtype=dtype, device=device)
    w = torch.ones(N, F, dtype=dtype, device=device)
    x[1, 3], x[2, 4], x[3, 5] = math.inf, -math.inf, math.nan
    w[7, 9] = -math.inf
    y = layers.DenseOp().forward(x, w).float().cpu()
    want = torch.full((n, N), float(F))
    want[:, 7] = -math.inf
    want[1], want[2], want[3] = math.inf, -math.inf, math.nan
    want[1, 7] = math.nan
    assert torch.equal(torch.nan_to_num(y, nan=-1.0), torch.nan_to_num(want, nan=-1.0))
    op = layers.DenseOp()
    op.forward(torch.ones(n, F, dtype=dtype, device=device), torch.ones(N, F, dtype=dtype, device=device))
    g = torch.ones(n, N, dtype=dtype, device=device)
    g[2, 6] = math.inf
    gx = op.backward(g).float().cpu()
    gw, _ = op.get_additional_grad()
    assert (gx[2] == math.inf).all() and (gx[torch.arange(n) != 2] == N).all()
    assert (gw[6].float() == math.inf).all() and (gw.float()[torch.arange(N) != 6] == n).all()


def test_dense_gradient_against_differences(device):
    """The gradients of a sum of outputs times g are what small steps of the operands change it by."""
    n, F, N = 12, 9, 7
    (x, w, b, r, g), (x64, w64, b64, r64, g64), factors, dropout = dense_case(device, n, F, N, F32, "gelu", True, True, 0.3)
    op = layers.DenseOp("gelu", dropout)
    op.forward(x, w, b, r)
    got = [op.backward(g), *op.get_additional_grad()]
    h = 1e-4

    def total(x, w, b):
        return float((ref.activation(x @ w.T + b, "gelu")[0] * factors * g64).sum())

    for which, grad in enumerate(got):
        args = [x64, w64, b64]
        for at in np.ndindex(args[which].shape):
            up, down = [a.copy() for a in args], [a.copy() for a in args]
            up[which][at] += h
            down[which][at] -= h
            # central differences are off by h^2 times the third derivative, some hundreds here; the gradient by its sums
            assert abs((total(*up) - total(*down)) / (2 * h) - float(grad.cpu()[at])) < 1e-4


def test_dense_without_what_is_not_wanted(device):
    (x, w, b, r, g), plain, factors, dropout = dense_case(device, 200, 30, 20, F32, "relu", True, False, 0.5)
    op = layers.DenseOp("relu", dropout, rows_grad=False)
    op.forward(x, w, b)
    want = ref.dense(*plain, "relu", factors, F32)
    assert op.backward(g) is None
    ref.check(op.get_additional_grad()[0], want["w"], "gradient of w")


def test_dense_of_no_rows(device):
    for dtype in TYPES:
        op = layers.DenseOp("relu", layers.Dropout(0.5, 1))
        x, w, b = (torch.ones(s, dtype=dtype, device=device) for s in ((0, 8), (6, 8), (6,)))
        assert op.forward(x, w, b).shape == (0, 6)
        assert op.backward(torch.ones(0, 6, dtype=dtype, device=device)).shape == (0, 8)
        gw, gb = op.get_additional_grad()
        assert (gw == 0).all() and (gb == 0).all() and gw.shape == (6, 8)


def test_dense_is_the_same_every_time_and_leaves_rows_behind(device):
    (x, w, b, r, g), *_, dropout = dense_case(device, 5000, 64, 96, BF16, "gelu", True, True, 0.1)
    runs = []
    for _ in range(3):
        op = layers.DenseOp("gelu", dropout)
        runs.append([op.forward(x, w, b, r), op.backward(g), *op.get_additional_grad()])
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))
    out = torch.full((5100, 96), 7.0, dtype=BF16, device=device)
    desc = layers._Drawn(dropout, device).desc
    work = layers._work(layers.call("nts_dense_work_bytes", 1, 5000, 96, 64), device)
    layers.call("nts_dense", out.data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), 1, 5000, 96, 64, 2, layers._ref(desc),
                work.data_ptr(), layers._stream(x.device))
    assert torch.equal(out[:5000], runs[0][0]) and (out[5000:] == 7.0).all()


# ---- attention --------------------------------------------------------------------------------------


def layer_of(co, ri, Vs, device, bound=0):
    ro, ci = ref.by_source(co, ri, Vs)
    sg = SampledLayer()
    sg.v_size, sg.e_size, sg.src_size, sg.max_in_degree = len(co) - 1, int(co[-1] - co[0]), Vs, bound
    sg.dev_column_offset, sg.dev_row_indices = dev(co, device), dev(ri, device)
    sg.dev_row_offset, sg.dev_column_indices = dev(ro, device), dev(ci, device)
    return sg


def graph(rng, Vd, Vs, mean, missing=0.0, hub=0):
    deg = rng.poisson(mean, Vd)
    deg[::7] = 0
    if hub:
        deg[Vd // 2] = hub
    co = np.zeros(Vd + 1, dtype=np.uint32)
    co[1:] = np.cumsum(deg)
    ri = rng.integers(0, max(Vs, 1), int(co[-1])).astype(np.uint32)
    ri[rng.random(ri.size) < 0.2] = 0  # a source with many edges
    gone = rng.random(ri.size) < missing
    ri[gone] = rng.choice(np.array([0xFFFFFFFF, Vs, Vs + 5], dtype=np.uint32), int(gone.sum()))
    return co, ri


def check_attention(device, co, ri, Vs, H, Hk, D, dtype, p=0.0, bound=0, scale=None, seed=3, shift=0, size=1.0):
    Vd = len(co) - 1
    q, q64 = rows(Vd, H * D, seed, dtype, device, size, shift)
    k, k64 = rows(Vs, Hk * D, seed + 1, dtype, device, size, shift)
    v, v64 = rows(Vs, Hk * D, seed + 2, dtype, device, 1.0, shift)
    g, g64 = rows(Vd, H * D, seed + 3, dtype, device, 1.0, shift)
    drop = (p, 99991 + seed, 12) if p else None
    used = 1 / math.sqrt(D) if scale is None else scale
    want = ref.attention(q64, k64, v64, g64, co, ri, H, Hk, np.float32(used).astype(np.float64), drop, dtype)
    op = layers.DotAttentionOp(layer_of(co, ri, Vs, device, bound), H, Hk, scale, layers.Dropout(*drop) if p else None)
    out = op.forward(q, k, v)
    ref.check(out, want["out"], "out")
    ref.check(op.lse, want["lse"], "lse")
    gq = op.backward(g)
    gk, gv = op.get_additional_grad()
    for name, got in (("q", gq), ("k", gk), ("v", gv)):
        ref.check(got, want[name], f"gradient of {name}")
    return out, op.lse, gq, gk, gv


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(1, 1, 1), (1, 1, 8), (4, 4, 32), (3, 3, 20), (2, 1, 47), (8, 2, 64), (6, 3, 16), (5, 5, 3), (16, 4, 128),
                                    (2, 2, 256), (3, 1, 200), (12, 12, 7), (4, 2, 96), (40, 1, 8), (64, 64, 4)])
def test_attention(device, dtype, H, Hk, D):
    rng = np.random.default_rng(H * 1000 + D)
    co, ri = graph(rng, 60, 45, 9, missing=0.1)
    check_attention(device, co, ri, 45, H, Hk, D, dtype)
    check_attention(device, co, ri, 45, H, Hk, D, dtype, p=0.3)
    check_attention(device, co, ri, 45, H, Hk, D, dtype, p=0.5, bound=int(np.diff(co.astype(np.int64)).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 32), (8, 2, 64), (3, 1, 20), (2, 2, 256)])
def test_attention_of_hubs(device, dtype, H, Hk, D):
    """Destinations and sources of thousands of edges among short ones, cut at the ends of spans."""
    rng = np.random.default_rng(D)
    co, ri = graph(rng, 400, 300, 12, missing=0.05, hub=9000)
    check_attention(device, co, ri, 300, H, Hk, D, dtype, p=0.2)


@pytest.mark.parametrize("degree", [0, 1, 2, 63, 64, 65, 300, 5000])
def test_attention_of_one_destination(device, degree):
    rng = np.random.default_rng(degree)
    co, ri = np.array([0, degree], dtype=np.uint32), rng.integers(0, 50, degree).astype(np.uint32)
    for dtype in TYPES:
        check_attention(device, co, ri, 50, 4, 4, 32, dtype)
        check_attention(device, co, ri, 50, 6, 2, 24, dtype, p=0.5)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_at_any_alignment_and_offset(device, dtype):
    """Operands that begin between aligned addresses; offsets that do not begin at 0."""
    rng = np.random.default_rng(8)
    co, ri = graph(rng, 50, 40, 7)
    for shift in (1, 3):
        check_attention(device, co, ri, 40, 4, 2, 32, dtype, shift=shift, p=0.1)
    padded = np.concatenate([rng.integers(0, 40, 11).astype(np.uint32), ri])
    a = check_attention(device, co, ri, 40, 4, 2, 32, dtype)
    b = check_attention(device, co + np.uint32(11), padded, 40, 4, 2, 32, dtype)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_attention_scales(device):
    rng = np.random.default_rng(9)
    co, ri = graph(rng, 40, 30, 8)
    for scale in (0.0, -0.7, 3.0):
        check_attention(device, co, ri, 30, 2, 2, 32, F32, scale=scale)
    check_attention(device, co, ri, 30, 2, 2, 32, F32, size=8.0)  # scores of some hundred: one neighbour has all


def test_attention_without_edges_sources_or_destinations(device):
    none = np.zeros(0, dtype=np.uint32)
    for dtype in TYPES:
        check_attention(device, np.zeros(6, dtype=np.uint32), none, 4, 2, 2, 16, dtype)
        check_attention(device, np.zeros(1, dtype=np.uint32), none, 4, 2, 2, 16, dtype)
        check_attention(device, np.array([0, 2, 2], dtype=np.uint32), np.array([0, 0xFFFFFFFF], dtype=np.uint32), 0, 2, 2, 16, dtype, p=0.5)


def test_attention_never_reads_sources_that_are_not_there(device):
    """Rows behind the last source hold NaN; edges name them, and ids far behind."""
    rng = np.random.default_rng(4)
    co, ri = graph(rng, 50, 30, 6, missing=0.5)
    whole = [torch.full((40, 64), math.nan, device=device) for _ in range(2)]
    q, g = torch.randn(50, 64, device=device), torch.randn(50, 64, device=device)
    k, v = (t[:30] for t in whole)
    k.normal_(), v.normal_()
    op = layers.DotAttentionOp(layer_of(co, ri, 30, device), 2)
    for t in (op.forward(q, k, v), op.backward(g), *op.get_additional_grad()):
        assert torch.isfinite(t).all()


def test_attention_of_infinite_scores(device):
    """-infinity as a score: no weight, also where all of a destination's are; +infinity or NaN: NaN, at that head of that destination alone."""
    D = 16
    co = np.array([0, 3, 5, 8, 10], dtype=np.uint32)
    ri = np.array([0, 1, 2, 3, 3, 0, 4, 1, 0, 5], dtype=np.uint32)
    k = torch.zeros(6, 2 * D, device=device)
    k[3, 0], k[4, 0], k[5, 0] = -math.inf, math.inf, math.nan
    q = torch.ones(4, 2 * D, device=device)
    v = torch.randn(6, 2 * D, device=device)
    op = layers.DotAttentionOp(layer_of(co, ri, 6, device), 2)
    out = op.forward(q, k, v).view(4, 2, D).cpu()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[:, 1]).all()
    assert (out[1, 0] == 0).all() and op.lse[1, 0] == -math.inf
    assert torch.isnan(out[2, 0]).all() and torch.isnan(out[3, 0]).all()
    mixed = layers.DotAttentionOp(layer_of(np.array([0, 3], dtype=np.uint32), np.array([0, 3, 1], dtype=np.uint32), 6, device), 2)
    got = mixed.forward(q[:1], k, v).view(2, D)
    assert torch.allclose(got[0], (v[0, :D] + v[1, :D]) / 2, atol=1e-6)
    gq = mixed.backward(torch.ones(1, 2 * D, device=device))
    assert torch.isfinite(gq[0, D:]).all()


def test_attention_gradient_against_differences(device):
    rng = np.random.default_rng(5)
    co = np.array([0, 4, 4, 9, 10], dtype=np.uint32)
    ri = rng.integers(0, 6, 10).astype(np.uint32)
    H, Hk, D, Vs, scale = 4, 2, 5, 6, 0.6
    drop = (0.3, 17, 2)
    q, q64 = rows(4, H * D, 1, F32, device)
    k, k64 = rows(Vs, Hk * D, 2, F32, device)
    v, v64 = rows(Vs, Hk * D, 3, F32, device)
    g, g64 = rows(4, H * D, 4, F32, device)
    op = layers.DotAttentionOp(layer_of(co, ri, Vs, device), H, Hk, scale, layers.Dropout(*drop))
    op.forward(q, k, v)
    got = [op.backward(g), *op.get_additional_grad()]
    h = 1e-4

    def total(q, k, v):
        return float((ref.attention(q, k, v, None, co, ri, H, Hk, float(np.float32(scale)), drop, F32)["out"][0] * g64).sum())

    for which, grad in enumerate(got):
        args = [q64, k64, v64]
        for at in np.ndindex(args[which].shape):
            up, down = [a.copy() for a in args], [a.copy() for a in args]
            up[which][at] += h
            down[which][at] -= h
            assert abs((total(*up) - total(*down)) / (2 * h) - float(grad.cpu()[at])) < 1e-4


def test_attention_over_a_full_graph_is_the_same_every_time(device):
    V, E, H, D = 3000, 60000, 4, 32
    src, dst = synth.rmat_edges(V, E, seed=3, device=device)
    chunk = FullGraphChunk.from_edges(src, dst, V)
    q, k, v, g = (torch.randn(V, H * D, device=device) for _ in range(4))
    first = None
    for _ in range(3):
        op = layers.DotAttentionOp(chunk, H, dropout=layers.Dropout(0.1, 4))
        got = [op.forward(q, k, v), op.lse, op.backward(g), *op.get_additional_grad()]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    co, ri = host_u32(chunk.column_offset_gpu), host_u32(chunk.row_indices_gpu)
    arrays = [t.double().cpu().numpy() for t in (q, k, v, g)]
    want = ref.attention(*arrays, co, ri, H, H, float(np.float32(1 / math.sqrt(D))), (0.1, 4, 0), F32)
    for name, t in zip(("out", "lse", "q", "k", "v"), first):
        ref.check(t, want[name], name)


def test_attention_of_sources_beyond_4_gb(device):
    """Offsets of rows that pass 32 bits."""
    Vs, H, D = 9_000_000, 4, 64
    k = torch.zeros(Vs, H * D, dtype=BF16, device=device)
    v = torch.zeros(Vs, H * D, dtype=BF16, device=device)
    rng = np.random.default_rng(2)
    at = np.unique(np.concatenate([[0, Vs - 1, Vs // 2, 8_388_607, 8_388_608], rng.integers(0, Vs, 60)]))
    small, k64 = rows(len(at), H * D, 1, BF16, device)
    small_v, v64 = rows(len(at), H * D, 2, BF16, device)
    where = torch.from_numpy(at).to(device)
    k[where], v[where] = small, small_v
    co, local = graph(rng, 30, len(at), 10)
    ri = at[local].astype(np.uint32)
    q, q64 = rows(30, H * D, 3, BF16, device)
    g, g64 = rows(30, H * D, 4, BF16, device)
    op = layers.DotAttentionOp(layer_of(co, ri, Vs, device), H)
    out = op.forward(q, k, v)
    gq = op.backward(g)
    gk, gv = op.get_additional_grad()
    want = ref.attention(q64, k64, v64, g64, co, local, H, H, 0.125, None, BF16)
    for name, t in (("out", out), ("lse", op.lse), ("q", gq), ("k", gk[where]), ("v", gv[where])):
        ref.check(t, want[name], name)
    other = torch.ones(Vs, dtype=torch.bool, device=device)
    other[where] = False
    assert (gk[other].abs().amax() == 0) and (gv[other].abs().amax() == 0)


def test_a_layer_of_a_graph_transformer(device):
    """Projections, attention, output with residual and the two dense layers behind it, forward and backward over a sampled layer, as a
    model would chain them: against the same in 64 bits with torch's own differentiation."""
    V, E, H, D = 500, 6000, 4, 16
    W = H * D
    src, dst = synth.rmat_edges(V, E, seed=5, device=device, sort=True)
    co, ri = synth.build_csc(src, dst, V)
    builder = BatchBuilder(as_u32(co), as_u32(ri), [6], 64, want_perm=False, graph=0)
    builder.enqueue(as_u32(synth.permutation(V, 3, device)[:64]), 7)
    sg = builder.collect()[0]
    n, m = sg.src_size, sg.v_size
    gen = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(n, W, device=device, generator=gen)
    weights = [torch.randn(a, W if i < 5 else 2 * W, device=device, generator=gen) / math.sqrt(W) for i, a in enumerate((W, W, W, W, 2 * W, W))]
    bias = [torch.randn(w.shape[0], device=device, generator=gen) * 0.1 for w in weights]
    rates = dict(attention=(0.2, 101, 6), up=(0.3, 102, 6))
    co_h, ri_h = (u32_to_i64(torch.from_numpy(host_u32(t).view(np.int32))) for t in (sg.dev_c_o(), sg.dev_r_i()))
    # the framework's operators
    top = x[:m].contiguous()  # stands for the destinations' own rows
    proj = [layers.DenseOp() for _ in range(3)]
    q = proj[0].forward(top, weights[0], bias[0])
    k, v = (proj[i].forward(x, weights[i], bias[i]) for i in (1, 2))
    att = layers.DotAttentionOp(sg, H, dropout=layers.Dropout(*rates["attention"]))
    a = att.forward(q, k, v)
    mix = layers.DenseOp()
    h = mix.forward(a, weights[3], bias[3], top)
    up, down = layers.DenseOp("gelu", layers.Dropout(*rates["up"])), layers.DenseOp()
    u = up.forward(h, weights[4], bias[4])
    y = down.forward(u, weights[5], bias[5], h)
    g = torch.randn(m, W, device=device, generator=gen)
    gu = down.backward(g)
    gh = up.backward(gu) + g
    ga = mix.backward(gh)
    gq = att.backward(ga)
    gk, gv = att.get_additional_grad()
    gx = proj[1].backward(gk) + proj[2].backward(gv)
    gx[:m] += proj[0].backward(gq) + gh
    grads = [op.get_additional_grad() for op in (*proj, mix, up, down)]
    # the same in 64 bits
    xs = x.double().cpu().requires_grad_()
    ws, bs = [[t.double().cpu().requires_grad_() for t in l] for l in (weights, bias)]
    t = xs[:m]
    qr, kr, vr = t @ ws[0].T + bs[0], xs @ ws[1].T + bs[1], xs @ ws[2].T + bs[2]
    d = torch.repeat_interleave(torch.arange(m), co_h[1:] - co_h[:-1])
    s = (qr.view(m, H, D)[d] * kr.view(n, H, D)[ri_h]).sum(2) / math.sqrt(D)
    e = torch.exp(s)
    pr = e / torch.zeros(m, H, dtype=torch.float64).index_add(0, d, e)[d]
    f = torch.from_numpy(ref.edge_factors(ri_h.numpy(), d.numpy(), H, *rates["attention"]))
    ar = torch.zeros(m, H, D, dtype=torch.float64).index_add(0, d, (pr * f)[:, :, None] * vr.view(n, H, D)[ri_h]).view(m, W)
    hr = t + ar @ ws[3].T + bs[3]
    zr = hr @ ws[4].T + bs[4]
    ur = torch.nn.functional.gelu(zr) * torch.from_numpy(ref.row_factors(m, 2 * W, *rates["up"]))
    yr = hr + ur @ ws[5].T + bs[5]
    yr.backward(g.double().cpu())
    builder.close()
    # six products and a softmax deep, each 32-bit sums of up to 128 terms: some thousand roundings, of which most cancel
    for got, want in [(y, yr), (gx, xs.grad)] + [(a, b.grad) for i, (pair, two) in enumerate(zip(grads, zip(ws, bs)))
                                                 for a, b in zip(pair, two) if i != 1 or a.dim() == 2]:
        want = want.detach()
        assert float((got.double().cpu() - want).norm() / want.norm()) < 200 * ref.U
    # The keys' bias adds the same to all scores of a destination, which the softmax does not see: its gradient is 0, a sum that cancels
    # and is off as far as its terms are, by their magnitudes.
    assert float(bs[1].grad.norm()) < 1e-12
    assert float(grads[1][1].double().norm() / gk.double().abs().sum(0).norm()) < 200 * ref.U


# ---- streams, graphs, calls at once -----------------------------------------------------------------


def test_on_another_stream_and_in_a_graph(device):
    rng = np.random.default_rng(6)
    co, ri = graph(rng, 300, 200, 12, hub=3000)
    sg = layer_of(co, ri, 200, device)
    q, k, v, g = (torch.randn(r, 64, device=device) for r in (300, 200, 200, 300))
    w, b = torch.randn(48, 64, device=device), torch.randn(48, device=device)
    gd = torch.randn(300, 48, device=device)

    def work():
        att, dense = layers.DotAttentionOp(sg, 2, dropout=layers.Dropout(0.2, 3)), layers.DenseOp("silu")
        a = att.forward(q, k, v)
        y = dense.forward(a, w, b)
        return [a, att.lse, y, dense.backward(gd), *dense.get_additional_grad(), att.backward(g), *att.get_additional_grad()]

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        held = work()
    for i in range(4):
        for t in held:
            t.fill_(float(i))
        work()  # eager work between the replays
        captured.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want))
        q.mul_(1.25)
        want = work()
