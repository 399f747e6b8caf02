"""The cache of 8-bit keys and values and the attention over it against plain implementations in 64 bits: the cache's bytes
are exact, the attention's tolerance is derived in lowbit_ref.attention."""
import math

import numpy as np
import pytest
import torch

import lowbit_ref as ref
from gpu_util import dev, stream
from neutronbench_amd import lowbit, synth
from neutronbench_amd.abi import call, ptr
from neutronbench_amd.batch import BatchBuilder
from neutronbench_amd.layout import FullGraphChunk, SampledLayer

pytestmark = pytest.mark.gpu


def keys(n, width, seed, special=False):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, width)) * np.exp2(rng.integers(-6, 7, (n, 1)))).astype(np.float32)
    x[rng.random((n, width)) < 0.05] = 0.0
    if special and n > 6:
        x[0] = np.float32(1e-44)
        x[1, 0], x[2, width - 1], x[3, width // 2] = np.inf, np.nan, -np.inf
        x[4] = np.float32(3.4028235e38)
        x[5] = 448.0
        x[6] = -0.0
    return x


def empty(capacity, heads, D, block, fill=0):
    return (np.full((capacity, 2, heads, lowbit.kv8_row_width(D)), fill, dtype=np.uint8),
            np.full((-(-capacity // block), 2, heads), fill, dtype=np.uint8))


@pytest.mark.parametrize("heads,D,block", [(1, 1, 1), (1, 16, 4), (4, 32, 16), (3, 20, 16), (2, 47, 8), (2, 64, 16), (3, 47, 32), (8, 128, 64), (5, 256, 32),
                                           (2, 100, 1024)])
def test_append_in_pieces(device, heads, D, block):
    """Pieces that begin and end inside blocks, on blocks, and one row at a time; later rows larger, so that scales grow."""
    capacity = 700 if block < 512 else 2500
    cache, scales = empty(capacity, heads, D, block)
    kv = lowbit.Kv8Cache(capacity, heads, D, block, device=device)
    at = 0
    for i, n in enumerate((1, 1, 5, 40, block, 1, 130, 64, 0, 3)):
        special = i == 6 and block < 100
        with np.errstate(over="ignore"):
            k, v = keys(n, heads * D, i, special) * np.float32(2.0 ** i), keys(n, heads * D, 50 + i, special)
            kv.append(dev(k, device), dev(v, device))
            if n:
                ref.kv8_append(cache, scales, k, v, at, D, block)
        at += n
        assert kv.rows == at
    got = kv.cache.cpu().numpy()
    nan = (cache & 127) == 127
    assert (((got & 127) == 127) == nan).all() and (got == cache)[~nan].all()
    assert (kv.scales.cpu().numpy() == scales).all()


def test_append_again_from_the_middle(device):
    """Rows from `first` on are written anew, those before it stay, bytes behind the last new row are left alone."""
    heads, D, block, capacity = 2, 24, 16, 100
    cache, scales = empty(capacity, heads, D, block, fill=0x55)
    kv = lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, block, rows=0)
    for first, n, seed in ((0, 90, 1), (37, 5, 2), (32, 3, 3), (33, 30, 4)):
        k, v = keys(n, heads * D, seed) * np.float32(seed), keys(n, heads * D, seed + 9)
        ref.kv8_append(cache, scales, k, v, first, D, block)
        kv.append(dev(k, device), dev(v, device), first)
        assert (kv.cache.cpu().numpy() == cache).all() and (kv.scales.cpu().numpy() == scales).all()
        assert kv.rows == first + n
    with pytest.raises(ValueError):
        kv.append(dev(k, device), dev(v, device), 64)


@pytest.mark.parametrize("byte", [0, 130, 247, 253, 254, 255])
@pytest.mark.parametrize("D,block", [(16, 8), (64, 64), (250, 128)])
def test_append_behind_rows_of_any_scale(device, byte, D, block):
    """A cache from elsewhere whose begun block has any scale byte: the new rows are rounded at that scale or a larger one."""
    heads, first, n = 2, 5, block
    cache, scales = empty(2 * block, heads, D, block)
    rng = np.random.default_rng(byte + D)
    cache[:first, :, :, :D] = rng.integers(0, 0x7F, (first, 2, heads, D)) if byte < 240 else rng.integers(0, 2, (first, 2, heads, D))
    scales[0] = byte
    k = (rng.standard_normal((n, heads * D)) * np.exp2(rng.integers(-130, 126, (n, heads * D)))).astype(np.float32)
    v = np.full((n, heads * D), np.float32(3.4028235e38)) if byte > 130 else k[::-1].copy()
    kv = lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, block, rows=first)
    ref.kv8_append(cache, scales, k, v, first, D, block)
    kv.append(dev(k, device), dev(v, device))
    assert (kv.scales.cpu().numpy() == scales).all()
    assert (kv.cache.cpu().numpy() == cache).all()


def graph_of(degrees, V, seed, missing=0.0, offset=0):
    rng = np.random.default_rng(seed)
    co = np.concatenate([[0], np.cumsum(degrees)]).astype(np.uint32) + np.uint32(offset)
    ri = rng.integers(0, V, int(co[-1])).astype(np.uint32)
    ri[rng.random(ri.size) < missing] = 0xFFFFFFFF
    return co, ri


def check(device, degrees, *args, **kwargs):
    """As they are, and with enough destinations without neighbours behind them that none gets a block of its own."""
    check_one(device, degrees, *args, **kwargs)
    if len(degrees) <= 64:
        check_one(device, list(degrees) + [0] * 65, *args, **kwargs)


def check_one(device, degrees, V, q_heads, heads, D, block, seed=1, missing=0.0, bound=0, offset=0, mirrored=False, rows=None,
          scale=None, spread=1.0):
    degrees = np.asarray(degrees, dtype=np.int64)
    Vd = len(degrees)
    cache, scales = empty(V, heads, D, block)
    ref.kv8_append(cache, scales, keys(V, heads * D, seed), keys(V, heads * D, seed + 1), 0, D, block)
    rng = np.random.default_rng(seed + 2)
    q = (rng.standard_normal((Vd, q_heads * D)) * spread).astype(np.float32)
    rows = V if rows is None else rows
    scale = float(np.float32(D ** -0.5 / 8 if scale is None else scale))
    co, ri = graph_of(degrees, V, seed + 3, missing, offset)
    row, mirror = ri, None
    if mirrored:
        mirror, local = np.unique(ri, return_inverse=True)
        row, ri, mirror = mirror[local.reshape(-1)], local.reshape(-1).astype(np.uint32), dev(mirror, device)
    layer = SampledLayer()
    layer.v_size, layer.e_size, layer.max_in_degree = Vd, int(degrees.sum()), bound
    layer.dev_column_offset, layer.dev_row_indices = dev(co, device), dev(ri, device)
    kv = lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, block, rows=rows)
    print(f"case Vd={Vd} E={layer.e_size} heads={q_heads}/{heads} D={D} block={block} bound={bound} seed={seed}", flush=True)
    op = lowbit.NeighborAttentionOp(layer, q_heads, scale)
    out = op.forward(dev(q, device), kv, mirror)
    again = lowbit.NeighborAttentionOp(layer, q_heads, scale)
    assert torch.equal(again.forward(dev(q, device), kv, mirror), out) and torch.equal(again.lse, op.lse)
    want, lse, tol, ltol = ref.attention(q, ref.kv8_values(cache, scales, D, block), co.astype(np.int64), row, rows, q_heads, scale)
    got, glse = out.cpu().numpy().astype(np.float64), op.lse.cpu().numpy().astype(np.float64)
    nothing = np.isinf(lse)
    assert (np.isinf(glse) == nothing).all() and (glse[nothing] < 0).all()
    assert (got.reshape(Vd, q_heads, D)[nothing] == 0).all()
    assert (np.abs(glse[~nothing] - lse[~nothing]) <= ltol[~nothing]).all()
    worst = (np.abs(got - want) / np.maximum(tol, 1e-300)).max(initial=0.0)
    assert worst <= 1.0, f"{worst:.3g} of the tolerance"


HEADS = [(1, 1, 1), (1, 1, 16), (4, 4, 32), (8, 2, 64), (3, 3, 20), (6, 2, 47), (5, 1, 96), (10, 2, 128), (16, 8, 200), (2, 2, 256),
         (8, 8, 256), (12, 3, 8)]


@pytest.mark.parametrize("q_heads,heads,D", HEADS)
@pytest.mark.parametrize("bound", [0, 12])
def test_heads_and_widths(device, q_heads, heads, D, bound):
    degrees = [0, 1, 2, 3, 0, 0, 12, 7, 8, 9, 1, 0]
    check(device, degrees, 60, q_heads, heads, D, 16, seed=D + heads, bound=bound)


@pytest.mark.parametrize("degrees,bound", [
    ([1], 1), ([0], 0), ([300], 0), ([5000], 0), ([300], 256), ([0] * 500, 0), ([0] * 500, 5), ([1] * 1000, 0),
    ([0, 0, 900, 0, 0, 1, 2, 3, 4000, 0, 63, 64, 65, 0], 0), ([61, 63, 62, 64, 1, 0, 65, 127, 128, 129] * 8, 0),
    ([25] * 200, 25), ([31, 32, 33, 200, 256, 255], 256), (list(range(0, 130)), 0)])
def test_degrees(device, degrees, bound):
    check(device, degrees, 500, 4, 4, 32, 16, seed=len(degrees), bound=bound, missing=0.1)


@pytest.mark.parametrize("bound", [0, 40])
def test_neighbours_that_are_not_cached(device, bound):
    """Most neighbours missing, so whole destinations are left empty; rows from 90 of 150 on are beyond the cache's end."""
    check(device, [0, 1, 1, 2, 3, 40, 5, 6, 1, 1, 33], 150, 4, 2, 32, 4, missing=0.7, bound=bound, rows=90)
    check(device, [7, 8, 9], 150, 4, 2, 32, 4, missing=1.1, bound=bound)
    check(device, [7, 8, 9], 150, 4, 2, 32, 4, bound=bound, rows=0)


@pytest.mark.parametrize("block", [1, 2, 64, 1024])
def test_blocks_of_rows(device, block):
    check(device, [20, 300, 4], 1500, 2, 1, 48, block, seed=block)


def test_offsets_that_do_not_begin_at_zero_and_local_sources(device):
    check(device, [5, 0, 70, 300, 2], 200, 4, 4, 32, 16, offset=37)
    check(device, [5, 0, 70, 30, 2], 200, 4, 4, 32, 16, offset=37, bound=80)
    check(device, [5, 0, 70, 300, 2], 200, 4, 4, 32, 16, mirrored=True, missing=0.2)
    check(device, [5, 0, 7, 25, 2], 200, 8, 2, 64, 16, mirrored=True, missing=0.2, bound=25)


@pytest.mark.parametrize("degrees,bound", [([3, 0, 40, 1], 0), ([3, 0, 4, 9, 16], 16), ([3, 0, 5, 700, 1] * 20, 0)])
@pytest.mark.parametrize("known", [True, False])
def test_local_sources_beyond_the_mirror(device, degrees, bound, known):
    """A block a destination, a walker a row, and spans: sources that the mirror does not have count for nothing.  Where its length is
    not passed that is 0xFFFFFFFF alone."""
    Vd, V, heads, D, n_local = len(degrees), 90, 2, 32, 37
    rng = np.random.default_rng(8)
    cache, scales = empty(V, heads, D, 16)
    ref.kv8_append(cache, scales, keys(V, heads * D, 1), keys(V, heads * D, 2), 0, D, 16)
    co, ri = graph_of(np.array(degrees), n_local, 4)
    ri[::3] = 0xFFFFFFFF
    if known:
        ri[1::7], ri[2::11] = n_local, 0x80000000
    mirror = rng.permutation(V)[:n_local].astype(np.uint32)
    row = np.where(ri < n_local, mirror[np.minimum(ri, n_local - 1)], np.uint32(0xFFFFFFFF))
    q = rng.standard_normal((Vd, heads * D)).astype(np.float32)
    want, lse, tol, ltol = ref.attention(q, ref.kv8_values(cache, scales, D, 16), co.astype(np.int64), row, V, heads, 0.125)
    layer = SampledLayer()
    layer.v_size, layer.e_size, layer.max_in_degree = Vd, ri.size, bound
    layer.dev_column_offset, layer.dev_row_indices = dev(co, device), dev(ri, device)
    kv, dq, dm = lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, 16), dev(q, device), dev(mirror, device)
    if known:
        op = lowbit.NeighborAttentionOp(layer, heads, 0.125)
        out, glse = op.forward(dq, kv, dm), op.lse
        none = op.forward(dq, kv, dm[:0])
        assert not none.any() and (op.lse == -math.inf).all()
    else:
        out, glse = torch.empty(Vd, heads * D, device=device), torch.empty(Vd, heads, device=device)
        size = call("nts_kv8_attention_work_bytes", Vd, ri.size, heads, D, bound)
        work = torch.empty(size, dtype=torch.uint8, device=device)
        call("nts_kv8_attention", ptr(out), ptr(glse), ptr(dq), ptr(kv.cache), ptr(kv.scales), ptr(layer.dev_column_offset),
             ptr(layer.dev_row_indices), ptr(dm), Vd, ri.size, V, heads, heads, D, 16, 0.125, bound, ptr(work), stream())
    out, glse = out.cpu().numpy(), glse.cpu().numpy()
    some = np.isfinite(lse)
    assert (np.abs(out - want) <= tol).all() and (np.isfinite(glse) == some).all()
    assert (np.abs(glse[some] - lse[some]) <= ltol[some]).all()


def test_the_whole_graph_and_a_builders_layers(device):
    """Attention over a FullGraphChunk, whose sources are vertices, and over the layers that a BatchBuilder makes of the same graph,
    whose `source` is the mirror; neighbours that are not cached among both."""
    V, heads, D, rows = 700, 2, 32, 650
    src, dst = (t.to(device) for t in synth.rmat_edges(V, 9000, seed=3, device=device, sort=True))
    cache, scales = empty(V, heads, D, 16)
    ref.kv8_append(cache, scales, keys(V, heads * D, 1), keys(V, heads * D, 2), 0, D, 16)
    kv = lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, 16, rows=rows)
    values, rng = ref.kv8_values(cache, scales, D, 16), np.random.default_rng(4)
    chunk = FullGraphChunk.from_edges(src, dst, V)
    builder = BatchBuilder(chunk.column_offset_gpu, chunk.row_indices_gpu, [5, 40], 64)
    batch = builder.sample(dev(rng.choice(V, 64, replace=False).astype(np.uint32), device), 1)
    for layer in (chunk, *batch):
        mirror = layer.dev_source if layer is not chunk else None
        q = rng.standard_normal((layer.v_size, heads * D)).astype(np.float32)
        op = lowbit.NeighborAttentionOp(layer, heads, 0.125)
        out = op.forward(dev(q, device), kv, mirror).cpu().numpy()
        co, ri = (a.cpu().numpy().view(np.uint32) for a in (layer.dev_c_o(), layer.dev_r_i()))
        row = ri if mirror is None else mirror.cpu().numpy().view(np.uint32)[ri]
        want, lse, tol, ltol = ref.attention(q, values, co.astype(np.int64), row, rows, heads, 0.125)
        assert (np.abs(out - want) <= tol).all()
        got, some = op.lse.cpu().numpy(), np.isfinite(lse)
        assert (np.isfinite(got) == some).all() and (np.abs(got[some] - lse[some]) <= ltol[some]).all()
    builder.close()


def test_peaked_and_flat_scores(device):
    """Scores of several hundred (one neighbour takes all) and all equal (a scale of 0)."""
    check(device, [30, 700, 1, 5], 300, 4, 2, 32, 16, spread=40.0)
    check(device, [30, 700, 1, 5], 300, 4, 2, 32, 16, scale=0.0)
    check(device, [30, 700, 1, 5], 300, 4, 2, 32, 16, scale=-0.3)


def test_a_nan_key_reaches_its_destinations_alone(device):
    heads, D, V, block = 2, 16, 64, 4
    cache, scales = empty(V, heads, D, block)
    k, v = keys(V, heads * D, 1), keys(V, heads * D, 2)
    k[9, 3] = np.nan
    ref.kv8_append(cache, scales, k, v, 0, D, block)
    for Vd, bound in ((3, 0), (3, 8), (80, 0)):
        co = np.array([0, 3, 6] + [8] * (Vd - 2), dtype=np.uint32)
        ri = np.array([1, 9, 2, 3, 4, 5, 8, 10], dtype=np.uint32)
        layer = SampledLayer()
        layer.v_size, layer.e_size, layer.max_in_degree = Vd, 8, bound
        layer.dev_column_offset, layer.dev_row_indices = dev(co, device), dev(ri, device)
        op = lowbit.NeighborAttentionOp(layer, heads)
        out = op.forward(torch.randn(Vd, heads * D, device=device), lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, block))
        nan = torch.isnan(out.view(Vd, heads, D)).cpu()
        assert nan[0, 0].all() and not nan[0, 1].any() and not nan[1:].any()
        assert torch.isnan(op.lse[0, 0]) and torch.isfinite(op.lse[1:3]).all()


@pytest.mark.parametrize("Vd,bound", [(3, 0), (3, 8), (80, 0)])
def test_scores_of_minus_infinity(device, Vd, bound):
    """A destination all of whose scores are -infinity is one without neighbours; +infinity is NaN, in its head alone."""
    heads, D, V = 2, 16, 32
    cache, scales = empty(V, heads, D, 4)
    ref.kv8_append(cache, scales, np.ones((V, heads * D), dtype=np.float32), keys(V, heads * D, 2), 0, D, 4)
    layer = SampledLayer()
    layer.v_size, layer.e_size, layer.max_in_degree = Vd, 8, bound
    layer.dev_column_offset = dev(np.array([0, 3, 6] + [8] * (Vd - 2), dtype=np.uint32), device)
    layer.dev_row_indices = dev(np.array([1, 9, 2, 3, 4, 5, 8, 10], dtype=np.uint32), device)
    q = torch.ones(Vd, heads * D, device=device)
    q[0, 3], q[1, D + 2] = -math.inf, math.inf
    op = lowbit.NeighborAttentionOp(layer, heads)
    out = op.forward(q, lowbit.Kv8Cache.over(dev(cache, device), dev(scales, device), D, 4)).view(Vd, heads, D).cpu()
    lse = op.lse.cpu()
    assert (out[0, 0] == 0).all() and lse[0, 0] == -math.inf
    assert torch.isnan(out[1, 1]).all()
    assert torch.isfinite(out[0, 1]).all() and torch.isfinite(out[1, 0]).all() and torch.isfinite(out[2]).all()
    assert torch.isfinite(lse[0, 1]) and torch.isfinite(lse[1, 0]) and torch.isfinite(lse[2]).all()


def test_without_the_logarithms_and_beyond_the_rows(device):
    """lse NULL; nothing is written behind the last destination's row."""
    heads, D, V = 4, 20, 100
    cache, scales = empty(V, heads, D, 16)
    ref.kv8_append(cache, scales, keys(V, heads * D, 1), keys(V, heads * D, 2), 0, D, 16)
    co, ri = graph_of([3, 0, 200, 5], V, 4)
    dc, ds, dco, dri = (dev(a, device) for a in (cache, scales, co, ri))
    q = torch.randn(4, heads * D, device=device)
    outs = []
    for bound in (0, 250):
        out = torch.full((6, heads * D), 9.0, device=device)
        size = call("nts_kv8_attention_work_bytes", 4, 208, heads, D, bound)
        work = torch.full((size + 64,), 0xEE, dtype=torch.uint8, device=device)
        call("nts_kv8_attention", ptr(out), 0, ptr(q), ptr(dc), ptr(ds), ptr(dco), ptr(dri), 0, 4, 208, V, heads, heads, D, 16,
             0.25, bound, ptr(work), stream())
        assert (out[4:] == 9.0).all() and (work[size:] == 0xEE).all()
        outs.append(out[:4])
    assert torch.allclose(outs[0], outs[1], rtol=1e-4, atol=1e-5)  # two ways of summing the same edges


def test_many_destinations(device):
    """More destinations and edges than one span takes, with hubs of thousands of edges between short rows."""
    rng = np.random.default_rng(5)
    degrees = rng.integers(0, 9, 3000)
    degrees[[0, 700, 2999]] = 9000, 20000, 3000
    check(device, degrees, 900, 2, 1, 16, 16, missing=0.05)


def test_a_cache_beyond_32_bits(device):
    """A cache of more than 2^32 bytes: rows near its end."""
    heads, D, block, V = 8, 64, 16, 4_300_000  # 1,024 bytes a row
    kv = lowbit.Kv8Cache(V, heads, D, block, device=device)
    kv.rows = V - 30
    k, v = keys(30, heads * D, 1), keys(30, heads * D, 2)
    kv.append(dev(k, device), dev(v, device))
    small, scales = empty(46, heads, D, block)
    first = (V - 30) % block  # the same place within a block
    ref.kv8_append(small, scales, k, v, first, D, block)
    assert (kv.cache[-30:].cpu().numpy() == small[first:first + 30]).all()
    local = np.concatenate([np.arange(30), [0, 29, 7]])
    for Vd, bound in ((2, 0), (2, 30), (70, 0), (70, 30)):
        co = np.array([0, 30] + [33] * (Vd - 1), dtype=np.uint32)
        layer = SampledLayer()
        layer.v_size, layer.e_size, layer.max_in_degree = Vd, 33, bound
        layer.dev_column_offset, layer.dev_row_indices = dev(co, device), dev((local + V - 30).astype(np.uint32), device)
        q = np.random.default_rng(3).standard_normal((Vd, heads * D)).astype(np.float32)
        got = lowbit.NeighborAttentionOp(layer, heads, 0.125).forward(dev(q, device), kv).cpu().numpy()
        want, _, tol, _ = ref.attention(q, ref.kv8_values(small, scales, D, block), co.astype(np.int64), local + first, 46, heads, 0.125)
        assert (np.abs(got - want) <= tol).all()


def test_captured_and_replayed_beside_other_streams(device):
    """Append and attention recorded into a graph, replayed with eager calls on another stream in between."""
    heads, D, V, Vd = 4, 32, 400, 90
    kv = lowbit.Kv8Cache(V, heads, D, 16, device=device)
    k, v, q = (torch.zeros(n, heads * D, device=device) for n in (V, V, Vd))
    co, ri = graph_of(np.r_[np.full(Vd - 1, 7), 900], V, 3, missing=0.1)
    layer = SampledLayer()
    layer.v_size, layer.e_size = Vd, ri.size
    layer.dev_column_offset, layer.dev_row_indices = dev(co, device), dev(ri, device)
    op = lowbit.NeighborAttentionOp(layer, heads)

    def run():
        kv.append(k, v, 0)
        return op.forward(q, kv), op.lse

    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        recorded = run()
    for seed in range(3):
        torch.manual_seed(seed)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device=device))
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            eager = [t.clone() for t in run()]
        torch.cuda.current_stream().wait_stream(other)
        for t in recorded:
            t.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, eager)), f"replay {seed}"


def test_a_layer_from_features_to_attention(device):
    """The operators as a layer uses them: features rounded to 4 bits, queries, keys and values as products on rows gathered
    by id, keys and values into the cache, attention of a sampled layer; against the same in 64 bits, on the device's own
    products (a product's rounding may move a key to the next 8-bit value)."""
    V, F, H, D, n = 600, 100, 4, 32, 50
    rng = np.random.default_rng(1)
    x = dev(rng.standard_normal((V, F)).astype(np.float32), device)
    table = lowbit.MxTable.quantize(x)
    wq, wk, wv = (lowbit.MxTable.quantize(dev((rng.standard_normal((H * D, F)) / 10).astype(np.float32), device)) for _ in range(3))
    batch = dev(rng.choice(V, n, replace=False).astype(np.uint32), device)
    q = lowbit.MxProductOp(batch).forward(table, wq)
    k, v = (lowbit.MxProductOp().forward(table, w) for w in (wk, wv))
    kv = lowbit.Kv8Cache(V, H, D, device=device)
    kv.append(k[:250], v[:250])
    kv.append(k[250:], v[250:])
    co, ri = graph_of(np.minimum(np.arange(n), 10), V, 2)
    mirror, local = np.unique(ri, return_inverse=True)
    layer = SampledLayer()
    layer.v_size, layer.e_size, layer.max_in_degree = n, ri.size, 10
    layer.dev_column_offset, layer.dev_row_indices = dev(co, device), dev(local.reshape(-1).astype(np.uint32), device)
    op = lowbit.NeighborAttentionOp(layer, H)
    out = op.forward(q, kv, dev(mirror, device)).cpu().numpy()
    cache, scales = empty(V, H, D, 16)
    ref.kv8_append(cache, scales, k[:250].cpu().numpy(), v[:250].cpu().numpy(), 0, D, 16)
    ref.kv8_append(cache, scales, k[250:].cpu().numpy(), v[250:].cpu().numpy(), 250, D, 16)
    assert (kv.cache.cpu().numpy() == cache).all() and (kv.scales.cpu().numpy() == scales).all()
    want, _, tol, _ = ref.attention(q.cpu().numpy(), ref.kv8_values(cache, scales, D, 16), co.astype(np.int64), ri, V, H,
                                    float(np.float32(D ** -0.5)))
    assert (np.abs(out - want) <= tol).all()
