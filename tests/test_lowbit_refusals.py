"""Arguments that the operators on vertex tables in few bits refuse, before any device work (no GPU), and the reference
implementations that their GPU tests compare with."""
import numpy as np
import pytest
import torch

import lowbit_ref as ref
from neutronbench_amd import abi, batch, lowbit
from neutronbench_amd.layout import SampledLayer

P = 4096  # stands for a device pointer with any alignment that is asked for: refused calls never follow it
BIG = (1 << 17) + 1


def refused(text, name, *args):
    assert abi.status(name, *args) == abi.NTS_ERR_INVALID
    assert text in abi.last_error() and name in abi.last_error()


def test_quantize():
    refused("F is 0", "nts_mxfp4_quantize", P, P, P, 4, 0, 0)
    refused("above 2^17", "nts_mxfp4_quantize", P, P, P, 4, BIG, 0)
    for args in ((0, P, P), (P, 0, P), (P, P, 0)):
        refused("null pointer", "nts_mxfp4_quantize", *args, 4, 8, 0)
    refused("alignment", "nts_mxfp4_quantize", P + 8, P, P, 4, 8, 0)
    refused("alignment", "nts_mxfp4_quantize", P, P + 2, P, 4, 8, 0)
    refused("2^32 blocks", "nts_mxfp4_quantize", P, P, P, 0x80000000, 33, 0)
    assert abi.status("nts_mxfp4_quantize", 0, 0, 0, 0, 8, 0) == abi.NTS_OK


def test_gather():
    refused("F is 0", "nts_gather_rows_mxfp4", P, P, P, 5, P, 4, 0, 0)
    refused("above 2^17", "nts_gather_rows_mxfp4", P, P, P, 5, P, 4, BIG, 0)
    for args in ((0, P, P), (P, 0, P), (P, P, 0)):
        refused("null pointer", "nts_gather_rows_mxfp4", *args, 5, P, 4, 8, 0)
    refused("alignment", "nts_gather_rows_mxfp4", P, P + 4, P, 5, P, 4, 8, 0)
    assert abi.status("nts_gather_rows_mxfp4", 0, 0, 0, 5, 0, 0, 8, 0) == abi.NTS_OK


def test_product():
    name = "nts_mxfp4_product"
    for N, F in ((0, 8), (8, 0), (BIG, 8), (8, BIG)):
        refused("N or F", name, P, P, P, 5, 0, 4, P, P, N, F, 0, 0)
    for hole in (0, 1, 2, 6, 7):
        args = [P, P, P, 5, 0, 4, P, P, 8, 8, 0, 0]
        args[hole] = 0
        refused("null pointer", name, *args)
    refused("alignment", name, P, P, P, 5, 0, 4, P + 8, P, 8, 8, 0, 0)
    assert abi.status(name, 0, 0, 0, 5, 0, 0, 0, 0, 8, 8, 0, 0) == abi.NTS_OK


def test_gradients():
    name = "nts_mxfp4_product_grad_rows"
    for N, F in ((0, 8), (8, 0), (BIG, 8), (8, BIG)):
        refused("N or F", name, P, P, P, P, 4, N, F, 0, 0)
    for hole in range(4):
        args = [P, P, P, P, 4, 8, 8, 0, 0]
        args[hole] = 0
        refused("null pointer", name, *args)
    refused("alignment", name, P, P, P, P + 2, 4, 8, 8, 0, 0)
    assert abi.status(name, 0, 0, 0, 0, 0, 8, 8, 0, 0) == abi.NTS_OK
    name = "nts_mxfp4_product_grad_weight"
    for N, F in ((0, 8), (8, 0), (BIG, 8), (8, BIG)):
        refused("N or F", name, P, P, P, P, 5, 0, 4, N, F, 0, P, 0)
        assert abi.call(name + "_work_bytes", 4, N, F) == 0
    for hole in range(4):
        args = [P, P, P, P, 5, 0, 4, 8, 8, 0, P, 0]
        args[hole] = 0
        refused("null pointer", name, *args)
    refused("alignment", name, P, P, P + 8, P, 5, 0, 4, 8, 8, 0, P, 0)
    assert abi.call(name + "_work_bytes", 100000, 8, 8) > 0
    refused("work", name, P, P, P, P, 5, 0, 100000, 8, 8, 0, 0, 0)


def test_append():
    name = "nts_kv8_append"
    for heads, width, block, text in ((0, 8, 16, "heads"), (1025, 8, 16, "heads"), (4, 0, 16, "width"), (4, 257, 16, "width"),
                                      (4, 8, 0, "block_rows"), (4, 8, 12, "block_rows"), (4, 8, 2048, "block_rows")):
        refused(text, name, P, P, P, P, 0, 4, 100, heads, width, block, 0)
    refused("capacity", name, P, P, P, P, 97, 4, 100, 4, 8, 16, 0)
    refused("capacity", name, P, P, P, P, 101, 0, 100, 4, 8, 16, 0)
    refused("capacity", name, P, P, P, P, 8, 0xFFFFFFFF, 100, 4, 8, 16, 0)
    refused("alignment", name, P + 8, P, P, P, 0, 4, 100, 4, 8, 16, 0)
    for hole in range(4):
        args = [P, P, P, P, 0, 4, 100, 4, 8, 16, 0]
        args[hole] = 0
        refused("null pointer", name, *args)
    assert abi.status(name, 0, 0, 0, 0, 100, 0, 100, 4, 8, 16, 0) == abi.NTS_OK


def attention(**changed):
    args = dict(out=P, lse=P, q=P, cache=P, scales=P, co=P, ri=P, mirror=0, Vd=4, edges=9, cache_rows=50, q_heads=8, heads=4,
                width=16, block_rows=16, score_scale=1.0, max_degree=0, work=P, stream=0)
    assert not set(changed) - set(args)
    return list({**args, **changed}.values())


def test_attention():
    name = "nts_kv8_attention"
    for text, changed in (("heads", dict(heads=0)), ("heads", dict(heads=1025)), ("width", dict(width=0)),
                          ("width", dict(width=257)), ("block_rows", dict(block_rows=48)), ("alignment", dict(cache=P + 4)),
                          ("q_heads", dict(q_heads=0)), ("q_heads", dict(q_heads=6)), ("q_heads", dict(q_heads=1028)),
                          ("edges", dict(edges=0xFFFF0001)), ("work", dict(work=0, edges=100000)),
                          ("work", dict(work=P + 8, Vd=1000)), ("work", dict(work=0, edges=100000, max_degree=257))):
        refused(text, name, *attention(**changed))
    for hole in ("out", "q", "cache", "scales", "co", "ri"):
        refused("null pointer", name, *attention(**{hole: 0}))
    assert abi.status(name, *attention(Vd=0, out=0, q=0, co=0)) == abi.NTS_OK
    sizes = abi.call(name + "_work_bytes", 1000, 100000, 8, 32, 0)
    assert sizes > 0 and abi.call(name + "_work_bytes", 1000, 100000, 8, 32, 257) == sizes
    assert abi.call(name + "_work_bytes", 64, 4096, 8, 32, 0) == 0  # a block of wavefronts for each destination
    assert abi.call(name + "_work_bytes", 64, 4097, 8, 32, 0) > 0 and abi.call(name + "_work_bytes", 65, 4096, 8, 32, 0) > 0
    for bad in ((8, 32, 25), (0, 32, 0), (8, 0, 0), (8, 257, 0)):
        assert abi.call(name + "_work_bytes", 1000, 100000, *bad) == 0


def test_attention_by_local_sources():
    """The same refusals where the mirror's length is known, and a mirror that is not there."""
    name = "nts_kv8_attention_local"

    def local(mirror=P, mirror_rows=40, **changed):
        args = attention(**changed)
        return args[:7] + [mirror, mirror_rows] + args[8:]

    for text, changed in (("heads", dict(heads=0)), ("width", dict(width=257)), ("block_rows", dict(block_rows=48)),
                          ("alignment", dict(cache=P + 4)), ("q_heads", dict(q_heads=6)), ("edges", dict(edges=0xFFFF0001)),
                          ("work", dict(work=0, edges=100000)), ("null pointer", dict(mirror=0))):
        refused(text, name, *local(**changed))
    for hole in ("out", "q", "cache", "scales", "co", "ri"):
        refused("null pointer", name, *local(**{hole: 0}))
    assert abi.status(name, *local(Vd=0, mirror=0, mirror_rows=0)) == abi.NTS_OK


def table(rows, width):
    codes, scales = lowbit.mx_shapes(rows, width)
    return lowbit.MxTable(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), width)


def test_python_objects_check_their_operands():
    codes, scales = (torch.zeros(s, dtype=torch.uint8) for s in lowbit.mx_shapes(6, 100))
    for bad in ((codes[:, :32], scales, 100), (codes, scales[:5], 100), (codes.to(torch.int8), scales, 100), (codes, scales, 140)):
        with pytest.raises(ValueError):
            lowbit.MxTable(*bad)
    with pytest.raises(ValueError):
        lowbit.MxTable.quantize(torch.zeros(4, 8, dtype=torch.float64))
    with pytest.raises(ValueError):
        lowbit.MxTable.quantize(torch.zeros(4, 8).t())
    for ids in (torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            table(6, 100).gather(ids)
        with pytest.raises(ValueError):
            lowbit.MxProductOp(ids)
    with pytest.raises(ValueError):
        table(6, 100).gather(out=torch.zeros(5, 100))
    with pytest.raises(ValueError):
        lowbit.MxProductOp().forward(table(6, 100), table(6, 96))
    cache, scales = torch.zeros(40, 2, 3, 32, dtype=torch.uint8), torch.zeros(3, 2, 3, dtype=torch.uint8)
    kv = lowbit.Kv8Cache.over(cache, scales, 20, 16, rows=10)
    for bad in ((cache[:, :, :0], scales[:, :, :0], 20, 16), (cache, scales, 0, 16), (cache[:10], scales, 20, 5), (cache, scales, 33, 16), (cache, scales, 20, 8), (cache[:, :1], scales, 20, 16), (cache[:, 0], scales, 20, 16),
                (cache, scales, 20, 0)):
        with pytest.raises(ValueError):
            lowbit.Kv8Cache.over(*bad)
    with pytest.raises(ValueError):
        lowbit.Kv8Cache.over(cache, scales, 20, 16, rows=41)
    k = torch.zeros(5, 60)
    for bad in ((k, k[:4], 0), (k, k, 11), (k, k, 36), (k[:, :59], k, 0), (k.double(), k, 0)):
        with pytest.raises(ValueError):
            kv.append(*bad)
    layer = SampledLayer()
    layer.v_size, layer.dev_column_offset, layer.dev_row_indices = 4, torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    with pytest.raises(ValueError):
        lowbit.MxProductOp().backward(torch.zeros(4, 8))
    with pytest.raises(ValueError):  # five offsets for five destinations
        layer.v_size = 5
        lowbit.NeighborAttentionOp(layer, 6).forward(torch.zeros(5, 120), kv)
    layer.v_size, layer.e_size = 4, 1
    with pytest.raises(ValueError):  # fewer edges than the layer says
        lowbit.NeighborAttentionOp(layer, 6).forward(torch.zeros(4, 120), kv)
    layer.e_size = 0
    for q_heads, q in ((6, torch.zeros(5, 120)), (6, torch.zeros(4, 100)), (4, torch.zeros(4, 80))):
        with pytest.raises(ValueError):
            lowbit.NeighborAttentionOp(layer, q_heads).forward(q, kv)


def test_a_caches_shape_is_checked_before_it_is_made():
    for heads, width, block in ((0, 8, 16), (1025, 8, 16), (4, 0, 16), (4, 257, 16), (4, 8, 0), (4, 8, 12), (4, 8, 2048), (4, 8, -4)):
        with pytest.raises(ValueError):
            lowbit.Kv8Cache(1 << 50, heads, width, block, device="cpu")
    with pytest.raises(ValueError):  # blocks of more rows than any call takes
        lowbit.Kv8Cache.over(torch.zeros(10, 2, 1, 16, dtype=torch.uint8), torch.zeros(1, 2, 1, dtype=torch.uint8), 16, 2048)
    assert lowbit.Kv8Cache(40, 3, 20, 16, device="cpu").rows == 0


def test_a_batchs_rows_need_an_output_of_their_size():
    """load_feature_mxfp4 against outputs that are too narrow, too wide, too short, of another type or strided, and layers whose
    id array is shorter than they say."""
    layer = SampledLayer()
    layer.src_size, layer.dev_source = 4, torch.zeros(4, dtype=torch.int32)
    good = torch.zeros(4, 100)
    for bad in (good[:, :96], torch.zeros(4, 104), good[:3], good.double(), torch.zeros(100, 4).t(), torch.zeros(400)):
        with pytest.raises(ValueError):
            batch.load_feature_mxfp4(None, layer, bad, table(6, 100))
    for ids in (torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)[::2]):
        layer.dev_source = ids
        with pytest.raises(ValueError):
            batch.load_feature_mxfp4(None, layer, good, table(6, 100))


def test_reference_rounding():
    """The reference's own rounding against torch's conversion to e4m3, and its 4-bit grid against all halves and quarters."""
    y = np.concatenate([np.linspace(0, 448, 20011), ref.E4M3[:127], (ref.E4M3[:126] + ref.E4M3[1:127]) / 2])
    want = torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (ref.nearest(ref.E4M3[:127], y.astype(np.float32)) == want).all()
    x = np.zeros((1, 32), dtype=np.float32)
    x[0, :13] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 0.24, 0.26, 7.9]
    codes, scales = ref.mx_quantize(x)
    assert scales[0, 0] == 127
    assert ref.mx_values(codes, scales, 13)[0].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, 0, 0.5, 6]
