"""4-bit rows and the products on them against plain implementations in 64 bits.

Rounding, gathering: bit-exact.  Products: every term is exact, R of them are summed in 32 bits in some order, so a result
is off by at most R * 2^-23 of the sum of the terms' magnitudes (2^-24 a step, doubled for sums that cut off instead of
rounding); the gradients sum three exact terms for one.  Sums whose magnitudes lie below 2^-100 may lose bits
below 2^-126."""
import ctypes

import numpy as np
import pytest
import torch

import lowbit_ref as ref
from gpu_util import dev, stream
from neutronbench_amd import epoch, lowbit, synth
from neutronbench_amd.abi import call, ptr
from neutronbench_amd.batch import BatchBuilder, load_feature_mxfp4
from neutronbench_amd.stream import CudaStream

pytestmark = pytest.mark.gpu


def rows_of(n, F, seed, special=True):
    """Rows with blocks of many sizes, ties, zeros of both signs and, with `special`, blocks of denormals, of the largest
    floats, infinities and NaN."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, F)) * np.exp2(rng.integers(-20, 20, (n, 1)))).astype(np.float32)
    flat = x.reshape(-1)
    ties = rng.random(flat.size) < 0.3
    flat[ties] = (rng.integers(-32, 33, ties.sum()) / 4).astype(np.float32)
    flat[rng.random(flat.size) < 0.05] = -0.0
    if n > 2:
        x[1] = 0.0
    if special and n > 8:
        x[2, :] = np.float32(1e-45) * rng.integers(0, 9, F)
        x[3, :] = np.float32(2.0 ** -126) * rng.random(F).astype(np.float32)
        x[4, :] = np.float32(3.4028235e38) * rng.choice([-1, 1, 0.5], F).astype(np.float32)
        x[5, F // 2] = np.inf
        x[6, F - 1] = np.nan
        x[7, 0] = -np.inf
    return x


def same(got, want):
    assert got.shape == want.shape and ((got == want) | (np.isnan(got) & np.isnan(want))).all()


def table_of(x, device):
    codes, scales = ref.mx_quantize(x)
    return codes, scales, lowbit.MxTable(dev(codes, device), dev(scales, device), x.shape[1])


@pytest.mark.parametrize("n,F", [(1, 1), (9, 2), (10, 31), (33, 32), (70, 33), (1000, 100), (257, 128), (40, 602), (12, 1433)])
def test_quantize(device, n, F):
    x = rows_of(n, F, seed=n + F)
    t = lowbit.MxTable.quantize(dev(x, device))
    codes, scales = ref.mx_quantize(x)
    assert (t.codes.cpu().numpy() == codes).all()
    assert (t.scales.cpu().numpy() == scales).all()
    same(t.gather().cpu().numpy(), ref.mx_values(codes, scales, F).astype(np.float32))


def test_quantize_writes_nothing_beyond_its_rows(device):
    F, n = 70, 21
    x = dev(rows_of(n, F, 3), device)
    (_, cw), (_, sw) = lowbit.mx_shapes(n, F)
    codes = torch.full((n + 2, cw), 0xAB, dtype=torch.uint8, device=device)
    scales = torch.full((n + 2, sw), 0xAB, dtype=torch.uint8, device=device)
    call("nts_mxfp4_quantize", ptr(codes), ptr(scales), ptr(x), n, F, stream())
    assert (codes[n:] == 0xAB).all() and (scales[n:] == 0xAB).all()
    want = ref.mx_quantize(x.cpu().numpy())
    assert (codes[:n].cpu().numpy() == want[0]).all() and (scales[:n].cpu().numpy() == want[1]).all()


def test_gather_every_code_under_every_scale(device):
    codes = np.tile(np.arange(0, 256, 17, dtype=np.uint8), (256, 1))  # both halves of a byte take every code
    codes = np.concatenate([codes, codes[:, :0:-1], codes[:, :1]], 1)[:, :16]
    codes[:, 8:] = np.arange(256, dtype=np.uint8)[:, None] ^ np.arange(8, dtype=np.uint8) * 29
    scales = np.zeros((256, 4), dtype=np.uint8)
    scales[:, 0] = np.arange(256)
    t = lowbit.MxTable(dev(codes, device), dev(scales, device), 32)
    with np.errstate(over="ignore"):
        want = ref.mx_values(codes, scales, 32).astype(np.float32)
    got = t.gather().cpu().numpy()
    same(got, want)
    assert (np.signbit(got) == np.signbit(want))[~np.isnan(want)].all()


@pytest.mark.parametrize("F", [1, 7, 8, 9, 32, 100, 128, 602])
def test_gather_by_id(device, F):
    x = rows_of(300, F, seed=F)
    codes, scales, t = table_of(x, device)
    rng = np.random.default_rng(F)
    ids = rng.integers(0, 300, 777).astype(np.uint32)
    ids[::50] = 0xFFFFFFFF
    ids[1::50] = 300
    out = torch.full((779, F), 7.0, device=device)
    got = t.gather(dev(ids, device), out=out[:777])
    same(got.cpu().numpy(), ref.mx_rows(codes, scales, F, ids).astype(np.float32))
    assert (out[777:] == 7.0).all()


@pytest.mark.parametrize("F", [1, 6, 32, 47, 64, 100, 130, 256, 602, 1433])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_gather_to_any_float(device, F, shift):
    """An output that begins at any multiple of four bytes, the whole table with its last row, large enough to be written past
    the caches and small."""
    for V, n in ((50, 50), (70, 68_000_000 // F)):
        x = rows_of(V, F, seed=F + shift)
        codes, scales, t = table_of(x, device)
        ids = np.random.default_rng(shift).integers(0, V + 1, n).astype(np.uint32)
        ids[-1] = V - 1
        out = torch.full((n * F + 8,), 7.0, device=device)
        call("nts_gather_rows_mxfp4", ptr(out[shift:]), ptr(t.codes), ptr(t.scales), V, ptr(dev(ids, device)), n, F, stream())
        values = np.concatenate([ref.mx_values(codes, scales, F).astype(np.float32), np.zeros((1, F), dtype=np.float32)])
        want = torch.from_numpy(values).to(device)[torch.from_numpy(ids.astype(np.int64)).to(device)].reshape(-1)
        got = out[shift:shift + n * F]
        assert ((got == want) | (torch.isnan(got) & torch.isnan(want))).all()
        assert (out[:shift] == 7.0).all() and (out[shift + n * F:] == 7.0).all()


@pytest.mark.parametrize("F", [288, 384, 512, 1024, 1280])
@pytest.mark.parametrize("by_id", [True, False])
def test_gather_of_rows_of_whole_lines(device, F, by_id):
    """Large outputs of rows that fill whole lines, which pieces of the output may begin and end within."""
    V, n = 50, 9_000_000 // F
    codes, scales, t = table_of(rows_of(V, F, seed=F), device)
    values = np.concatenate([ref.mx_values(codes, scales, F).astype(np.float32), np.zeros((1, F), dtype=np.float32)])
    ids = np.random.default_rng(F).integers(0, V + 1, n) if by_id else np.minimum(np.arange(n), V)
    out = torch.full((n + 1, F), 7.0, device=device)
    dids = dev(ids.astype(np.uint32), device) if by_id else None
    call("nts_gather_rows_mxfp4", ptr(out), ptr(t.codes), ptr(t.scales), V, ptr(dids), n, F, stream())
    want = torch.from_numpy(values).to(device)[torch.from_numpy(ids).to(device)]
    assert ((out[:n] == want) | (torch.isnan(out[:n]) & torch.isnan(want))).all() and (out[n] == 7.0).all()


def test_gather_from_mapped_host_memory(device):
    F, V = 100, 5000
    x = rows_of(V, F, seed=5)
    codes, scales, _ = table_of(x, device)
    host = ctypes.c_void_p()
    call("nts_malloc_pinned_mapped", ctypes.byref(host), codes.nbytes)
    ctypes.memmove(host.value, codes.ctypes.data, codes.nbytes)
    alias = ctypes.c_void_p()
    call("nts_host_get_device_ptr", ctypes.byref(alias), host.value)
    ids = np.random.default_rng(6).integers(0, V, 20000).astype(np.uint32)
    dids, dscales = dev(ids, device), dev(scales, device)
    out = torch.empty(len(ids), F, device=device)
    call("nts_gather_rows_mxfp4", ptr(out), alias.value, ptr(dscales), V, ptr(dids), len(ids), F, stream())
    torch.cuda.synchronize()
    same(out.cpu().numpy(), ref.mx_rows(codes, scales, F, ids).astype(np.float32))
    call("nts_free_pinned", host.value)


def close(got, want, scale, terms):
    got = got.cpu().numpy().astype(np.float64)
    bound = terms * 2.0 ** -23 * scale + 2.0 ** -120
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{bad.sum()} of {bad.size} values, worst {np.nanmax(np.abs(got - want) / bound):.3g} of the bound"


PRODUCTS = [(1, 1, 1), (1, 256, 602), (2, 47, 100), (16, 16, 128), (17, 65, 129), (33, 64, 32), (100, 128, 100), (257, 130, 260),
            (300, 256, 602), (1000, 40, 128), (129, 513, 1433), (700, 300, 4100)]


@pytest.mark.parametrize("n,N,F", PRODUCTS)
@pytest.mark.parametrize("accumulate", [0, 1])
def test_product(device, n, N, F, accumulate):
    xa, xw = rows_of(200, F, n + F, special=False), rows_of(N, F, n + N, special=False)
    ca, sa, a = table_of(xa, device)
    cw, sw, w = table_of(xw, device)
    ids = np.random.default_rng(n).integers(0, 200, n).astype(np.uint32)
    ids[3::11] = 0xFFFFFFFF
    x, wv = ref.mx_rows(ca, sa, F, ids), ref.mx_values(cw, sw, F)
    start = np.random.default_rng(N).standard_normal((n, N)).astype(np.float32)
    out = torch.full((n + 1, N), 3.0, device=device)
    out[:n] = dev(start, device)
    dids = dev(ids, device)
    call("nts_mxfp4_product", ptr(out), ptr(a.codes), ptr(a.scales), 200, ptr(dids), n, ptr(w.codes), ptr(w.scales), N, F,
         accumulate, stream())
    want, scale = x @ wv.T, np.abs(x) @ np.abs(wv).T
    if accumulate:
        want, scale = want + start, scale + np.abs(start)
    close(out[:n], want, scale, F + 1)
    assert (out[n:] == 3.0).all()


@pytest.mark.parametrize("n,N,F,accumulate", [(66001, 1030, 1001, 0), (65600, 1024, 1056, 1), (40000, 1793, 2048, 0), (20100, 1797, 2100, 1)])
def test_product_in_the_larger_tiles(device, n, N, F, accumulate):
    """Against 64-bit products on the device, whose operands torch reads from the same rows."""
    V = 300
    ca, sa, a = table_of(rows_of(V, F, n, special=False), device)
    cw, sw, w = table_of(rows_of(N, F, N, special=False), device)
    ids = np.random.default_rng(n).integers(0, V, n).astype(np.uint32)
    ids[7::1000] = 0xFFFFFFFF
    dids = dev(ids, device)
    x = torch.from_numpy(np.concatenate([ref.mx_values(ca, sa, F), np.zeros((1, F))])).to(device)
    x, wv = x[torch.from_numpy(np.minimum(ids, V).astype(np.int64)).to(device)], torch.from_numpy(ref.mx_values(cw, sw, F)).to(device)
    start = torch.randn(n, N, device=device)
    out = start.clone()
    call("nts_mxfp4_product", ptr(out), ptr(a.codes), ptr(a.scales), V, ptr(dids), n, ptr(w.codes), ptr(w.scales), N, F,
         accumulate, stream())
    want, scale = torch.mm(x, wv.t().contiguous()), torch.mm(x.abs(), wv.abs().t().contiguous())
    if accumulate:
        want, scale = want + start, scale + start.abs()
    assert bool(((out.double() - want).abs() <= (F + 1) * 2.0 ** -23 * scale + 2.0 ** -120).all())


@pytest.mark.parametrize("n,V,N,F", [(70, 1, 1, 1), (200, 1, 1, 32), (200, 1, 2, 100), (200, 0, 3, 300), (130, 2, 1, 1433), (90, 1, 1, 8300),
                                     (262200, 2, 1, 1000), (131100, 1, 2, 2100)])
def test_product_of_tables_of_few_rows(device, n, V, N, F):
    """Many rows by id from tables that are shorter than a stage of the product's; ids that the table does not have give zeros."""
    xw = rows_of(N, F, n + N, special=False)
    cw, sw, w = table_of(xw, device)
    ids = np.random.default_rng(n).integers(0, max(V, 1), n).astype(np.uint32)
    ids[3::7] = 0xFFFFFFFF
    ids[5::7] = V
    if V:
        ca, sa, a = table_of(rows_of(V, F, n + F, special=False), device)
        x = ref.mx_values(ca, sa, F)
    else:
        a = lowbit.MxTable(*(torch.empty(s, dtype=torch.uint8, device=device) for s in lowbit.mx_shapes(0, F)), F)
        x = np.zeros((0, F))
    x, wv = np.concatenate([x, np.zeros((1, F))])[np.minimum(ids, V)], ref.mx_values(cw, sw, F)
    got = lowbit.MxProductOp(dev(ids, device)).forward(a, w)
    close(got, x @ wv.T, np.abs(x) @ np.abs(wv).T, F)
    assert not got.cpu().numpy()[ids >= V].any()


def test_product_without_ids_is_the_whole_table(device):
    ca, sa, a = table_of(rows_of(130, 96, 1, special=False), device)
    cw, sw, w = table_of(rows_of(50, 96, 2, special=False), device)
    got = lowbit.MxProductOp().forward(a, w)
    x, wv = ref.mx_values(ca, sa, 96), ref.mx_values(cw, sw, 96)
    close(got, x @ wv.T, np.abs(x) @ np.abs(wv).T, 96)


@pytest.mark.parametrize("n,N", [(40, 24), (700, 600)])
def test_product_of_far_scales_and_nan_blocks(device, n, N):
    """Scales from 2^-60 to 2^60 within a row; a NaN block makes its row or column NaN and nothing else."""
    rng = np.random.default_rng(9)
    F = 300
    ca, sa, _ = table_of(rows_of(n, F, 3, special=False), device)
    cw, sw, _ = table_of(rows_of(N, F, 4, special=False), device)
    sa[:, :10] = rng.integers(67, 188, (n, 10))
    sw[:, :10] = rng.integers(67, 188, (N, 10))
    x, w = ref.mx_values(ca, sa, F), ref.mx_values(cw, sw, F)
    sa[5, 9], sa[6, 0], sw[7, 4] = 255, 255, 255
    sa[:, 10:] = 255  # bytes behind the last block belong to none
    sw[:, 10:] = 255
    a = lowbit.MxTable(dev(ca, device), dev(sa, device), F)
    got = lowbit.MxProductOp().forward(a, lowbit.MxTable(dev(cw, device), dev(sw, device), F)).cpu()
    nan = np.zeros((n, N), dtype=bool)
    nan[5:7], nan[:, 7] = True, True
    assert (np.isnan(got.numpy()) == nan).all()
    keep_r, keep_c = np.arange(n) > 6, np.arange(N) > 7
    close(got[keep_r][:, keep_c], (x @ w.T)[keep_r][:, keep_c], (np.abs(x) @ np.abs(w).T)[keep_r][:, keep_c], F)


GRADS = [(1, 1, 1), (1, 256, 602), (31, 33, 65), (64, 64, 64), (65, 47, 100), (100, 3, 130), (513, 128, 128), (5000, 40, 100),
         (1111, 260, 33), (20000, 17, 602)]


@pytest.mark.parametrize("n,N,F", GRADS)
@pytest.mark.parametrize("accumulate", [0, 1])
def test_gradients(device, n, N, F, accumulate):
    xa, xw = rows_of(150, F, n + F, special=False), rows_of(N, F, n + N, special=False)
    ca, sa, a = table_of(xa, device)
    cw, sw, w = table_of(xw, device)
    rng = np.random.default_rng(n + 1)
    ids = rng.integers(0, 150, n).astype(np.uint32)
    ids[4::9] = 150
    g = (rng.standard_normal((n, N)) * np.exp2(rng.integers(-12, 12, (n, 1)))).astype(np.float32)
    x, wv, g64 = ref.mx_rows(ca, sa, F, ids), ref.mx_values(cw, sw, F), g.astype(np.float64)
    gx0, gw0 = rng.standard_normal((n, F)).astype(np.float32), rng.standard_normal((N, F)).astype(np.float32)
    gx, gw, dg, dids = (dev(v, device) for v in (gx0, gw0, g, ids))
    call("nts_mxfp4_product_grad_rows", ptr(gx), ptr(dg), ptr(w.codes), ptr(w.scales), n, N, F, accumulate, stream())
    work = torch.full((call("nts_mxfp4_product_grad_weight_work_bytes", n, N, F),), 0xFF, dtype=torch.uint8, device=device)
    call("nts_mxfp4_product_grad_weight", ptr(gw), ptr(dg), ptr(a.codes), ptr(a.scales), 150, ptr(dids), n, N, F, accumulate,
         ptr(work) if work.numel() else 0, stream())
    for got, start, p, q, terms in ((gx, gx0, g64, wv, N), (gw, gw0, g64.T, x, n)):
        want, scale = p @ q, np.abs(p) @ np.abs(q)
        if accumulate:
            want, scale = want + start, scale + np.abs(start)
        close(got, want, scale, 3 * terms + 1100)


@pytest.mark.parametrize("n,N,F", GRADS)
@pytest.mark.parametrize("accumulate", [0, 1])
def test_gradients_within_their_own_roundings(device, n, N, F, accumulate):
    """A value of g is three exact terms whose magnitudes add up to its own, so a result is a chain of at most 3 terms roundings
    within a part, one for each part and one for what was there: each off by 2^-23 of the magnitudes at most."""
    ca, sa, a = table_of(rows_of(150, F, n + F, special=False), device)
    cw, sw, w = table_of(rows_of(N, F, n + N, special=False), device)
    rng = np.random.default_rng(n + 2)
    ids = rng.integers(0, 150, n).astype(np.uint32)
    g = rng.standard_normal((n, N)).astype(np.float32)
    gx0, gw0 = rng.standard_normal((n, F)).astype(np.float32), rng.standard_normal((N, F)).astype(np.float32)
    gx, gw, dg, dids = (dev(v, device) for v in (gx0, gw0, g, ids))
    call("nts_mxfp4_product_grad_rows", ptr(gx), ptr(dg), ptr(w.codes), ptr(w.scales), n, N, F, accumulate, stream())
    size = call("nts_mxfp4_product_grad_weight_work_bytes", n, N, F)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    call("nts_mxfp4_product_grad_weight", ptr(gw), ptr(dg), ptr(a.codes), ptr(a.scales), 150, ptr(dids), n, N, F, accumulate,
         ptr(work), stream())
    x, wv, g64 = ref.mx_rows(ca, sa, F, ids), ref.mx_values(cw, sw, F), g.astype(np.float64)
    for got, start, p, q, steps in ((gx, gx0, g64, wv, 3 * N + 1), (gw, gw0, g64.T, x, 3 * n + max(1, size // (4 * N * F)) + 1)):
        want, scale = p @ q, np.abs(p) @ np.abs(q)
        if accumulate:
            want, scale = want + start, scale + np.abs(start)
        close(got, want, scale, steps)


@pytest.mark.parametrize("n,N,F", [(1, 1, 1), (40, 33, 70), (70, 128, 128), (97, 200, 40), (600, 40, 130), (20000, 17, 100)])
@pytest.mark.parametrize("by_id", [True, False])
def test_gradients_keep_every_bit_of_g(device, n, N, F, by_id):
    """One term other than zero to a result, a power of two times a value of g whose 24 bits are in use: the gradient is that
    product, exactly."""
    rng = np.random.default_rng(n + N)
    power = lambda *shape: (rng.choice([-1.0, 1.0], shape) * np.exp2(rng.integers(0, 3, shape))).astype(np.float32)
    columns, term, row = np.arange(F), np.arange(F) * 5 % N, np.arange(F) * 7919 % n
    xw, xa = np.zeros((N, F), dtype=np.float32), np.zeros((n, F), dtype=np.float32)
    xw[term, columns], xa[row, columns] = power(F), power(F)
    g = rng.standard_normal((n, N)).astype(np.float32)
    g = (g.view(np.uint32) | 1).view(np.float32)
    ids = rng.permutation(n) if by_id else np.arange(n)
    stored = np.empty_like(xa)
    stored[ids] = xa
    ca, sa, a = table_of(stored, device)
    cw, sw, w = table_of(xw, device)
    assert (ref.mx_values(ca, sa, F) == stored).all() and (ref.mx_values(cw, sw, F) == xw).all()
    op = lowbit.MxProductOp(dev(ids.astype(np.uint32), device) if by_id else None)
    op.forward(a, w)
    gx = op.backward(dev(g, device)).cpu().numpy()
    assert (gx == g[:, term] * xw[term, columns]).all()
    assert (op.get_additional_grad().cpu().numpy() == g[row].T * xa[row, columns]).all()


@pytest.mark.parametrize("n", [32, 63, 96, 128, 160, 193, 600])
@pytest.mark.parametrize("V", [0, 1, 40, 700])
def test_gradient_of_the_weight_by_stages(device, n, V):
    """From one whole stage of rows on, without ids, and from tables that end before the last row."""
    N, F = 37, 70
    rng = np.random.default_rng(n + V)
    g = rng.standard_normal((n, N)).astype(np.float32)
    x = np.zeros((n, F))
    if V:
        ca, sa, a = table_of(rows_of(V, F, V, special=False), device)
        x[:V] = ref.mx_values(ca, sa, F)[:n]
    gw, dg = torch.full((N, F), 5.0, device=device), dev(g, device)
    work = torch.empty(call("nts_mxfp4_product_grad_weight_work_bytes", n, N, F), dtype=torch.uint8, device=device)
    call("nts_mxfp4_product_grad_weight", ptr(gw), ptr(dg), ptr(a.codes) if V else 0, ptr(a.scales) if V else 0, V, 0, n, N, F, 0,
         ptr(work) if work.numel() else 0, stream())
    close(gw, g.astype(np.float64).T @ x, np.abs(g).astype(np.float64).T @ np.abs(x), 3 * n + 1100)


def test_gradients_are_the_products_differences(device):
    """The product is linear in each table's values: <g, y(A, W) - y(A, W')> = <gw, W - W'>, and alike for the rows."""
    n, N, F = 300, 40, 100
    rng = np.random.default_rng(2)
    cw, sw, w = table_of(rng.standard_normal((N, F)).astype(np.float32), device)
    cv, sv, v = table_of(rng.standard_normal((N, F)).astype(np.float32), device)
    cb, sb, b = table_of(rng.standard_normal((n, F)).astype(np.float32), device)
    ca, sa, a = table_of(rng.standard_normal((n, F)).astype(np.float32), device)
    g = rng.standard_normal((n, N)).astype(np.float32)
    op = lowbit.MxProductOp()
    y = op.forward(a, w).cpu().numpy().astype(np.float64)
    gx = op.backward(dev(g, device)).cpu().numpy().astype(np.float64)
    gw = op.get_additional_grad().cpu().numpy().astype(np.float64)
    other_w = lowbit.MxProductOp().forward(a, v).cpu().numpy().astype(np.float64)
    other_a = lowbit.MxProductOp().forward(b, w).cpu().numpy().astype(np.float64)
    va, vw, vv, vb = (ref.mx_values(c, s, F) for c, s in ((ca, sa), (cw, sw), (cv, sv), (cb, sb)))
    # both sides sum n * N * F exact products; each output is off by R * 2^-23 of its terms
    size = (np.abs(g) @ (np.abs(vw) + np.abs(vv)) * np.abs(va)).sum()
    assert abs((g * (y - other_w)).sum() - (gw * (vw - vv)).sum()) <= 2 ** -23 * (4 * n + F + 1100) * size
    size = (np.abs(g) @ np.abs(vw) * (np.abs(va) + np.abs(vb))).sum()
    assert abs((g * (y - other_a)).sum() - (gx * (va - vb)).sum()) <= 2 ** -23 * (4 * N + F + 1100) * size


def test_gradient_of_extreme_values(device):
    """Infinities and NaN reach their own row or column, the largest floats do not overflow in the split, and rows of padding
    ids count for nothing in the weight's gradient."""
    n, N, F = 70, 40, 64
    rng = np.random.default_rng(3)
    cw, sw, w = table_of(np.abs(rng.standard_normal((N, F))).astype(np.float32) + 0.5, device)
    ca, sa, a = table_of(np.abs(rng.standard_normal((n, F))).astype(np.float32) + 0.5, device)
    g = rng.standard_normal((n, N)).astype(np.float32)
    g[3, 4], g[7, 8] = np.inf, np.nan
    g[9] = 0.0
    g[9, 5] = np.float32(3.4028235e38)
    ids = np.arange(n, dtype=np.uint32)
    ids[60] = 0xFFFFFFFF
    g[60] = 2.0
    op = lowbit.MxProductOp(dev(ids, device))
    op.forward(a, w)
    gx = op.backward(dev(g, device)).cpu().numpy()
    gw = op.get_additional_grad().cpu().numpy()
    wv = ref.mx_values(cw, sw, F)
    assert (gx[3] == np.inf).all() and np.isnan(gx[7]).all()
    with np.errstate(over="ignore"):
        largest = (g[9, 5].astype(np.float64) * wv[5]).astype(np.float32)
    assert (np.isinf(gx[9]) == np.isinf(largest)).all()
    fine = np.isfinite(largest)
    assert (gx[9][fine] == largest[fine]).all() and fine.any()
    rest = np.delete(np.arange(n), [3, 7])
    assert np.isfinite(gx[rest[rest != 9]]).all()
    assert (gw[4] == np.inf).all() and np.isnan(gw[8]).all() and np.isfinite(np.delete(gw, [4, 5, 8], 0)).all()
    keep = np.delete(np.arange(N), [4, 5, 8])
    full = ref.mx_rows(ca, sa, F, ids)
    want = g[:, keep].astype(np.float64).T @ full
    close(torch.from_numpy(gw[keep]), want, np.abs(g[:, keep]).astype(np.float64).T @ np.abs(full), 3 * n + 1100)


def test_a_low_nan_payload_stays_nan(device):
    _, _, w = table_of(np.ones((4, 32), dtype=np.float32), device)
    g = np.ones((3, 4), dtype=np.float32)
    g[1, 2] = np.array([0x7F800001], dtype=np.uint32).view(np.float32)[0]
    _, _, a = table_of(np.ones((3, 32), dtype=np.float32), device)
    op = lowbit.MxProductOp()
    op.forward(a, w)
    gx = op.backward(dev(g, device)).cpu().numpy()
    assert np.isnan(gx[1]).all() and (gx[[0, 2]] == 4.0).all()


def test_gradient_of_no_rows_is_zero(device):
    _, _, w = table_of(np.ones((5, 40), dtype=np.float32), device)
    _, _, a = table_of(np.ones((3, 40), dtype=np.float32), device)
    op = lowbit.MxProductOp(torch.zeros(0, dtype=torch.int32, device=device))
    assert op.forward(a, w).shape == (0, 5)
    assert op.backward(torch.zeros(0, 5, device=device)).shape == (0, 40)
    assert (op.get_additional_grad() == 0).all()
    op = lowbit.MxProductOp(torch.full((6,), -1, dtype=torch.int32, device=device), rows_grad=False)
    assert (op.forward(a, w) == 0).all()
    assert op.backward(torch.ones(6, 5, device=device)) is None and (op.get_additional_grad() == 0).all()


def test_repeated_calls_give_the_same_bits(device):
    _, _, a = table_of(rows_of(900, 100, 1, special=False), device)
    _, _, w = table_of(rows_of(70, 100, 2, special=False), device)
    g = torch.randn(40000, 70, device=device)
    ids = torch.randint(0, 900, (40000,), device=device, dtype=torch.int32)
    op = lowbit.MxProductOp(ids)
    first = None
    for _ in range(3):
        y = op.forward(a, w)
        got = [y, op.backward(g), op.get_additional_grad()]
        assert first is None or all(torch.equal(p, q) for p, q in zip(first, got))
        first = got


def test_a_table_beyond_32_bits(device):
    """Codes of more than 2^32 bytes and more than 2^32 output floats' worth of rows: offsets need 64 bits."""
    F, V = 2048, 4_300_000  # 1,024 bytes of codes a row: 4.4 GB
    (cs, ss) = lowbit.mx_shapes(V, F)
    codes, scales = torch.zeros(cs, dtype=torch.uint8, device=device), torch.full(ss, 127, dtype=torch.uint8, device=device)
    last = rows_of(5, F, 8, special=False)
    c, s = ref.mx_quantize(last)
    codes[-5:], scales[-5:] = dev(c, device), dev(s, device)
    t = lowbit.MxTable(codes, scales, F)
    ids = torch.arange(V - 6, V, dtype=torch.int32, device=device)
    want = np.concatenate([np.zeros((1, F)), ref.mx_values(c, s, F)])
    same(t.gather(ids).cpu().numpy(), want.astype(np.float32))
    cw, sw, w = table_of(rows_of(20, F, 9, special=False), device)
    wv = ref.mx_values(cw, sw, F)
    op = lowbit.MxProductOp(ids, rows_grad=False)
    close(op.forward(t, w), want @ wv.T, np.abs(want) @ np.abs(wv).T, F)
    many = lowbit.MxProductOp(ids.repeat(22))
    close(many.forward(t, w), np.tile(want @ wv.T, (22, 1)), np.tile(np.abs(want) @ np.abs(wv).T, (22, 1)), F)
    g = np.random.default_rng(1).standard_normal((6, 20)).astype(np.float32)
    op.backward(dev(g, device))
    close(op.get_additional_grad(), g.T.astype(np.float64) @ want, np.abs(g.T.astype(np.float64)) @ np.abs(want), 3 * 6 + 1100)


def test_captured_and_replayed(device):
    """Rounding, product and both gradients recorded into a graph; every replay equals the eager run on new inputs."""
    n, N, F = 3000, 64, 100
    x, w0 = torch.zeros(500, F, device=device), torch.zeros(N, F, device=device)
    g = torch.zeros(n, N, device=device)
    ids = torch.randint(0, 500, (n,), device=device, dtype=torch.int32)
    op = lowbit.MxProductOp(ids)

    def run():
        table = lowbit.MxTable.quantize(x)
        y = op.forward(table, lowbit.MxTable.quantize(w0))
        return y, op.backward(g), op.get_additional_grad(), table.gather(ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        recorded = run()
    for seed in range(3):
        torch.manual_seed(seed)
        for t in (x, w0, g):
            t.copy_(torch.randn(t.shape, device=device))
        eager = [t.clone() for t in run()]
        for t in recorded:
            t.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(recorded, eager)), f"replay {seed}"


@pytest.mark.parametrize("config,scale", [("arxiv", 0.1), ("gat", 0.02)])
def test_an_epoch_on_rows_in_4_bits(device, config, scale):
    """The epoch's own path with such a feature table: the same batches as with floats, and the same result with one batch and
    with several in flight."""
    plain = epoch.run(config, scale=scale, max_batches=4, warmup_batches=1, quiet=True)
    runs = [epoch.run(config, scale=scale, max_batches=4, warmup_batches=1, pipeline=p, quiet=True, checksum=True, features="mxfp4")
            for p in (1, 2, 4)]
    for r in runs:
        assert r["features"] == "mxfp4" and r["sampled_edges"] == plain["sampled_edges"] and r["gathered_rows"] == plain["gathered_rows"]
        assert r["checksum"] == runs[0]["checksum"] and np.isfinite(r["checksum"])
    assert plain["features"] == "f32"
    with pytest.raises(ValueError):
        epoch.run(config, features="int3")


@pytest.mark.parametrize("pipeline", [1, 2, 4])
def test_the_attention_epoch_reads_the_products_rows(device, monkeypatch, pipeline):
    """The first layer's input in the attention configuration: the batch's rows times the first layer's weight."""
    seen = []

    class Recorded(epoch.GATAggregateOp):
        def forward(self, x, alpha):
            seen.append((self.sg.dev_source.tensor().clone(), x.clone()))
            return super().forward(x, alpha)

    monkeypatch.setattr(epoch, "GATAggregateOp", Recorded)
    scale, cfg = 0.05, epoch.CONFIGS["gat"]
    V, F, hops = int(cfg["V"] * scale), cfg["F"], len(cfg["fanout"])
    out = epoch.run("gat", scale=scale, max_batches=3, warmup_batches=0, pipeline=pipeline, quiet=True, features="mxfp4")
    assert len(seen) == out["batches"] * hops == 3 * hops
    x = ref.mx_values(*ref.mx_quantize(synth.normal_features(V, F, seed=cfg["seed"] + 40).numpy()), F)
    weight = synth.normal_features(cfg["hidden"], F, seed=cfg["seed"] + 43, device=device).cpu().numpy() * np.float32(F ** -0.5)
    w = ref.mx_values(*ref.mx_quantize(weight), F)
    rows = 0
    for ids, got in seen[::hops]:  # input side first
        at = ids.cpu().numpy().view(np.uint32).astype(np.int64)
        close(got, x[at] @ w.T, np.abs(x[at]) @ np.abs(w).T, F)
        rows += at.size
    assert rows == out["gathered_rows"]


def test_a_sampled_layers_rows(device):
    """load_feature_mxfp4 and a product by the builder's own id array (a range of its arena)."""
    V, F = 500, 70
    codes, scales, t = table_of(rows_of(V, F, 2, special=False), device)
    rng = np.random.default_rng(3)
    deg = rng.integers(0, 12, V)
    co = np.concatenate([[0], np.cumsum(deg)]).astype(np.uint32)
    builder = BatchBuilder(dev(co, device), dev(rng.integers(0, V, int(co[-1])).astype(np.uint32), device), [5], 64)
    layer = builder.sample(dev(np.arange(64, dtype=np.uint32), device), 1)[0]
    ids = layer.dev_source.cpu().numpy().view(np.uint32)
    want = ref.mx_rows(codes, scales, F, ids)
    x = torch.empty(layer.src_size, F, device=device)
    load_feature_mxfp4(CudaStream(), layer, x, t)
    same(x.cpu().numpy(), want.astype(np.float32))
    same(t.gather(layer.dev_source).cpu().numpy(), want.astype(np.float32))
    cw, sw, w = table_of(rows_of(30, F, 4, special=False), device)
    wv = ref.mx_values(cw, sw, F)
    close(lowbit.MxProductOp(layer.dev_source).forward(t, w), want @ wv.T, np.abs(want) @ np.abs(wv).T, F)
    builder.close()
