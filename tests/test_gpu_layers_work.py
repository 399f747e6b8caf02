"""Layers in training: no write behind the work that a call asks for."""
import pytest
import torch

from neutronbench_amd import layers
from test_gpu_layers import BF16, F16, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,act", [(BF16, "gelu"), (F16, "silu")])
@pytest.mark.parametrize("n,F,N,weight", [(7424, 2176, 2176, True), (4352, 520, 3900, False), (4352, 3900, 520, True), (9000, 1024, 2048, False)])
@pytest.mark.parametrize("shift", [0, 1])
def test_dense_gradients_stay_in_their_work(device, dtype, act, n, F, N, weight, shift):
    """Products large enough for large tiles, whose operands begin at aligned addresses or between them; the weight's gradient of one part, of several
    or not wanted, so that nothing else lies behind the bias's sums."""
    x, _ = rows(n, F, 1, dtype, device, shift=shift)
    w, _ = rows(N, F, 2, dtype, device, F ** -0.5, shift)
    b, _ = rows(1, N, 3, dtype, device)
    g, _ = rows(n, N, 4, dtype, device)
    kind, code, guard = layers.TYPES[dtype], layers.ACTIVATIONS[act], 1 << 20
    size = layers.call("nts_dense_grad_work_bytes", kind, n, N, F, code, 0, 0, 0, int(weight), 1)
    work = torch.full((size + guard,), 0xA5, dtype=torch.uint8, device=device)
    gw, gb = torch.empty(N, F, dtype=dtype, device=device) if weight else None, torch.empty(N, dtype=dtype, device=device)
    layers.call("nts_dense_grad", 0, layers.ptr(gw), gb.data_ptr(), g.data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), 0, kind, n, N, F, code, 0,
                work.data_ptr(), layers._stream(x.device))
    assert (work[size:] == 0xA5).all()
    # the same sums by way of operands that the rest of the tests cover, a few rows at a time
    parts = []
    for i in range(0, n, 1000):
        op = layers.DenseOp(act, rows_grad=False)
        op.forward(x[i:i + 1000].float().contiguous(), w.float(), b[0].float())
        op.backward(g[i:i + 1000].float().contiguous())
        parts.append(op.get_additional_grad()[1].double())
    want = torch.stack(parts).sum(0)
    # Both are 32-bit sums of n terms g slope(z), of which a slope is at most 1.13, rounded once; z is off by F + 4 half steps of its terms'
    # magnitudes on either side, and a slope changes by at most 0.8 of that.
    size = float((x.float().abs() @ w.float().abs().t()).max())
    off = (gb.double() - want).abs()
    bound = 2 ** -24 * (2 * 1.13 * (n + 20) + 2 * 0.8 * (F + 4) * size) * g.double().abs().sum(0)
    assert (off <= want.abs() * torch.finfo(dtype).eps / 2 + bound).all()
