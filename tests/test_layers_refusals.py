"""Arguments that the operators of layers in training refuse, before any device work (no GPU)."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

from neutronbench_amd import abi, epoch, layers
from neutronbench_amd.layout import SampledLayer

P = 4096  # stands for a device pointer with any alignment that is asked for: refused calls never follow it
BIG = (1 << 17) + 1


def drop(p=0.5):
    return abi.DropoutDesc(p, 0, 1, 0, 0)


def refused(text, name, *args):
    assert abi.status(name, *args) == abi.NTS_ERR_INVALID
    assert text in abi.last_error() and name in abi.last_error()


def ref(desc):
    return ctypes.addressof(desc)


def test_dropout():
    d = drop()
    refused("unknown type", "nts_dropout", P, P, 3, 4, 8, ref(d), 0)
    refused("unknown type", "nts_dropout", P, P, -1, 4, 8, ref(d), 0)
    for F in (0, BIG):
        refused("F is 0", "nts_dropout", P, P, 0, 4, F, ref(d), 0)
    for args in ((0, P), (P, 0)):
        refused("null pointer", "nts_dropout", *args, 0, 4, 8, ref(d), 0)
    refused("null pointer", "nts_dropout", P, P, 0, 4, 8, 0, 0)
    for p in (-0.1, 1.1, math.nan, math.inf):
        bad = drop(p)
        refused("within 0 .. 1", "nts_dropout", P, P, 0, 4, 8, ref(bad), 0)
    refused("alignment", "nts_dropout", P + 2, P, 0, 4, 8, ref(d), 0)
    refused("alignment", "nts_dropout", P, P + 1, 1, 4, 8, ref(d), 0)
    assert abi.status("nts_dropout", 0, 0, 0, 0, 8, ref(d), 0) == abi.NTS_OK


def test_dense():
    name = "nts_dense"
    good = [P, P, P, 0, 0, 0, 40, 8, 8, 0, 0, P, 0]
    for N, F in ((0, 8), (8, 0), (BIG, 8), (8, BIG)):
        refused("N or F", name, *good[:7], N, F, *good[9:])
    refused("unknown type", name, *good[:5], 7, *good[6:])
    for act in (-1, 4):
        refused("unknown activation", name, *good[:9], act, *good[10:])
    for hole in range(3):
        args = list(good)
        args[hole] = 0
        refused("null pointer", name, *args)
    for at in range(5):
        args = list(good)
        args[at] = P + 2
        refused("alignment", name, *args)
    for work in (0, P + 8):
        refused("work_bytes", name, *good[:11], work, 0)
    bad = drop(2.0)
    refused("within 0 .. 1", name, *good[:10], ref(bad), P, 0)
    assert abi.status(name, 0, 0, 0, 0, 0, 0, 0, 8, 8, 0, 0, 0, 0) == abi.NTS_OK
    assert abi.call("nts_dense_work_bytes", 0, 1, 8, 8) == 0


def test_dense_gradients():
    name = "nts_dense_grad"
    good = [P, P, P, P, P, P, P, 0, 0, 40, 8, 8, 2, 0, P, 0]
    for N, F in ((0, 8), (8, 0), (BIG, 8), (8, BIG)):
        refused("N or F", name, *good[:10], N, F, *good[12:])
    refused("unknown activation", name, *good[:12], 9, *good[13:])
    for hole in (3, 4, 5):
        args = list(good)
        args[hole] = 0
        refused("null pointer", name, *args)
    for work in (0, P + 8):
        refused("work_bytes", name, *good[:14], work, 0)
    for at in range(8):
        args = list(good)
        args[at] = P + 1
        refused("alignment", name, *args)
    assert abi.status(name, 0, 0, 0, P, P, P, 0, 0, 0, 4, 8, 8, 1, 0, 0, 0) == abi.NTS_OK  # nothing wanted
    # y says what relu's gradient needs: neither z nor the gradient of z is stored
    with_y, without = (abi.call("nts_dense_grad_work_bytes", 0, 1000, 128, 64, 1, 1, y, 1, 1, 1) for y in (1, 0))
    assert without - with_y >= 1000 * 128 * 4


def test_attention():
    name = "nts_dot_attention"
    good = [P, P, P, P, P, 0, P, P, 100, 5, 6, 4, 2, 16, 1.0, 0, 0, P, 0]
    for q_heads, heads in ((0, 1), (4, 0), (4, 3), (2048, 2), (2, 4)):
        refused("q_heads", name, *good[:11], q_heads, heads, *good[13:])
    for width in (0, 257):
        refused("width", name, *good[:13], width, *good[14:])
    refused("unknown type", name, *good[:5], 5, *good[6:])
    refused("2^32 - 2^16", name, *good[:10], 0xFFFF0001, *good[11:])
    for hole in (0, 1, 2, 3, 4, 6, 7):
        args = list(good)
        args[hole] = 0
        refused("null pointer", name, *args)
    for at in (0, 2, 3, 4):
        args = list(good)
        args[at] = P + 2
        refused("alignment", name, *args)
    for work in (0, P + 4):
        refused("work_bytes", name, *good[:17], work, 0)
    bad = drop(-1.0)
    refused("within 0 .. 1", name, *good[:16], ref(bad), P, 0)
    assert abi.status(name, *[0] * 5, 0, 0, 0, 0, 5, 6, 4, 2, 16, 1.0, 0, 0, 0, 0) == abi.NTS_OK


def test_attention_gradients():
    name = "nts_dot_attention_grad"
    good = [P] * 8 + [0, P, P, P, P, 4, 5, 6, 4, 2, 16, 1.0, 0, 0, P, 0]
    for q_heads, heads in ((0, 1), (4, 0), (4, 3), (2048, 2)):
        refused("q_heads", name, *good[:16], q_heads, heads, *good[18:])
    for hole in [*range(8), 9, 10, 11, 12]:
        args = list(good)
        args[hole] = 0
        refused("null pointer", name, *args)
    for at in range(7):
        args = list(good)
        args[at] = P + 2
        refused("alignment", name, *args)
    for work in (0, P + 4):
        refused("work_bytes", name, *good[:22], work, 0)
    assert abi.status(name, *[0] * 8, 0, 0, 0, 0, 0, 0, 0, 6, 4, 2, 16, 1.0, 0, 0, 0, 0) == abi.NTS_OK
    assert abi.call("nts_dot_attention_grad_work_bytes", 4, 5, 6, 0, 1, 16, 0) == 0


def test_dropout_objects():
    for p in (-0.1, 1.5, math.nan):
        with pytest.raises(ValueError, match="p:"):
            layers.Dropout(p, 1)
    for seed in (-1, 2**64):
        with pytest.raises(ValueError, match="seed"):
            layers.Dropout(0.5, seed)
    for step in (-1, 2**32, torch.zeros(1), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="step"):
            layers.Dropout(0.5, 1, step)
    with pytest.raises(ValueError, match="dropout"):
        layers.DropoutOp(0.5)
    with pytest.raises(ValueError, match="dropout"):
        layers.DenseOp("relu", 0.5)
    op = layers.DropoutOp(layers.Dropout(0.5, 1))
    with pytest.raises(ValueError, match="before forward"):
        op.backward(torch.zeros(2, 2))
    for x in (torch.zeros(4), torch.zeros(4, 4).t()[:2], torch.zeros(2, 2, dtype=torch.float64), torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="x:"):
            op.forward(x)


def test_dense_objects():
    with pytest.raises(ValueError, match="activation"):
        layers.DenseOp("tanh")
    op = layers.DenseOp()
    with pytest.raises(ValueError, match="before forward"):
        op.backward(torch.zeros(2, 2))
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for args, what in (((x.double(), w), "x:"), ((x, torch.zeros(6, 7)), "weight"), ((x, w.bfloat16()), "weight"), ((x, w.t()), "weight"),
                       ((x, w, torch.zeros(5)), "bias"), ((x, w, torch.zeros(6).half()), "bias"), ((x, w, torch.zeros(12)[::2]), "bias"),
                       ((x, w, None, torch.zeros(4, 5)), "residual"), ((x, w, None, torch.zeros(3, 6)), "residual")):
        with pytest.raises(ValueError, match=what):
            op.forward(*args)


def test_attention_objects():
    sg = SampledLayer()
    for heads in ((0, 1), (4, 3), (4, 0)):
        with pytest.raises(ValueError, match="q_heads"):
            layers.DotAttentionOp(sg, *heads)
    sg.v_size, sg.e_size, sg.src_size = 3, 4, 5
    sg.dev_column_offset, sg.dev_row_indices = torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    op = layers.DotAttentionOp(sg, 4, 2)
    with pytest.raises(ValueError, match="before forward"):
        op.backward(torch.zeros(2, 2))
    q, k = torch.zeros(3, 64), torch.zeros(5, 32)
    for args, what in (((q[:2], k, k), "q:"), ((torch.zeros(3, 63), k, k), "q:"), ((q, k[:4], k), "k:"), ((q, k, torch.zeros(5, 64)), "v:"),
                       ((q, k.half(), k), "k:"), ((q.double(), k, k), "q:"), ((torch.zeros(3, 0), k, k), "q:")):
        with pytest.raises(ValueError, match=what):
            op.forward(*args)
    sg.dev_column_offset = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="offsets"):
        op.forward(q, k, k)
    sg.dev_column_offset, sg.dev_row_indices = torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="offsets"):
        op.forward(q, k, k)


@pytest.mark.parametrize("options,text", [
    (["--config", "arxiv", "--attention", "dot"], "heads"), (["--config", "gat", "--attention", "dot", "--native"], "--attention gat"),
    (["--config", "gat", "--attention", "dot", "--write-inputs", "inputs"], "--attention gat"),
    (["--config", "gat", "--dropout", "0.5"], "--dropout"), (["--config", "gat", "--attention", "dot", "--dropout", "1.5"], "--dropout"),
    (["--config", "gat", "--attention", "dot", "--dropout", "nan"], "--dropout"), (["--config", "gat", "--attention", "add"], "--attention")])
def test_options_of_the_epoch(options, text, tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(epoch.__file__)))
    got = subprocess.run([sys.executable, "-m", "neutronbench_amd.epoch", *options], cwd=tmp_path, env={**os.environ, "PYTHONPATH": root},
                         capture_output=True, text=True)
    assert got.returncode == 2 and text in got.stderr and not os.listdir(tmp_path)


def test_arguments_of_the_epoch():
    for args in (dict(name="gat", attention="add"), dict(name="arxiv", attention="dot"), dict(name="gat", dropout=0.5),
                 dict(name="gat", attention="dot", dropout=-0.1), dict(name="gat", attention="dot", dropout=math.nan)):
        with pytest.raises(ValueError, match="attention|dropout"):
            epoch.run(**args)
