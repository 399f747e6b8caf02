"""Layers of vertices in training: what lies between the graph operators of a model, and attention with dot products as scores
(nts_dropout, nts_dense* and nts_dot_attention* of include/nts_hip.h, which say what is computed and how it is rounded).

  Dropout          which values are dropped: a rate, a seed and a step
  DropoutOp        rows with some of their values zeroed and the others scaled up; no mask is stored
  DenseOp          rows times a weight with bias, activation, dropout and residual, and its gradients
  DotAttentionOp   every destination's attention over its edges' sources, and the gradients of queries, keys and values

Operands are 2-D contiguous tensors of float32, bfloat16 or float16, one type in a call.  Work is enqueued on torch's current stream of the
operands' device.
"""
import ctypes
import math

import torch

from .abi import DropoutDesc, allocate, call, ptr
from .lowbit import _indices, _on, _same_device, _stream

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _type(t, what):
    if t.dtype not in TYPES:
        raise ValueError(f"{what}: float32, bfloat16 or float16")
    return TYPES[t.dtype]


def _rows(t, rows, columns, like, what):
    """Checks a 2-D operand (rows, columns None: any number) of the type of `like`."""
    if t.dim() != 2 or not t.is_contiguous() or t.dtype != like.dtype or (rows is not None and t.shape[0] != rows) or (
            columns is not None and t.shape[1] != columns):
        shape = f"[{'n' if rows is None else rows}, {'columns' if columns is None else columns}]"
        raise ValueError(f"{what}: a contiguous {like.dtype} tensor {shape}")
    if max(t.shape) >= 1 << 32:
        raise ValueError(f"{what}: fewer than 2^32 rows and columns")


class Dropout:
    """Values are dropped with probability p (in steps of 1 / 65,536).  Which ones follows from seed, step and their place alone: an
    operator draws the same in its backward pass.  Operators of one training step take different seeds; every training step takes
    another `step`: a number, or an int32 tensor of one element (a uint32 bit pattern) on the operands' device, which the kernels read
    when they run, so that replays of a captured graph draw other numbers once it has changed.  A backward pass uses the step that its
    forward pass found."""
    __slots__ = ("p", "seed", "step")

    def __init__(self, p, seed, step=0):
        if not 0.0 <= p <= 1.0:
            raise ValueError("p: 0 .. 1")
        if not 0 <= seed < 2**64:
            raise ValueError("seed: 0 .. 2^64 - 1")
        self.p, self.seed, self.step = p, seed, step
        self._check()

    def _check(self):
        if isinstance(self.step, torch.Tensor):
            if self.step.dtype != torch.int32 or self.step.numel() != 1:
                raise ValueError("step: an int32 tensor of one element")
        elif not 0 <= self.step < 2**32:
            raise ValueError("step: 0 .. 2^32 - 1")


class _Drawn:
    """What a forward pass drew: its dropout with the step it used."""
    __slots__ = ("desc", "step", "kept")

    def __init__(self, dropout, device):
        dropout._check()
        self.step = self.kept = None
        if isinstance(dropout.step, torch.Tensor):
            _same_device(device, dropout.step)
            self.step = dropout.step
            self.kept = allocate(torch.empty, 1, dtype=torch.int32, device=device)
            self.desc = DropoutDesc(dropout.p, 0, dropout.seed, ptr(self.step), ptr(self.kept))
        else:
            self.desc = DropoutDesc(dropout.p, dropout.step, dropout.seed, 0, 0)

    def again(self):
        """For the backward pass."""
        if self.kept is not None:
            return DropoutDesc(self.desc.p, 0, self.desc.seed, ptr(self.kept), 0)
        return self.desc


def _drawn(dropout, device):
    return None if dropout is None else _Drawn(dropout, device)


def _ref(desc):
    return 0 if desc is None else ctypes.addressof(desc)


def _work(size, device):
    return allocate(torch.empty, size, dtype=torch.uint8, device=device) if size else None


class DropoutOp:
    """y = x where it is kept, times 1 / (1 - p), 0 elsewhere; backward returns the gradient of x."""

    def __init__(self, dropout):
        if not isinstance(dropout, Dropout):
            raise ValueError("dropout: a Dropout")
        self.dropout = dropout
        self.drawn = self.shape = None

    def _run(self, x, desc):
        out = allocate(torch.empty_like, x)
        with _on(x.device):
            call("nts_dropout", ptr(out), ptr(x), _type(x, "x"), x.shape[0], x.shape[1], _ref(desc), _stream(x.device))
        return out

    def forward(self, x):
        _rows(x, None, None, x, "x")
        _type(x, "x")
        drawn = _Drawn(self.dropout, x.device)
        out = self._run(x, drawn.desc)
        self.drawn, self.shape, self.device = drawn, x.shape, x.device
        return out

    def backward(self, g_out):
        if self.drawn is None:
            raise ValueError("backward before forward")
        _rows(g_out, *self.shape, g_out, "g_out")
        _same_device(self.device, g_out)
        return self._run(g_out, self.drawn.again())


class DenseOp:
    """y = residual + drop(act(x W^T + bias)), W with a row per output; activation: none, relu, gelu or silu.  backward returns the
    gradient of x (None with rows_grad=False: feature rows are constants), get_additional_grad() those of W and bias (None without
    one); the residual's is the gradient of y itself.  The backward pass computes the sums again, or with relu and no residual reads from y
    which were above 0: x, W, bias and y have to be what they were."""

    def __init__(self, activation="none", dropout=None, rows_grad=True):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation: one of {', '.join(ACTIVATIONS)}")
        if dropout is not None and not isinstance(dropout, Dropout):
            raise ValueError("dropout: a Dropout or None")
        self.activation, self.dropout, self.rows_grad = activation, dropout, rows_grad
        self.x = self.weight = self.bias = self.y = self.drawn = self.gw = self.gb = None

    def forward(self, x, weight, bias=None, residual=None):
        kind = _type(x, "x")
        _rows(x, None, None, x, "x")
        (n, F), dev = x.shape, x.device
        _rows(weight, None, F, x, "weight")
        N = weight.shape[0]
        if bias is not None and (bias.dim() != 1 or bias.shape[0] != N or bias.dtype != x.dtype or not bias.is_contiguous()):
            raise ValueError(f"bias: a contiguous {x.dtype} tensor [{N}]")
        if residual is not None:
            _rows(residual, n, N, x, "residual")
        _same_device(dev, weight, bias, residual)
        drawn = _drawn(self.dropout, dev)
        y = allocate(torch.empty, n, N, dtype=x.dtype, device=dev)
        with _on(dev):
            work = _work(call("nts_dense_work_bytes", kind, n, N, F), dev)
            call("nts_dense", ptr(y), ptr(x), ptr(weight), ptr(bias), ptr(residual), kind, n, N, F, ACTIVATIONS[self.activation],
                 _ref(drawn and drawn.desc), ptr(work), _stream(dev))
        self.x, self.weight, self.bias, self.drawn = x, weight, bias, drawn
        self.y = y if self.activation == "relu" and residual is None else None
        return y

    def backward(self, g_out):
        x, weight, bias = self.x, self.weight, self.bias
        if x is None:
            raise ValueError("backward before forward")
        (n, F), N, dev, kind, act = x.shape, weight.shape[0], x.device, TYPES[x.dtype], ACTIVATIONS[self.activation]
        _rows(g_out, n, N, x, "g_out")
        _same_device(dev, g_out)
        gx = allocate(torch.empty_like, x) if self.rows_grad else None
        self.gw = allocate(torch.empty_like, weight)
        self.gb = None if bias is None else allocate(torch.empty_like, bias)
        drawn = self.drawn and self.drawn.again()
        with _on(dev):
            work = _work(call("nts_dense_grad_work_bytes", kind, n, N, F, act, drawn is not None, self.y is not None, gx is not None, 1,
                              bias is not None), dev)
            call("nts_dense_grad", ptr(gx), ptr(self.gw), ptr(self.gb), ptr(g_out), ptr(x), ptr(weight), ptr(bias), ptr(self.y), kind, n, N, F,
                 act, _ref(drawn), ptr(work), _stream(dev))
        return gx

    def get_additional_grad(self):
        return self.gw, self.gb


class DotAttentionOp:
    """out[d, h, :] = sum over d's edges of drop(softmax(scale * <q[d, h], k[src, h']>)) v[src, h']; the log of each softmax's denominator is
    in `lse` afterwards.  layer: a SampledLayer, or a FullGraphChunk; q has a row for each of its destinations, k and v for each of its
    sources, of q_heads and heads times the width.  backward returns the gradient of q, get_additional_grad() those of k
    and v; the probabilities are computed again, so q, k, v and lse have to be what they were.  Edges whose source the layer does not
    have are left out."""

    def __init__(self, layer, q_heads, heads=None, scale=None, dropout=None):
        heads = q_heads if heads is None else heads
        if q_heads < 1 or heads < 1 or q_heads % heads:
            raise ValueError("q_heads: a multiple of heads")
        if dropout is not None and not isinstance(dropout, Dropout):
            raise ValueError("dropout: a Dropout or None")
        self.sg, self.q_heads, self.heads, self.scale, self.dropout = layer, q_heads, heads, scale, dropout
        self.q = self.k = self.v = self.lse = self.drawn = self.gk = self.gv = None

    def _edges(self, offsets, ids, rows, exact, dev, what):
        _indices(offsets, f"{what} offsets")
        _indices(ids, f"{what} indices")
        if offsets.numel() != rows + 1 or (exact and ids.numel() < self.sg.e_size):
            raise ValueError(f"layer: {what} offsets of {rows} rows and {self.sg.e_size} edges")
        _same_device(dev, offsets, ids)

    def forward(self, q, k, v):
        sg, H, Hk = self.sg, self.q_heads, self.heads
        kind, dev = _type(q, "q"), q.device
        if q.dim() != 2 or q.shape[1] == 0 or q.shape[1] % H:
            raise ValueError(f"q: {H} heads of one width")
        D = q.shape[1] // H
        _rows(q, sg.v_size, H * D, q, "q")
        _rows(k, sg.src_size, Hk * D, q, "k")
        _rows(v, sg.src_size, Hk * D, q, "v")
        co, ri = sg.dev_c_o(), sg.dev_r_i()
        self._edges(co, ri, sg.v_size, True, dev, "column")
        _same_device(dev, k, v)
        bound = getattr(sg, "max_in_degree", 0)
        scale = 1.0 / math.sqrt(D) if self.scale is None else self.scale
        drawn = _drawn(self.dropout, dev)
        out = allocate(torch.empty_like, q)
        lse = allocate(torch.empty, sg.v_size, H, dtype=torch.float32, device=dev)
        with _on(dev):
            work = _work(call("nts_dot_attention_work_bytes", sg.v_size, sg.e_size, H, D, bound), dev)
            call("nts_dot_attention", ptr(out), ptr(lse), ptr(q), ptr(k), ptr(v), kind, ptr(co), ptr(ri), sg.v_size, sg.src_size, sg.e_size,
                 H, Hk, D, scale, bound, _ref(drawn and drawn.desc), ptr(work), _stream(dev))
        self.q, self.k, self.v, self.lse, self.drawn, self.used_scale = q, k, v, lse, drawn, scale
        return out

    def backward(self, g_out):
        q, k, v, sg, H, Hk = self.q, self.k, self.v, self.sg, self.q_heads, self.heads
        if q is None:
            raise ValueError("backward before forward")
        dev, D, bound = q.device, q.shape[1] // H, getattr(sg, "max_in_degree", 0)
        _rows(g_out, *q.shape, q, "g_out")
        co, ri, ro, ci = sg.dev_c_o(), sg.dev_r_i(), sg.dev_r_o(), sg.dev_c_i()
        if ro is None or ci is None:
            raise ValueError("layer: the edges by source (row offsets, column indices) are needed")
        self._edges(co, ri, sg.v_size, True, dev, "column")
        self._edges(ro, ci, sg.src_size, False, dev, "row")
        _same_device(dev, g_out)
        gq, self.gk, self.gv = allocate(torch.empty_like, q), allocate(torch.empty_like, k), allocate(torch.empty_like, v)
        drawn = self.drawn and self.drawn.again()
        with _on(dev):
            work = _work(call("nts_dot_attention_grad_work_bytes", sg.v_size, sg.src_size, sg.e_size, H, Hk, D, bound), dev)
            call("nts_dot_attention_grad", ptr(gq), ptr(self.gk), ptr(self.gv), ptr(g_out), ptr(q), ptr(k), ptr(v), ptr(self.lse),
                 TYPES[q.dtype], ptr(co), ptr(ri), ptr(ro), ptr(ci), sg.v_size, sg.src_size, sg.e_size, H, Hk, D, self.used_scale, bound,
                 _ref(drawn), ptr(work), _stream(dev))
        return gq

    def get_additional_grad(self):
        return self.gk, self.gv
