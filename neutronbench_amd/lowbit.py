"""Vertex tables in few bits: feature rows and weights in 4 bits, a cache of keys and values in 8, and the operators that
read them by vertex id (nts_mxfp4_*, nts_gather_rows_mxfp4 and nts_kv8_* of include/nts_hip.h, which say how they are laid
out and rounded).

  MxTable              rows of 4-bit values with a power-of-two scale for every 32
  MxProductOp          rows gathered from one such table times a weight held in another, with both gradients
  Kv8Cache             keys and values of vertices, a scale for a block of vertices and a head
  NeighborAttentionOp  every destination's attention over its neighbours' rows of such a cache

Work is enqueued on torch's current stream of the operands' device.
"""
import contextlib
import math

import torch

from .abi import allocate, call, ptr

MX_BLOCK = 32


def mx_shapes(rows, width):
    """Shapes of the code and scale arrays of a 4-bit table."""
    blocks = -(-width // MX_BLOCK)
    return (rows, 16 * blocks), (rows, -(-blocks // 4) * 4)


def kv8_row_width(width):
    return -(-width // 16) * 16


# The raw handle of torch's current stream; a Stream object for it takes 2 us more to make, a fifth of a small call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    return _raw_stream(device.index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream


_HERE = contextlib.nullcontext()


def _on(device):
    """The device made current for a call, if it is not."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _floats(t, columns, what):
    if t.dim() != 2 or t.dtype != torch.float32 or not t.is_contiguous() or (columns is not None and t.shape[1] != columns):
        raise ValueError(f"{what}: a 2-D contiguous fp32 tensor" + (f" of {columns} columns" if columns is not None else ""))


def _bytes(t, shape, what):
    if t.dtype != torch.uint8 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous uint8 tensor of shape {tuple(shape)}")


def _indices(t, what):
    """int32 device tensors (uint32 bit patterns), or ranges of an arena (batch.DevArray)."""
    if t.dtype != torch.int32 or (isinstance(t, torch.Tensor) and not t.is_contiguous()):
        raise ValueError(f"{what}: contiguous int32 (uint32 bit patterns)")


def _same_device(device, *tensors):
    if any(t is not None and t.device != device for t in tensors):
        raise ValueError(f"operands on another device than {device}")


class MxTable:
    """Rows of `width` values in 4 bits: `codes` and `scales` are uint8 tensors of mx_shapes(rows, width)."""
    __slots__ = ("codes", "scales", "rows", "width", "device")

    def __init__(self, codes, scales, width):
        code_shape, scale_shape = mx_shapes(codes.shape[0], width)
        _bytes(codes, code_shape, "codes")
        _bytes(scales, scale_shape, "scales")
        _same_device(codes.device, scales)
        self._hold(codes, scales, codes.shape[0], width, codes.device)

    def _hold(self, codes, scales, rows, width, device):
        self.codes, self.scales, self.rows, self.width, self.device = codes, scales, rows, width, device

    @classmethod
    def quantize(cls, x):
        """The rows of x [n, width] rounded to the nearest values their blocks can hold."""
        _floats(x, None, "x")
        (n, width), dev = x.shape, x.device
        code_shape, scale_shape = mx_shapes(n, width)
        codes = allocate(torch.empty, code_shape, dtype=torch.uint8, device=dev)
        scales = allocate(torch.empty, scale_shape, dtype=torch.uint8, device=dev)
        with _on(dev):
            call("nts_mxfp4_quantize", ptr(codes), ptr(scales), ptr(x), n, width, _stream(dev))
        self = cls.__new__(cls)  # its own arrays need no checks
        self._hold(codes, scales, n, width, dev)
        return self

    def gather(self, row_ids=None, out=None):
        """The rows as floats: all of them, or those that row_ids names (an id beyond the table: zeros)."""
        n = self.rows if row_ids is None else row_ids.numel()
        if row_ids is not None:
            _indices(row_ids, "row_ids")
        if out is None:
            out = allocate(torch.empty, n, self.width, dtype=torch.float32, device=self.device)
        else:
            _floats(out, self.width, "out")
            if out.shape[0] != n:
                raise ValueError(f"out: {n} rows")
        _same_device(self.device, row_ids, out)
        with _on(self.device):
            call("nts_gather_rows_mxfp4", ptr(out), ptr(self.codes), ptr(self.scales), self.rows, ptr(row_ids), n, self.width,
                 _stream(self.device))
        return out


class MxProductOp:
    """y[i, :] = A[row_ids[i], :] W^T for 4-bit tables A (vertex rows) and W (a row per output); two-input operator: backward
    returns the gradient of the gathered rows' values (None with rows_grad=False: feature rows are constants),
    get_additional_grad() the gradient of W's values."""

    def __init__(self, row_ids=None, rows_grad=True):
        if row_ids is not None:
            _indices(row_ids, "row_ids")
        self.row_ids, self.rows_grad = row_ids, rows_grad
        self.table = self.weight = self.gw = None

    def _rows(self, table):
        return table.rows if self.row_ids is None else self.row_ids.numel()

    def forward(self, table, weight):
        if table.width != weight.width:
            raise ValueError(f"rows of {table.width} values and a weight of {weight.width}")
        dev = table.device
        _same_device(dev, weight.codes, self.row_ids)
        n = self._rows(table)
        y = allocate(torch.empty, n, weight.rows, dtype=torch.float32, device=dev)
        with _on(dev):
            call("nts_mxfp4_product", ptr(y), ptr(table.codes), ptr(table.scales), table.rows, ptr(self.row_ids), n,
                 ptr(weight.codes), ptr(weight.scales), weight.rows, table.width, 0, _stream(dev))
        self.table, self.weight = table, weight
        return y

    def backward(self, g_out):
        table, weight = self.table, self.weight
        if table is None:
            raise ValueError("backward before forward")
        n, N, F, dev = self._rows(table), weight.rows, table.width, table.device
        _floats(g_out, N, "g_out")
        if g_out.shape[0] != n:
            raise ValueError(f"g_out: {n} rows")
        _same_device(dev, g_out)
        stream = _stream(dev)
        gx = None
        with _on(dev):
            if self.rows_grad:
                gx = allocate(torch.empty, n, F, dtype=torch.float32, device=dev)
                call("nts_mxfp4_product_grad_rows", ptr(gx), ptr(g_out), ptr(weight.codes), ptr(weight.scales), n, N, F, 0, stream)
            self.gw = allocate(torch.empty, N, F, dtype=torch.float32, device=dev)
            size = call("nts_mxfp4_product_grad_weight_work_bytes", n, N, F)
            work = allocate(torch.empty, size, dtype=torch.uint8, device=dev) if size else None
            call("nts_mxfp4_product_grad_weight", ptr(self.gw), ptr(g_out), ptr(table.codes), ptr(table.scales), table.rows,
                 ptr(self.row_ids), n, N, F, 0, ptr(work), stream)
        return gx

    def get_additional_grad(self):
        return self.gw


class Kv8Cache:
    """Keys and values of up to `capacity` vertices in 8 bits, with a scale for every block of `block_rows` vertices and
    head, for keys and values each.  `rows` is how many the cache holds."""

    def __init__(self, capacity, heads, width, block_rows=16, device="cuda"):
        self._check(heads, width, block_rows)
        cache = allocate(torch.zeros, (capacity, 2, heads, kv8_row_width(width)), dtype=torch.uint8, device=device)
        scales = allocate(torch.zeros, (-(-capacity // block_rows), 2, heads), dtype=torch.uint8, device=device)
        self._hold(cache, scales, width, block_rows, 0)

    @classmethod
    def over(cls, cache, scales, width, block_rows, rows=None):
        """A cache in the caller's arrays, whose first `rows` rows are filled (all by default)."""
        self = cls.__new__(cls)
        self._hold(cache, scales, width, block_rows, cache.shape[0] if rows is None else rows)
        return self

    @staticmethod
    def _check(heads, width, block_rows):
        if not 1 <= heads <= 1024 or not 1 <= width <= 256 or not 1 <= block_rows <= 1024 or block_rows & (block_rows - 1):
            raise ValueError("cache: 1 .. 1,024 heads, width 1 .. 256, block_rows a power of two up to 1,024")

    def _hold(self, cache, scales, width, block_rows, rows):
        if cache.dim() != 4:
            raise ValueError("cache: [capacity, 2, heads, row width]")
        capacity, _, heads, _ = cache.shape
        self._check(heads, width, block_rows)
        _bytes(cache, (capacity, 2, heads, kv8_row_width(width)), "cache")
        _bytes(scales, (-(-capacity // block_rows), 2, heads), "scales")
        _same_device(cache.device, scales)
        if not 0 <= rows <= capacity:
            raise ValueError(f"rows: 0 .. {capacity}")
        self.cache, self.scales, self.width, self.block_rows, self.rows = cache, scales, width, block_rows, rows
        self.capacity, self.heads, self.device = capacity, heads, cache.device

    def append(self, k, v, first=None):
        """Writes the rows of k and v [n, heads * width] at `first` (default: behind the last row), where the cache then ends."""
        first = self.rows if first is None else first
        _floats(k, self.heads * self.width, "k")
        _floats(v, self.heads * self.width, "v")
        n = k.shape[0]
        if v.shape[0] != n or first < 0 or first > self.rows or first + n > self.capacity:
            raise ValueError(f"k and v: as many rows, from at most row {self.rows} on, up to row {self.capacity}")
        _same_device(self.device, k, v)
        with _on(self.device):
            call("nts_kv8_append", ptr(self.cache), ptr(self.scales), ptr(k), ptr(v), first, n, self.capacity, self.heads,
                 self.width, self.block_rows, _stream(self.device))
        self.rows = first + n


class NeighborAttentionOp:
    """out[d, h, :] = sum over d's edges of softmax(scale * <q[d, h], K[row, h']>) V[row, h'], read from a Kv8Cache; the log of
    each softmax's denominator is in `lse` afterwards.  layer: a SampledLayer, or a FullGraphChunk, whose row_indices are vertices.
    The cached rows are constants: there is no backward."""

    def __init__(self, layer, q_heads, scale=None):
        self.sg, self.q_heads, self.scale = layer, q_heads, scale
        self.lse = None

    def forward(self, q, cache, mirror=None):
        """mirror: the cache row of every local source (a sampled layer's dev_source where the cache holds all vertices);
        None: row_indices name cache rows.  Sources beyond mirror and rows that the cache does not hold are left out."""
        sg, H, D, dev = self.sg, self.q_heads, cache.width, cache.device
        _floats(q, H * D, "q")
        if q.shape[0] != sg.v_size or H % cache.heads:
            raise ValueError(f"q: a row for each of {sg.v_size} destinations; q_heads: a multiple of {cache.heads}")
        if mirror is not None:
            _indices(mirror, "mirror")
        co, ri = sg.dev_c_o(), sg.dev_r_i()
        _indices(co, "column_offset")
        _indices(ri, "row_indices")
        if co.numel() != sg.v_size + 1 or ri.numel() < sg.e_size:
            raise ValueError(f"layer: offsets of {sg.v_size} destinations and {sg.e_size} edges")
        _same_device(dev, q, mirror, co, ri)
        bound = getattr(sg, "max_in_degree", 0)
        scale = 1.0 / math.sqrt(D) if self.scale is None else self.scale
        out = allocate(torch.empty, sg.v_size, H * D, dtype=torch.float32, device=dev)
        lse = allocate(torch.empty, sg.v_size, H, dtype=torch.float32, device=dev)
        with _on(dev):
            size = call("nts_kv8_attention_work_bytes", sg.v_size, sg.e_size, H, D, bound)
            work = allocate(torch.empty, size, dtype=torch.uint8, device=dev) if size else None
            if mirror is None:
                call("nts_kv8_attention", ptr(out), ptr(lse), ptr(q), ptr(cache.cache), ptr(cache.scales), ptr(co), ptr(ri), 0,
                     sg.v_size, sg.e_size, cache.rows, H, cache.heads, D, cache.block_rows, scale, bound, ptr(work), _stream(dev))
            else:
                call("nts_kv8_attention_local", ptr(out), ptr(lse), ptr(q), ptr(cache.cache), ptr(cache.scales), ptr(co), ptr(ri),
                     ptr(mirror), mirror.numel(), sg.v_size, sg.e_size, cache.rows, H, cache.heads, D, cache.block_rows, scale,
                     bound, ptr(work), _stream(dev))
        self.lse = lse
        return out
