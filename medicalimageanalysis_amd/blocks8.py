"""8-bit blocks: activations kept and multiplied in 8 bits, for the hidden layers of wide models.

A block is 128 consecutive elements of a row, for a weight matrix a tile of 128 x 128: e4m3 values and one power-of-two
scale.  A hidden layer's activation in blocks is one byte per element where float32 keeps four, and it serves twice: as the
operand of the next layer's product and as the checkpoint that the backward pass reads.

  quantize(x, activation, beta)    blocks of x, or of softplus(x)                       -> Blocks8
  quantize_weight(w)               tiles of w and of its transpose                      -> Weight8
  Blocks8.dequantize(dtype)        what the blocks hold
  matmul(a, b, bias, dtype)        a b^T + bias
  softplus_grad(g, q, beta)        g * (1 - exp(-beta q)): the gradient through the softplus that q keeps
  weight_grad(g, q)                g^T q and the sum of g's rows: the gradients of the weight and the bias
  linear(x, weight, bias, activation, beta)
                                   blocks(activation(x)) tiles(weight)^T + bias, differentiable once

linear's gradients: gx = (blocks(gy) tiles(weight)) * softplus slope, gw = gy^T blocks(activation(x)), gb = the sum of
gy's rows; the roundings to 8 bits pass their gradient on as it is.  float32 results come from 32-bit sums, float16 and
bfloat16 ones from the 8-bit matrix instruction, which takes half the time: off by 1.3e-5 for normal values (a 37th and a
300th of their own half step), by at most 8.5e-4 of the sum of the terms' magnitudes where sizes differ widely inside a
block.  matmul(..., dtype=torch.float32) has 32-bit sums of any blocks, and so has the weight's gradient.  NaN and
infinities are NaN in blocks.  Only linear takes part in autograd, backwards (forward-mode derivatives are refused): the
other functions' results carry no gradient.  There is no CPU path.
"""
import torch

from . import _lib

BLOCK = 128
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_ACTIVATIONS = {None: _lib.ACT_NONE, "softplus": _lib.ACT_SOFTPLUS}


def _up(n, to):
    return -(-n // to) * to


class Blocks8:
    """A tensor in 8-bit blocks along its last dimension; `tiled`: one exponent per 128 x 128 tile (a weight).

    values     (rows, ceil(width / 128) * 128) uint8, e4m3 bits, zero behind the width
    exponents  (ceil(width / 128), pitch) uint8, e + 127; column r belongs to row r, tiled to rows 128 r ... 128 r + 127
    One allocation holds both."""

    __slots__ = ("storage", "shape", "rows", "width", "tiled", "exp_pitch", "exp_offset", "offset")

    def __init__(self, storage, shape, tiled=False, offset=0):
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] < 1 or (tiled and len(shape) != 2):
            raise ValueError(f"Blocks8: shape {tuple(shape)}")
        need = self.bytes_for(shape.numel() // shape[-1], shape[-1], tiled)
        if (storage.dtype != torch.uint8 or storage.dim() != 1 or not storage.is_contiguous() or offset < 0 or offset % 16
                or storage.numel() < offset + need):
            raise ValueError(f"Blocks8: {tuple(shape)} needs {need} bytes of a dense uint8 tensor from a multiple of 16 on, "
                             f"got {storage.dtype} of {tuple(storage.shape)} from {offset} on")
        self._set(storage, shape, shape.numel() // shape[-1], bool(tiled), offset)

    def _set(self, storage, shape, rows, tiled, offset):
        width = shape[-1]
        self.storage, self.shape, self.rows, self.width, self.tiled, self.offset = storage, shape, rows, width, tiled, offset
        self.exp_pitch = max(1, -(-rows // BLOCK)) if tiled else max(16, -(-rows // 16) * 16)
        self.exp_offset = offset - (-width // BLOCK) * BLOCK * rows

    @classmethod
    def _empty(cls, like, shape, rows):
        """blocks by rows, not yet written, on `like`'s device"""
        q = cls.__new__(cls)
        q._set(like.new_empty(cls.bytes_for(rows, shape[-1]), dtype=torch.uint8), shape, rows, False, 0)
        return q

    @staticmethod
    def bytes_for(rows, width, tiled=False):
        pitch = max(1, _up(rows, BLOCK) // BLOCK) if tiled else max(16, _up(rows, 16))
        return _up(rows * _up(width, BLOCK) + _up(width, BLOCK) // BLOCK * pitch, 16)

    @property
    def device(self):
        return self.storage.device

    @property
    def values(self):
        pitch = _up(self.width, BLOCK)
        return self.storage[self.offset:self.offset + self.rows * pitch].view(self.rows, pitch)

    @property
    def exponents(self):
        blocks = _up(self.width, BLOCK) // BLOCK
        return self.storage[self.exp_offset:self.exp_offset + blocks * self.exp_pitch].view(blocks, self.exp_pitch)

    def _addresses(self):
        base = self.storage.data_ptr()
        return base + self.offset, base + self.exp_offset

    def dequantize(self, dtype=torch.float32):
        """the elements as `dtype` (every one is exact in float32 and bfloat16)"""
        code = _code(dtype, "dequantize")
        dev = _lib.require_hip(self.storage)
        out = self.storage.new_empty(self.shape, dtype=dtype)
        v, e = self._addresses()
        with _lib.on_device(dev):
            rc = _lib.lib().vmf_blocks8_dequantize(v, e, self.exp_pitch, self.tiled, out.data_ptr(), self.rows,
                                                   self.width, code, _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "vmf_blocks8_dequantize")
        return out

    def __repr__(self):
        return f"Blocks8({tuple(self.shape)}{', tiled' if self.tiled else ''}, device='{self.device}')"


class Weight8:
    """A weight matrix (n, k) laid out for `linear`: its 128 x 128 tiles (`rows`, k wide) and the same tiles transposed
    (`columns`, n wide; None if left out), which the gradient of the layer's input reads."""

    __slots__ = ("rows", "columns", "dtype")

    def __init__(self, rows, columns, dtype):
        _blocks("Weight8", rows, *(() if columns is None else (columns,)))
        if not rows.tiled or (columns is not None and (not columns.tiled or columns.shape != rows.shape[::-1]
                                                       or columns.device != rows.device)):
            raise ValueError(f"Weight8: {rows} and {columns} are not the tiles of a matrix and of its transpose")
        self.rows, self.columns, self.dtype = rows, columns, dtype

    @property
    def shape(self):
        return self.rows.shape

    @property
    def device(self):
        return self.rows.device


def _code(dtype, what):
    if dtype not in _FLOATS:
        raise TypeError(f"{what} takes float32, float16 or bfloat16, got {dtype}")
    return _lib.FLOAT_CODES[dtype]


def _blocks(what, *operands):
    for q in operands:
        if not isinstance(q, Blocks8):
            raise TypeError(f"{what} takes Blocks8 (quantize, or the rows / columns of quantize_weight), got "
                            f"{type(q).__name__}")


def _activation(activation, beta, what):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None or 'softplus', got {activation!r}")
    beta = float(beta)
    if activation is not None and not 1e-30 <= beta <= 1e30:
        raise ValueError(f"{what}: beta must be positive, got {beta}")
    return _ACTIVATIONS[activation], beta


def _width(x, what):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: the last dimension must hold at least one element, got the shape {tuple(x.shape)}")


def _quantize(x, act, beta, code, dev):
    rows, stride = _lib.as_rows(x.detach())
    n, width = rows.shape
    q = Blocks8._empty(x, x.shape, n)
    v, e = q._addresses()
    with _lib.on_device(dev):
        rc = _lib.lib().vmf_blocks8_quantize(rows.data_ptr(), stride, v, e, q.exp_pitch, n, width, act, beta, code,
                                             _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_blocks8_quantize")
    return q


def quantize(x, activation=None, beta=1.0):
    """8-bit blocks of x, or with activation="softplus" of log(1 + exp(beta x)) / beta."""
    _width(x, "quantize")
    code = _code(x.dtype, "quantize")
    act, beta = _activation(activation, beta, "quantize")
    return _quantize(x, act, beta, code, _lib.require_hip(x))


def _quantize_weight(w, transpose, dev):
    rows, stride = _lib.as_rows(w.detach())
    n, k = w.shape
    first = Blocks8.bytes_for(n, k, True)
    storage = torch.empty(first + (Blocks8.bytes_for(k, n, True) if transpose else 0), device=dev, dtype=torch.uint8)
    by_rows = Blocks8(storage, (n, k), True)
    by_columns = Blocks8(storage, (k, n), True, first) if transpose else None
    v, e = by_rows._addresses()
    vt, et = by_columns._addresses() if transpose else (None, None)
    with _lib.on_device(dev):
        rc = _lib.lib().vmf_blocks8_quantize_tiles(rows.data_ptr(), stride, v, e, vt, et, n, k,
                                                   _lib.FLOAT_CODES[w.dtype], _lib.raw_stream(dev))
    _lib.check(rc, "vmf_blocks8_quantize_tiles")
    return Weight8(by_rows, by_columns, w.dtype)


def quantize_weight(w, transpose=True):
    """The 128 x 128 tiles of a weight matrix (n, k); transpose=False leaves out what only an input gradient reads."""
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"quantize_weight: a matrix is wanted, got the shape {tuple(w.shape)}")
    _code(w.dtype, "quantize_weight")
    return _quantize_weight(w, transpose, _lib.require_hip(w))


def _matmul(a, b, bias, gate, beta, dtype, dev):
    m, n, k = a.rows, b.rows, a.width
    code = _lib.FLOAT_CODES[dtype]
    out = a.storage.new_empty(a.shape[:-1] + (n,), dtype=dtype)
    lib = _lib.lib()
    need = _lib.workspace_bytes("vmf_blocks8_matmul_workspace", m, n, k, code)
    ws = a.storage.new_empty(need) if need else None
    av, ae = a._addresses()
    bv, be = b._addresses()
    gv, ge = gate._addresses() if gate is not None else (None, None)
    with _lib.on_device(dev):
        rc = lib.vmf_blocks8_matmul(av, ae, a.exp_pitch, a.tiled, bv, be, b.exp_pitch, b.tiled, _lib.address(bias),
                                    _lib.FLOAT_CODES[bias.dtype] if bias is not None else 0, gv, ge,
                                    gate.exp_pitch if gate is not None else 0, beta, out.data_ptr(), m, n, k,
                                    _lib.address(ws), need, code, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_blocks8_matmul")
    return out


def _check_bias(bias, n, what):
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"{what}: the bias must have shape ({n},), got {tuple(bias.shape)}")
        _code(bias.dtype, what)


def matmul(a, b, bias=None, dtype=torch.float32):
    """a b^T + bias of two Blocks8 of the same width: (..., k), (n, k) -> (..., n)."""
    _blocks("matmul", a, b)
    if len(b.shape) != 2 or a.width != b.width:
        raise ValueError(f"matmul: shapes {tuple(a.shape)} and {tuple(b.shape)}")
    _code(dtype, "matmul")
    _check_bias(bias, b.rows, "matmul")
    dev = _lib.require_hip(a.storage, b.storage, bias)
    return _matmul(a, b, None if bias is None else bias.detach().contiguous(), None, 1.0, dtype, dev)


def softplus_grad(g, q, beta=1.0):
    """g * (1 - exp(-beta q)), q = quantize(h, "softplus", beta): the gradient with respect to h."""
    _blocks("softplus_grad", q)
    code = _code(g.dtype, "softplus_grad")
    _, beta = _activation("softplus", beta, "softplus_grad")
    if g.shape != q.shape or q.tiled:
        raise ValueError(f"softplus_grad: shapes {tuple(g.shape)} and {tuple(q.shape)}")
    dev = _lib.require_hip(g, q.storage)
    rows, stride = _lib.as_rows(g.detach())
    out = torch.empty_like(g, memory_format=torch.contiguous_format)
    v, e = q._addresses()
    with _lib.on_device(dev):
        rc = _lib.lib().vmf_blocks8_softplus_grad(rows.data_ptr(), stride, v, e, q.exp_pitch, out.data_ptr(), q.rows,
                                                  q.width, beta, code, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_blocks8_softplus_grad")
    return out


def _weight_grad(g, q, bias, dtype, dev):
    rows, stride = _lib.as_rows(g.detach())
    m, n = rows.shape
    k = q.width
    gw = g.new_empty((n, k), dtype=dtype)
    gb = g.new_empty(n, dtype=dtype) if bias else None
    lib = _lib.lib()
    code = _lib.FLOAT_CODES[g.dtype]
    need = _lib.workspace_bytes("vmf_blocks8_weight_grad_workspace", m, n, k, code)
    ws = q.storage.new_empty(need) if need else None
    v, e = q._addresses()
    with _lib.on_device(dev):
        rc = lib.vmf_blocks8_weight_grad(rows.data_ptr(), stride, v, e, q.exp_pitch, gw.data_ptr(), _lib.address(gb), None,
                                         None, 0, m, n, k, _lib.address(ws), need, code, _lib.FLOAT_CODES[dtype],
                                         _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_blocks8_weight_grad")
    return gw, gb


def weight_grad(g, q, bias=True, dtype=torch.float32):
    """(g^T q, sum of g's rows) over all leading dimensions: the gradients of a layer's weight and bias from the
    gradient g (..., n) of its result and its kept input q (..., k); bias=False leaves the second out (None)."""
    _blocks("weight_grad", q)
    _code(g.dtype, "weight_grad")
    _width(g, "weight_grad")
    if dtype not in (torch.float32, g.dtype):
        raise TypeError(f"weight_grad: results are float32 or the gradient's {g.dtype}, got {dtype}")
    if q.tiled or g.shape[:-1] != q.shape[:-1]:
        raise ValueError(f"weight_grad: shapes {tuple(g.shape)} and {tuple(q.shape)}")
    return _weight_grad(g, q, bias, dtype, _lib.require_hip(g, q.storage))


def _linear(x, weight, laid_out, bias, act, beta, dev, keep, columns):
    """(y, kept, wt, sizes).  keep: kept holds x's blocks and, if `columns`, those of the transposed weight from wt[0] on
    (wt: where its values and its exponents start; None without).  What is not kept lives in the workspace, and ends with
    the call."""
    rows, stride = _lib.as_rows(x)
    m, k = rows.shape
    code = _lib.FLOAT_CODES[x.dtype]
    lib = _lib.lib()
    w = wv = we = kept = wt = base = base_e = tv = te = None
    w_stride = w_code = pitch = 0
    if laid_out is None:
        n = weight.shape[0]
        w, w_stride = _lib.as_rows(weight)
        w_code = _lib.FLOAT_CODES[w.dtype]
    else:
        n = laid_out.rows.rows
        wv, we = laid_out.rows._addresses()
    need = _lib.workspace_bytes("vmf_blocks8_linear_fwd_workspace", m, n, k, laid_out is not None, keep, code)
    if keep:
        kp = _up(k, BLOCK)
        pitch = max(16, _up(m, 16))
        size = _up(m * kp + kp // BLOCK * pitch, 16)  # Blocks8.bytes_for(m, k)
        if columns and laid_out is None:
            wt = (size, size + k * _up(n, BLOCK))
            size += Blocks8.bytes_for(k, n, True)
        kept = x.new_empty(size, dtype=torch.uint8)
        base = kept.data_ptr()
        base_e = base + m * kp
        if wt is not None:
            tv, te = base + wt[0], base + wt[1]
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    y = x.new_empty(x.shape[:-1] + (n,))
    b = _lib.dense(bias)
    with _lib.on_device(dev):
        rc = lib.vmf_blocks8_linear_fwd(rows.data_ptr(), stride, _lib.address(w), w_stride, w_code, wv, we, tv, te,
                                        _lib.address(b), 0 if b is None else _lib.FLOAT_CODES[b.dtype], act, beta, base,
                                        base_e, pitch, y.data_ptr(), m, n, k, _lib.address(ws), need, code,
                                        _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_blocks8_linear_fwd")
    return y, kept, wt, (m, n, k)


def _bias_grad(g, stride, gb, m, n, code, dev):
    """the sum of g's rows into gb (float32 or g's type)"""
    need = _lib.workspace_bytes("vmf_blocks8_bias_grad_workspace", m, n, code)
    ws = g.new_empty(need, dtype=torch.uint8) if need else None
    with _lib.on_device(dev):
        rc = _lib.lib().vmf_blocks8_bias_grad(g.data_ptr(), stride, gb.data_ptr(), m, n, _lib.address(ws), need, code,
                                              _lib.FLOAT_CODES[gb.dtype], _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_blocks8_bias_grad")


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, how):
        laid_out, act, beta, dev = how
        need_x = ctx.needs_input_grad[0]
        if need_x and laid_out is not None and laid_out.columns is None:
            raise ValueError("linear: the laid-out weight has no columns (quantize_weight(..., transpose=True)), which "
                             "the gradient of x reads")
        keep = need_x or ctx.needs_input_grad[1]  # (a bias's gradient reads neither)
        y, kept, wt, sizes = _linear(x, weight, laid_out, bias, act, beta, dev, keep, need_x)
        # kept for the backward pass: x in 8 bits and, for its own gradient, the transposed weight in 8 bits
        other = None
        if need_x and laid_out is not None:
            columns = laid_out.columns
            other, wt = columns.storage, (columns.offset, columns.exp_offset)
        ctx.save_for_backward(kept, other)
        ctx.meta = (x.shape, sizes, wt, act, beta, None if weight is None else weight.dtype,
                    None if bias is None else bias.dtype, dev, kept.numel() if keep else 0,
                    0 if other is None else other.numel())
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, gy):
        kept, other = ctx.saved_tensors
        shape, (m, n, k), wt, act, beta, w_dtype, bias_dtype, dev, kept_bytes, other_bytes = ctx.meta
        kept = _lib.dense(_lib.unpacked(kept, torch.uint8, (kept_bytes,), dev))
        other = _lib.dense(_lib.unpacked(other, torch.uint8, (other_bytes,), dev))
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        code = _lib.FLOAT_CODES[gy.dtype]
        g, stride = _lib.as_rows(gy)
        # the weight's gradient has the weight's type, the bias's its own: where the call that computes it does not give that,
        # from the 32-bit sums
        out = w_dtype or torch.float32
        gx = gw = gb = gb_too = None
        if need_b:
            gb = gy.new_empty(n, dtype=bias_dtype if bias_dtype == (out if need_w else gy.dtype) else torch.float32)
            if need_w:
                gb_too = gb.data_ptr()
            else:
                _bias_grad(g, stride, gb, m, n, code, dev)
        if need_x or need_w:
            if need_x:
                gx = gy.new_empty(shape)
            if need_w:
                gw = gy.new_empty((n, k), dtype=out)
            need = _lib.workspace_bytes("vmf_blocks8_linear_bwd_workspace", m, n, k, code)
            ws = gy.new_empty(need, dtype=torch.uint8)
            base = kept.data_ptr()
            tv = te = None
            if need_x:
                at = base if other is None else other.data_ptr()
                tv, te = at + wt[0], at + wt[1]
            out_code = _lib.FLOAT_CODES[out]
            if gb_too is not None and gb.dtype != out:
                out_code |= _lib.GBIAS_F32
            with _lib.on_device(dev):
                rc = _lib.lib().vmf_blocks8_linear_bwd(g.data_ptr(), stride, base, base + m * _up(k, BLOCK),
                                                       max(16, _up(m, 16)), tv, te, act, beta, _lib.address(gx),
                                                       _lib.address(gw), gb_too, m, n, k, ws.data_ptr(), need, code,
                                                       out_code, _lib.raw_stream(dev))
            if rc:
                _lib.check(rc, "vmf_blocks8_linear_bwd")
        if gb is not None and gb.dtype != bias_dtype:
            gb = gb.to(bias_dtype)
        return gx, gw, gb, None


def linear(x, weight, bias=None, activation=None, beta=1.0):
    """blocks(activation(x)) tiles(weight)^T + bias for x (..., k): (..., n) of x's type.

    weight: a matrix (n, k) of x's type or float32, quantised in the call (training), or a Weight8 that was laid out once
    (serving; no gradient of its own).  Keeps one byte per element of x for the backward pass (none where only the bias takes
    a gradient).  bias: float32, float16 or bfloat16, and so is its gradient."""
    _width(x, "linear")
    _code(x.dtype, "linear")
    act, beta = _activation(activation, beta, "linear")
    laid_out = weight if isinstance(weight, Weight8) else None
    if laid_out is None:
        if weight.dim() != 2 or weight.shape[0] < 1:
            raise ValueError(f"linear: the weight must be a matrix, got the shape {tuple(weight.shape)}")
        if weight.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"linear: the weight of {x.dtype} rows is {x.dtype} or float32, got {weight.dtype}")
    n, k = weight.shape
    if k != x.shape[-1]:
        raise ValueError(f"linear: x of shape {tuple(x.shape)} and a weight of shape {tuple(weight.shape)}")
    _check_bias(bias, n, "linear")
    dev = _lib.require_hip(x, weight if laid_out is None else laid_out.rows.storage, bias)
    tensor = weight if laid_out is None else None
    if _lib.differentiated(x, tensor, bias):
        return _Linear.apply(x, tensor, bias, (laid_out, act, beta, dev))
    return _linear(x, tensor, laid_out, bias, act, beta, dev, False, False)[0]
