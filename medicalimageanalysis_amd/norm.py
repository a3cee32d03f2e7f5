"""Layer norm over the last dimension, for the hidden layers of wide models:

    y = (x - mean) / sqrt(var + eps) * weight + bias

layer_norm is differentiable once, in x, weight and bias, backwards only (forward-mode derivatives are refused); LayerNorm
is the module.  The rows may be float32, float64, float16 or bfloat16, the weight and the bias of the same type or, with
16-bit rows, float32; sums and statistics are held in 32 bits (64 for float64 rows).  x may be any view whose last dimension
is dense and whose rows have one stride; other views are copied.  There is no CPU path.
"""
import torch

from . import _lib


_ROWS = (torch.float32, torch.float64, torch.float16, torch.bfloat16)


def _check(x, weight, bias):
    if x.dim() < 1:
        raise ValueError("layer_norm: x needs at least one dimension")
    width = x.shape[-1]
    if width < 1:
        raise ValueError("layer_norm: the last dimension is empty")
    code = wcode = _lib.float_code(x, "layer_norm", _ROWS)
    first = None
    for p in (weight, bias):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != width:
            raise ValueError(f"layer_norm: weight and bias must have shape ({width},), got {tuple(p.shape)}")
        if first is not None and p.dtype != first:
            raise TypeError(f"layer_norm: weight and bias differ in type ({first}, {p.dtype})")
        first = p.dtype
        wcode = _lib.FLOAT_CODES.get(first, -1)
        if wcode != code and not (wcode == _lib.VMF_F32 and code in (_lib.VMF_F16, _lib.VMF_BF16)):
            raise TypeError(f"layer_norm: weight and bias of {x.dtype} rows are {x.dtype}"
                            f"{' or float32' if code in (_lib.VMF_F16, _lib.VMF_BF16) else ''}, got {first}")
    return _lib.require_hip(x, weight, bias), code, wcode


def _forward(x, w, b, eps, dev, code, wcode, keep):
    rows, stride = _lib.as_rows(x)
    n, width = rows.shape
    w, b = _lib.dense(w), _lib.dense(b)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)  # (empty_like: half the host time of empty)
    stats = mean = rstd = None
    if keep:  # the rows' means, then their reciprocal deviations
        stats = rows.new_empty(2 * n, dtype=torch.float64 if code == _lib.VMF_F64 else torch.float32)
        mean = stats.data_ptr()
        rstd = mean + n * (8 if code == _lib.VMF_F64 else 4)
    with _lib.on_device(dev):
        rc = _lib.lib().vmf_layer_norm_fwd(rows.data_ptr(), stride, _lib.address(w), _lib.address(b), y.data_ptr(),
                                           mean, rstd, n, width, eps, code, wcode, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "vmf_layer_norm_fwd")
    return y, rows, w, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, how):
        eps, dev, code, wcode = how
        y, rows, w, stats = _forward(x, weight, bias, eps, dev, code, wcode, True)
        ctx.save_for_backward(rows, w, stats)
        ctx.meta = (rows.shape, x.dtype, None if w is None else w.dtype, stats.dtype, code, wcode, dev,
                    None if bias is None else bias.dtype)
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, gy):
        rows, w, stats = ctx.saved_tensors
        shape, x_dtype, w_dtype, stats_dtype, code, wcode, dev, b_dtype = ctx.meta
        n, width = shape
        rows, x_stride = _lib.as_rows(_lib.unpacked(rows, x_dtype, shape, dev))
        w = _lib.dense(_lib.unpacked(w, w_dtype, (width,), dev))
        stats = _lib.dense(_lib.unpacked(stats, stats_dtype, (2 * n,), dev))
        g, g_stride = _lib.as_rows(gy)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        gx = torch.empty_like(gy, memory_format=torch.contiguous_format) if need_x else None
        gw = torch.empty_like(w) if need_w else None
        gb = rows.new_empty(width, dtype=b_dtype) if need_b else None
        ws, need = None, 0
        if need_w or need_b:
            need = _lib.workspace_bytes("vmf_layer_norm_bwd_workspace", n, width, code)
            if need:
                ws = rows.new_empty(need, dtype=torch.uint8)
        mean = stats.data_ptr()
        with _lib.on_device(dev):
            rc = _lib.lib().vmf_layer_norm_bwd(rows.data_ptr(), x_stride, g.data_ptr(), g_stride, _lib.address(w), mean,
                                               mean + n * (8 if code == _lib.VMF_F64 else 4), _lib.address(gx),
                                               _lib.address(gw), _lib.address(gb), n, width, _lib.address(ws), need, code,
                                               wcode, _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "vmf_layer_norm_bwd")
        return gx, gw, gb, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x."""
    dev, code, wcode = _check(x, weight, bias)
    eps = float(eps)
    if _lib.differentiated(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, (eps, dev, code, wcode))
    return _forward(x, weight, bias, eps, dev, code, wcode, False)[0]


class LayerNorm(torch.nn.LayerNorm):
    """torch.nn.LayerNorm over one dimension with the kernels of this module: the same parameters and state dict."""

    def __init__(self, width, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(int(width), eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device,
                         dtype=dtype)

    def forward(self, x):
        if x.dim() < 1 or x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm({self.normalized_shape[0]}): got the shape {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
