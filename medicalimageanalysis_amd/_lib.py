"""ctypes binding of libvmf_hip.so (the C ABI declared in include/vmf_hip.h).

There is no CPU fallback: a missing library, a failed call or a tensor that is not on a HIP device
raises.  PyTorch supplies device memory and the current stream; every kernel is in the .so.
"""
import ctypes as C
import functools
import os
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

_HERE = os.path.dirname(os.path.abspath(__file__))
_DEFAULT = os.path.join(_HERE, "libvmf_hip.so")

VMF_F32, VMF_F64, VMF_F16, VMF_BF16 = range(4)
FLOAT_CODES = {torch.float32: VMF_F32, torch.float64: VMF_F64, torch.float16: VMF_F16, torch.bfloat16: VMF_BF16}
FLAG_NORMALIZE_MU = 1
FLAG_SOFTPLUS_KAPPA = 2
KIND_GENERAL, KIND_ROWS, KIND_OUTER = 0, 1, 2
KL_SPHERICAL_PIECEWISE, KL_TORUS_RAW, KL_CIRCULAR_EPS, KL_S1_I0I1, KL_STABLE_M3, KL_STABLE_M2 = range(6)
KL_WORKSPACE_DOUBLES = 1024
KL_STATIC_MAX_N = 1 << 30
ELBO_WORKSPACE_DOUBLES = 2048
LATENT_S1, LATENT_S2, LATENT_T2 = range(3)
ACT_NONE, ACT_SOFTPLUS = range(2)
GBIAS_F32 = 0x100

# (the module object `C` is re-used by callers for byref / c_int64)
_P, _I64, _U64, _I, _D = C.c_void_p, C.c_int64, C.c_uint64, C.c_int, C.c_double
_I64P = C.POINTER(C.c_int64)

# name -> argtypes; every function returns int except the two noted below
_PROTOS = {
    "vmf3_rsample_fwd": [_P, _P, _P, _P, _P, _P, _P, _I, _I64P, _I64P, _I64P, _I64P, _I64P, _I, _I, _U64, _U64, _U64,
                         _P, _P],
    "vmf3_broadcast_kind": [_I, _I64P, _I64P, _I64P, _I64P, _I64P, _I64P, _I64P],
    "vmf3_rsample_bwd": [_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I, _I64P, _I64P, _I64P, _I64P, _I64P, _I, _I,
                         _U64, _U64, _U64, _P, _P],
    "vmf3_rsample_bwd_outer_workspace": [_I64, _I64, _I, _I64P],
    "vmf3_rsample_bwd_outer": [_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _P, _I64, _I, _I, _U64, _U64, _U64, _P, _P],
    "vmf3_sample_w_fwd": [_P, _P, _P, _I64, _I64, _I, _U64, _U64, _U64, _P, _P],
    "vmf3_sample_w_bwd": [_P, _P, _P, _P, _I64, _I64, _I, _U64, _U64, _U64, _P, _P],
    "vmf3_log_prob_ref": [_P, _P, _P, _P, _P, _I64, _I, _P],
    "vmf3_log_prob_ref_bwd": [_P, _P, _P, _P, _P, _P, _P, _I64, _I, _P],
    "vmf3_mean": [_P, _P, _P, _I64, _I, _P],
    "vmf_ive_fwd": [_D, _P, _P, _I64, _I, _P],
    "vmf_ive_bwd": [_D, _P, _P, _P, _I64, _I, _P],
    "vmf_log_ive_fwd": [_D, _P, _P, _I64, _I, _P],
    "vmf_bessel_ratio_fwd": [_D, _P, _P, _I64, _I, _P],
    "vmf_kl_fwd": [_P, _P, _P, _P, _D, _I64, _I, _I, _P],
    "vmf_kl_fwd_static": [_P, _P, _P, _D, _I64, _I, _I, _P],
    "vmf_allreduce_scalars": [_P, _P, _I, _P],
    "vmf_philox_ticket": [_P, _P, _P],
    "vmf_kl_bwd": [_P, _P, _I64, _D, _P, _I64, _I, _I, _P],
    "vmf_rsample_fwd": [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P, _I64, _I, _P, _P, _I, _P, _I, _U64, _U64, _U64, _P,
                        _I, _I, _P],
    "vmf_rsample_bwd": [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P, _P, _I64, _I, _U64, _U64, _U64, _P, _I, _I, _P],
    "vmf_log_prob_fwd": [_P, _I64, _P, _I64, _P, _P, _I64, _I, _I, _P],
    "vmf_log_prob_bwd": [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _I64, _I, _I, _P],
    "vmf_entropy_kl_fwd": [_P, _P, _P, _P, _I64, _I, _I, _P],
    "vmf_sphere_uniform_sample": [_P, _P, _I64, _I, _U64, _U64, _U64, _P, _I, _P],
    "vmf_s1_projnormal_fwd": [_P, _P, _P, _P, _I64, _I, _U64, _U64, _U64, _P, _I, _P],
    "vmf_s1_projnormal_bwd": [_P, _P, _P, _P, _P, _P, _I64, _I, _U64, _U64, _U64, _P, _I, _P],
    "vmf_elbo_fwd": [_P, _P, _P, _P, _P, _P, _D, _D, _I64, _I64, _I64, _I, _I, _P],
    "vmf_elbo_bwd": [_P, _P, _P, _P, _P, _P, _D, _D, _I64, _I64, _I64, _I, _I, _P],
    "vmf_build_torus_fwd": [_P, _P, _P, _I64, _I, _D, _D, _I, _P],
    "vmf_build_torus_bwd": [_P, _P, _P, _P, _P, _I64, _I, _D, _D, _I, _P],
    "vmf_latent_loss_fwd": [_P, _P, _P, _P, _P, _I64, _I, _I64, _I, _I, _D, _D, _I, _P],
    "vmf_latent_loss_bwd": [_P, _P, _P, _P, _I64, _I, _I64, _I, _I, _D, _D, _I, _P],
    "vmf_layer_norm_fwd": [_P, _I64, _P, _P, _P, _P, _P, _I64, _I64, _D, _I, _I, _P],
    "vmf_layer_norm_bwd_workspace": [_I64, _I64, _I, _I64P],
    "vmf_layer_norm_bwd": [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P, _I64, _I64, _P, _I64, _I, _I, _P],
    "vmf_blocks8_quantize": [_P, _I64, _P, _P, _I64, _I64, _I64, _I, _D, _I, _P],
    "vmf_blocks8_quantize_tiles": [_P, _I64, _P, _P, _P, _P, _I64, _I64, _I, _P],
    "vmf_blocks8_dequantize": [_P, _P, _I64, _I, _P, _I64, _I64, _I, _P],
    "vmf_blocks8_softplus_grad": [_P, _I64, _P, _P, _I64, _P, _I64, _I64, _D, _I, _P],
    "vmf_blocks8_matmul_workspace": [_I64, _I64, _I64, _I, _I64P],
    "vmf_blocks8_matmul": [_P, _P, _I64, _I, _P, _P, _I64, _I, _P, _I, _P, _P, _I64, _D, _P, _I64, _I64, _I64, _P, _I64,
                           _I, _P],
    "vmf_blocks8_weight_grad_workspace": [_I64, _I64, _I64, _I, _I64P],
    "vmf_blocks8_weight_grad": [_P, _I64, _P, _P, _I64, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _I64, _I, _I, _P],
    "vmf_blocks8_bias_grad_workspace": [_I64, _I64, _I, _I64P],
    "vmf_blocks8_bias_grad": [_P, _I64, _P, _I64, _I64, _P, _I64, _I, _I, _P],
    "vmf_blocks8_linear_fwd_workspace": [_I64, _I64, _I64, _I, _I, _I, _I64P],
    "vmf_blocks8_linear_fwd": [_P, _I64, _P, _I64, _I, _P, _P, _P, _P, _P, _I, _I, _D, _P, _P, _I64, _P, _I64, _I64, _I64,
                               _P, _I64, _I, _P],
    "vmf_blocks8_linear_bwd_workspace": [_I64, _I64, _I64, _I, _I64P],
    "vmf_blocks8_linear_bwd": [_P, _I64, _P, _P, _I64, _P, _P, _I, _D, _P, _P, _P, _I64, _I64, _I64, _P, _I64, _I, _I,
                               _P],
}
EXPORTS = sorted(list(_PROTOS) + ["vmf_version", "vmf_last_error_string"])

_lib = None
_lock = threading.Lock()


def library_path():
    return os.environ.get("VMF_HIP_LIB", _DEFAULT)


def lib():
    """Load the shared library once; raise loudly when it is missing or incomplete."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                path = library_path()
                if not os.path.exists(path):
                    raise RuntimeError(
                        f"libvmf_hip.so not found at {path}: build it with "
                        "`make -C medicalimageanalysis_amd/csrc` (or `python -c 'import __graft_entry__ as g; "
                        "g.build()'`); there is no CPU fallback")
                h = C.CDLL(path)
                for name, argtypes in _PROTOS.items():
                    f = getattr(h, name)  # AttributeError if the symbol is missing
                    f.argtypes = argtypes
                    f.restype = C.c_int
                h.vmf_version.restype = C.c_int
                h.vmf_last_error_string.restype = C.c_char_p
                _lib = h
    return _lib


def check(rc, what):
    if rc != 0:
        msg = lib().vmf_last_error_string().decode("utf-8", "replace")
        raise RuntimeError(f"{what} failed (status {rc}): {msg}")


def dtype_code(t):
    if t.dtype == torch.float32:
        return VMF_F32
    if t.dtype == torch.float64:
        return VMF_F64
    raise TypeError(f"libvmf_hip supports float32 and float64 tensors, got {t.dtype}")


def float_code(t, what, accepted):
    """the library's code of a tensor's type, for the calls that take more than dtype_code's two"""
    if t.dtype not in accepted:
        names = ", ".join(str(d).replace("torch.", "") for d in accepted)
        raise TypeError(f"{what} takes {names} tensors, got {t.dtype}")
    return FLOAT_CODES[t.dtype]


def as_rows(t):
    """(n, width) view of a tensor with its row stride; a copy only where the last dimension is not dense or the
    leading ones have no common stride"""
    width = t.shape[-1]
    n = t.numel() // width if width else 0
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1):
        r = t
    else:
        try:
            r = t.view(n, width)
        except RuntimeError:
            r = t.contiguous().view(n, width)
        if r.stride(1) != 1 and width != 1:
            r = r.contiguous()
    return r, (r.stride(0) if n > 1 else width)


def unpacked(t, dtype, shape, device):
    """A saved tensor as autograd hands it back.  Saved-tensor hooks (torch.autograd.graph.save_on_cpu among them) may give
    it another layout, so strides are read from it and never remembered; one of another type, shape or device is refused
    before a kernel gets its address."""
    if t is not None and (t.dtype != dtype or t.shape != shape or t.device != device):
        raise RuntimeError(f"a saved tensor came back as {t.dtype} of {tuple(t.shape)} on {t.device}, saved was {dtype} of "
                           f"{tuple(shape)} on {device}")
    return t


def require_hip(*tensors):
    """Every tensor must live on one HIP device; returns that device."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                "medicalimageanalysis_amd runs on MI355X only: got a tensor on "
                f"'{t.device}'. Move the inputs to a HIP device (tensor.to('cuda')); there is no CPU path.")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    return dev


class _Noop:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NOOP = _Noop()


def on_device(dev):
    """Context that makes `dev` the current device for a launch (the library launches on the current device).  When
    it already is -- the usual case -- nothing is switched: torch.cuda.device() costs several microseconds per call,
    a visible share of a launch at the reference's batch sizes."""
    if dev.index is None or torch.cuda.current_device() == dev.index:
        return _NOOP
    return torch.cuda.device(dev)


_workspaces = {}
_retired_workspaces = []


def workspace(dev, n_doubles):
    """Scratch of AT LEAST `n_doubles` float64 for a reduction's block partials (callers pass its real size on): ONE
    buffer per (device, stream), grown in powers of two to the largest request seen, kept for the life of the process.
    Launches on one stream are ordered, so back-to-back calls may share it, and a train step captured into a HIP graph
    contains no allocation for it (the warm-up steps before the capture created it).  A buffer that is outgrown is kept
    alive as well -- a graph captured earlier may still point at it -- which at most doubles the footprint of the
    largest request.  A first call made while the stream is capturing gets a buffer of its own from the capture's pool."""
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < n_doubles:
        size = 1 << max(10, int(n_doubles - 1).bit_length())
        new = torch.empty(size, device=dev, dtype=torch.float64)
        if torch.cuda.is_current_stream_capturing():
            return new
        if ws is not None:
            _retired_workspaces.append(ws)
        _workspaces[key] = ws = new
    return ws


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def stream_ptr(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


@functools.lru_cache(maxsize=1024)
def workspace_bytes(entry, *sizes):
    """the answer of a `..._workspace` entry point, which hangs on the sizes alone"""
    need = C.c_int64(0)
    check(getattr(lib(), entry)(*sizes, need), entry)
    return need.value


def differentiated(*tensors):
    """Whether a call on these tensors goes through its autograd Function: a gradient is wanted of one of them, or
    forward-mode derivatives are being taken (a dual tensor has no requires_grad; the Function refuses it, where the call
    without one would drop its tangent)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def first_order(backward):
    """A Function's backward that is differentiable once.  Under create_graph=True it goes through torch's
    once_differentiable, which makes a second derivative an error; otherwise, the usual case, it is called directly: the
    wrapper's bookkeeping costs more than the calls of a small layer."""
    checked = once_differentiable(backward)

    def call(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return call


def dense(t):
    """a vector (or None) whose elements lie side by side"""
    return t if t is None or t.is_contiguous() else t.contiguous()


def address(t):
    """a tensor's address as a plain integer (ctypes takes it for a pointer argument without building an object)"""
    return None if t is None else t.data_ptr()


def raw_stream(device):
    """the current stream's handle as a plain integer"""
    return torch._C._cuda_getCurrentRawStream(device.index)


def i64_array(seq):
    return (C.c_int64 * len(seq))(*[int(s) for s in seq])
