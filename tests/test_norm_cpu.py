"""Layer norm: what is refused, without a GPU."""
import ctypes as C

import pytest
import torch

from medicalimageanalysis_amd import _lib, norm


@pytest.mark.parametrize("x,weight,bias,error,match", [
    (torch.zeros(()), None, None, ValueError, "at least one dimension"),
    (torch.zeros(3, 0), None, None, ValueError, "empty"),
    (torch.zeros(3, 4, dtype=torch.int32), None, None, TypeError, "takes float32"),
    (torch.zeros(3, 4), torch.ones(3), None, ValueError, r"shape \(4,\)"),
    (torch.zeros(3, 4), torch.ones(4), torch.ones(1, 4), ValueError, r"shape \(4,\)"),
    (torch.zeros(3, 4), torch.ones(4, dtype=torch.bfloat16), None, TypeError, "float32"),
    (torch.zeros(3, 4, dtype=torch.float64), torch.ones(4), None, TypeError, "float64"),
    (torch.zeros(3, 4, dtype=torch.bfloat16), torch.ones(4), torch.ones(4, dtype=torch.bfloat16), TypeError, "differ"),
    (torch.zeros(3, 4), torch.ones(4), torch.ones(4), RuntimeError, "HIP device"),
])
def test_refusals(x, weight, bias, error, match):
    with pytest.raises(error, match=match):
        norm.layer_norm(x, weight, bias)


def test_module_has_the_state_of_torchs():
    ours, theirs = norm.LayerNorm(5), torch.nn.LayerNorm(5)
    assert {k: v.shape for k, v in ours.state_dict().items()} == {k: v.shape for k, v in theirs.state_dict().items()}
    with pytest.raises(ValueError, match="shape"):
        ours(torch.zeros(2, 4))


def test_c_entry_refusals():
    lib = _lib.lib()
    p = C.c_void_p(16)

    def fwd(n, width, stride=8, dtype=0, wdtype=0, x=p, mean=None, rstd=None):
        return lib.vmf_layer_norm_fwd(x, stride, None, None, p, mean, rstd, n, width, 1e-5, dtype, wdtype, None)

    assert fwd(-1, 8) == -1 and fwd(4, 0) == -1 and fwd(4, 8, stride=-8) == -1
    assert fwd(4, (1 << 24) + 1) == -4
    assert fwd(4, 8, dtype=4) == -2 and fwd(4, 8, dtype=0, wdtype=3) == -2 and fwd(4, 8, dtype=1, wdtype=0) == -2
    assert fwd(4, 8, x=None) == -1 and fwd(4, 8, mean=p) == -1
    assert fwd(0, 8, x=None) == 0
    nb = C.c_int64(-1)
    assert lib.vmf_layer_norm_bwd_workspace(10000, 128, 0, C.byref(nb)) == 0 and nb.value > 0
    assert lib.vmf_layer_norm_bwd_workspace(10000, 128, 0, None) == -1
    rc = lib.vmf_layer_norm_bwd(p, 128, p, 128, None, p, p, None, p, None, 10000, 128, p, nb.value - 1, 0, 0, None)
    assert rc == -1 and b"workspace" in lib.vmf_last_error_string()


class _Recorder:
    """in the library's place: every call succeeds, the backward call's arguments are kept"""

    def __init__(self):
        self.bwd = None

    def vmf_layer_norm_fwd(self, *args):
        return 0

    def vmf_layer_norm_bwd(self, *args):
        self.bwd = args
        return 0


@pytest.fixture
def recorder(monkeypatch):
    r = _Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: r)
    monkeypatch.setattr(_lib, "require_hip", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(_lib, "raw_stream", lambda dev: 0)
    monkeypatch.setattr(_lib, "workspace_bytes", lambda *sizes: 64)
    return r


def _backward_under(unpack, x):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = norm.layer_norm(x, torch.ones(x.shape[-1]), None)
    return torch.autograd.grad(y, x, torch.ones_like(y))


@pytest.mark.parametrize("rows,wide,width", [(40, 256, 128), (7, 5, 5), (1, 9, 4)])
def test_backward_reads_the_row_stride_of_the_tensor_that_a_hook_returns(recorder, rows, wide, width):
    """torch.autograd.graph.save_on_cpu gives a strided view back as a dense tensor; another hook may do the opposite"""
    returned = {}

    def dense(t):
        if t.dim() == 2:
            t = returned["x"] = t.clone(memory_format=torch.contiguous_format)
        return t

    def strided(t):
        if t.dim() == 2:
            out = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype)
            out[:, 1:1 + t.shape[1]] = t
            t = returned["x"] = out[:, 1:1 + t.shape[1]]
        return t

    for hook in (dense, strided):
        x = torch.randn(rows, wide)[:, :width].requires_grad_()
        _backward_under(hook, x)
        assert recorder.bwd[0] == returned["x"].data_ptr()
        if rows > 1:
            assert recorder.bwd[1] == returned["x"].stride(0)


@pytest.mark.parametrize("wrong", [lambda t: t.double(), lambda t: t[:-1], lambda t: t.to("meta")])
def test_backward_refuses_a_hook_that_returns_another_tensor(recorder, wrong):
    x = torch.randn(6, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="saved tensor came back"):
        _backward_under(wrong, x)
    assert recorder.bwd is None


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(recorder, which, grad):
    """a dual tensor has no requires_grad; without an error its tangent would read as zero"""
    from torch.autograd import forward_ad

    args = [torch.randn(3, 4), torch.ones(4), torch.zeros(4)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        assert forward_ad.unpack_dual(norm.layer_norm(*args)).tangent is None
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward mode"):
            norm.layer_norm(*args)


@pytest.mark.parametrize("dtype,size,wide", [(0, 4, 4), (1, 8, 8), (2, 2, 4), (3, 2, 4)])
@pytest.mark.parametrize("n,width", [(1, 40000), (5, 40001), (16, 1 << 24), (300, 40000), (16384, 40000), (4000, 1 << 20)])
def test_backward_workspace_of_long_rows_stays_below_the_input(n, width, dtype, size, wide):
    """two parts of a row for each 16 rows, and 2 MB (double: 4) for few rows that have to fill the chip"""
    need = C.c_int64(-1)
    assert _lib.lib().vmf_layer_norm_bwd_workspace(n, width, dtype, need) == 0
    assert 0 < need.value <= max(-(-n // 16) * 2 * width * wide, (1024 + -(-width // 256)) * 256 * 2 * wide)
