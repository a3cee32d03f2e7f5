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
