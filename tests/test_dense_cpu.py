"""CPU: the dense operators' refusals, through Python and the C ABI (no GPU calls)."""
import ctypes

import pytest
import torch

import velvetoptimizer_b200 as vb
from velvetoptimizer_b200 import _lib


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        vb.linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        vb.gated_ffn(x, w, w, w.t())
    with pytest.raises(RuntimeError, match="CUDA"):
        vb.grad_norm([x])
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        vb.clip_grad_norm_(p, 1.0)


def test_arguments_are_checked_before_the_device():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(ValueError):
        vb.linear(x, w, activation="tanh")
    with pytest.raises(ValueError):
        vb.gated_ffn(x, w, w, w.t(), activation="none")
    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            vb.clip_grad_norm_([p], bad)
    with pytest.raises(ValueError):
        vb.clip_grad_norm_([p], 1.0, norm_type=3)
    with pytest.raises(TypeError):
        vb.grad_norm([1.0])
    with pytest.raises(TypeError):
        vb.grad_norm([torch.sparse_coo_tensor([[0]], [1.0], (3,))])


def test_nothing_to_clip():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(vb.clip_grad_norm_([p], 1.0)) == 0.0
    assert float(vb.grad_norm([])) == 0.0


def test_null_arguments():
    lib = _lib.load()
    n = ctypes.c_size_t()
    bad = _lib.VMOE_ERR_INVALID_ARG
    assert lib.vmoe_ops_create(0, None) == bad
    assert lib.vmoe_ops_destroy(None) == bad
    assert lib.vmoe_ops_device_status(None, None, None) == bad
    assert lib.vmoe_ops_last_error(None) == b""
    d, f = _lib.VmoeLinear(), _lib.VmoeGatedFfn()
    assert lib.vmoe_linear_workspace_size(None, d, 0, n) == bad
    assert lib.vmoe_linear_forward(None, d, None, None, None, None, None, None, None, 0, None) == bad
    assert lib.vmoe_linear_backward(None, d, None, None, None, None, 0, None, None, None, None, 0,
                                    None) == bad
    assert lib.vmoe_gated_ffn_workspace_size(None, f, 0, n, None) == bad
    w, g = _lib.VmoeFfnWeights(), _lib.VmoeFfnGrads()
    assert lib.vmoe_gated_ffn_forward(None, f, None, w, None, None, None, 0, None, 0, None) == bad
    assert lib.vmoe_gated_ffn_backward(None, f, None, w, None, 0, None, g, None, 0, None, 0,
                                       None) == bad
    assert lib.vmoe_grad_norm_workspace_size(None, 0, n) == bad
    assert lib.vmoe_grad_norm(None, None, None, None, 0, 2, 1.0, None, None, 0, None) == bad


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU error path")
def test_context_without_gpu_is_a_clean_error():
    h = ctypes.c_void_p()
    assert _lib.load().vmoe_ops_create(0, ctypes.byref(h)) == _lib.VMOE_ERR_CUDA and not h.value
    with pytest.raises(_lib.VmoeError):
        _lib.Ops(0)
