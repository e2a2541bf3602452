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


def elements(t):
    """Byte offsets of a tensor's elements."""
    at = [t.data_ptr()]
    for n, s in zip(t.shape, t.stride()):
        at = [a + i * s * t.element_size() for a in at for i in range(n)]
    return {a + k for a in at for k in range(t.element_size())}


def test_shared_memory_is_found_exactly():
    """The overlap check of gradients that are not dense against sets of addresses."""
    import random

    from velvetoptimizer_b200.lib import _dense_ops
    rng = random.Random(0)
    buf = torch.zeros(4096)
    seen = [0, 0]
    for _ in range(4000):
        two = []
        for _ in range(2):
            dims = rng.randint(1, 3)
            shape = [rng.randint(1, 5) for _ in range(dims)]
            stride = [rng.choice((0, 1, 2, 3, 4, 5, 8, 12, 20)) for _ in range(dims)]
            t = torch.as_strided(buf, shape, stride, rng.randint(0, 40))
            two.append(t.view(torch.bfloat16)[..., 1:] if stride[-1] == 1 and rng.random() < 0.3 else t)
        a, b = two
        want = bool(elements(a) & elements(b))
        assert _dense_ops.share_memory(a, b) == want, (a.shape, a.stride(), b.shape, b.stride())
        seen[want] += 1
    assert min(seen) > 500
    wide = torch.zeros(1000, 64)
    assert not _dense_ops.share_memory(wide[:, :10], wide[:, 10:30])
    assert _dense_ops.share_memory(wide[:, :11], wide[:, 10:30])
    assert not _dense_ops.share_memory(wide[::2], wide[1::2])
    assert _dense_ops.share_memory(wide[::2], wide[998:])


def test_tangents_are_refused_before_the_device():
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        t = fwd.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(NotImplementedError, match="tangent"):
            vb.grad_norm([t])


def test_the_eager_path_gives_way_to_tracers():
    """Tracers and dispatch modes get the registered ops; tensors with a dispatch of their own, in
    any place, do too."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    from velvetoptimizer_b200.lib._dense_ops import eager
    t = torch.ones(2)
    assert eager(t, torch.nn.Parameter(t))
    seen = []

    def fn(x):
        seen.append(eager(t, t))
        return x + 1

    make_fx(fn)(t)
    make_fx(fn, pre_dispatch=True)(t)
    make_fx(fn, tracing_mode="fake")(t)
    torch.jit.trace(fn, t, check_trace=False)

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Mode():
        fn(t)
    assert seen == [False] * 5 and eager(t, t)
    fake = FakeTensorMode().from_tensor(t)
    assert not eager(t, fake) and not eager(fake, t)
    for trace in (lambda f: make_fx(f)(t), lambda f: make_fx(f, pre_dispatch=True)(t),
                  lambda f: torch.jit.trace(f, t, check_trace=False)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace(lambda x: vb.grad_norm([x]))


def test_device_status_wants_a_cuda_device():
    for bad in ("cpu", torch.device("cpu")):
        with pytest.raises(ValueError, match="CUDA"):
            vb.device_status(bad)


def test_what_is_no_tensor_is_refused():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    for bad in ([1.0], 2.0, "x"):
        with pytest.raises(TypeError):
            vb.linear(bad, w)
        with pytest.raises(TypeError):
            vb.linear(x, w, bad)
        with pytest.raises(TypeError):
            vb.gated_ffn(x, w, bad, w.t())
    with pytest.raises(TypeError):
        vb.linear(None, w)
    with pytest.raises(TypeError):
        vb.linear(x, None)
    with pytest.raises(TypeError):
        vb.linear(x, w, activation="silu", gamma="a")
