"""Dense training operators over weights the caller keeps: ``linear`` and ``gated_ffn``.

``linear`` is ``residual + act(x W^T + b)`` in one kernel, with its gradients; ``gated_ffn`` is
the reference's dense feed-forward block (python/vesper/model.py:249-270) with its gradients.
Both read the weights where they are, in ``nn.Linear``'s layout: nothing is packed or kept
between calls, so weights that change every step need no repacking.  They run on torch's
current stream of x's device through the C ABI (``vmoe_linear_*``, ``vmoe_gated_ffn_*``).
bfloat16 runs on the tensor cores; float32 does too, as six bfloat16 products, except for up to 16
rows in a forward and for sums that are not finite, which take the CUDA cores.  Everything
accumulates in fp32.  They need an sm_100 GPU; there is no CPU path.

Parameters may have another floating type than x (fp32 masters of a bf16 step): they are cast
to x's type for the call, and their gradients come back in their own type, from fp32 sums.
"""
from __future__ import annotations

import threading

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3, "era": 4}
_DTYPES = {torch.float32: _lib.VMOE_F32, torch.bfloat16: _lib.VMOE_BF16}
_local = threading.local()


def ops_for(device: torch.device) -> _lib.Ops:
    """The calling thread's ``vmoe_ops`` context on ``device``."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    contexts = _local.__dict__
    o = contexts.get(index)
    if o is None:
        o = contexts[index] = _lib.Ops(index)
    return o


def device_status(device: torch.device | int | str | None = None) -> int:
    """Whether a kernel of ``linear``, ``gated_ffn`` or their gradients on ``device`` (the current
    one), launched from any thread, gave up a bounded wait since the last call: raises
    ``VmoeError`` if so, and clears it.  Waits for the device's current stream.  Returns 0."""
    if not isinstance(device, torch.device):
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device or "cuda")
    if device.type != "cuda":
        raise ValueError(f"device_status: {device} is not a CUDA device")
    return ops_for(device).device_status(torch.cuda.current_stream(device).cuda_stream)


def _native():
    """The host module of the eager path (csrc_py/dense_ops.cpp, built beside the library)."""
    global _module
    if _module is None:
        _lib.load()
        from .lib import _dense_ops
        _module = _dense_ops
    return _module


_module = None


_PLAIN = (torch.Tensor, torch.nn.Parameter)


# ------------------------------------------------------------------------------ the kernels
def _linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                    residual: torch.Tensor | None, activation: int, gamma: float,
                    keep: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(y [T, N], z [T, N] or empty) for x [T, K]."""
    return _native().linear_forward(x, weight, bias, residual, activation, gamma, keep)


def _linear_backward(x: torch.Tensor, weight: torch.Tensor, z: torch.Tensor, dy: torch.Tensor,
                     activation: int, gamma: float, want: list[bool],
                     grad_f32: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dW, db), empty where not wanted."""
    return _native().linear_backward(x, weight, z, dy, activation, gamma, want, grad_f32)


def _gated_ffn_forward(x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor,
                       down_w: torch.Tensor, gate_b: torch.Tensor | None,
                       up_b: torch.Tensor | None, down_b: torch.Tensor | None,
                       residual: torch.Tensor | None, activation: int, gamma: float,
                       keep: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(y [T, H], what the backward reads, as bytes, or empty) for x [T, H]."""
    return _native().gated_ffn_forward(x, gate_w, up_w, down_w, gate_b, up_b, down_b, residual,
                                       activation, gamma, keep)


def _gated_ffn_backward(x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor,
                        down_w: torch.Tensor, saved: torch.Tensor, dy: torch.Tensor,
                        activation: int, gamma: float, want: list[bool], grad_f32: bool) -> tuple[
                            torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                            torch.Tensor, torch.Tensor]:
    """(dx, dWg, dWu, dWd, dbg, dbu, dbd), empty where not wanted."""
    return _native().gated_ffn_backward(x, gate_w, up_w, down_w, saved, dy, activation, gamma, want,
                                        grad_f32)


# Registered as custom ops for the tracers (torch.compile, export); an eager call goes through
# the native module's own autograd node.
_custom = lambda name, fn: torch.library.custom_op(  # noqa: E731
    f"vesper_moe::{name}", mutates_args=(), device_types="cuda")(fn)
linear_forward_op = _custom("linear_forward", _linear_forward)
linear_backward_op = _custom("linear_backward", _linear_backward)
gated_ffn_forward_op = _custom("gated_ffn_forward", _gated_ffn_forward)
gated_ffn_backward_op = _custom("gated_ffn_backward", _gated_ffn_backward)


@linear_forward_op.register_fake
def _(x, weight, bias, residual, activation, gamma, keep):
    y = x.new_empty((x.shape[0], weight.shape[0]))
    return y, (torch.empty_like(y) if keep else x.new_empty((0,)))


@linear_backward_op.register_fake
def _(x, weight, z, dy, activation, gamma, want, grad_f32):
    gt = torch.float32 if grad_f32 else x.dtype
    N = weight.shape[0]
    return (x.new_empty(x.shape if want[0] else (0,)),
            x.new_empty((N, x.shape[1]) if want[1] else (0,), dtype=gt),
            x.new_empty((N,) if want[2] else (0,), dtype=gt))


@gated_ffn_forward_op.register_fake
def _(x, gate_w, up_w, down_w, gate_b, up_b, down_b, residual, activation, gamma, keep):
    T, I = x.shape[0], gate_w.shape[0]
    n = T * ((I + 7) // 8 * 8)  # g and u in fp32, h
    size = 2 * ((4 * n + 255) // 256 * 256) + (n * x.element_size() + 255) // 256 * 256
    return x.new_empty(x.shape), x.new_empty((size if keep else 0,), dtype=torch.uint8)


@gated_ffn_backward_op.register_fake
def _(x, gate_w, up_w, down_w, saved, dy, activation, gamma, want, grad_f32):
    gt = torch.float32 if grad_f32 else x.dtype
    H, I = x.shape[1], gate_w.shape[0]
    shapes = (x.shape, (I, H), (I, H), (H, I), (I,), (I,), (H,))
    return tuple(x.new_empty(s if on else (0,), dtype=x.dtype if i == 0 else gt)
                 for i, (s, on) in enumerate(zip(shapes, want)))


# ------------------------------------------------------------------------------ autograd (traced)
def _as(g: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return g if g.dtype == like.dtype else g.to(like.dtype)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, gamma):
        run = torch.ops.vesper_moe.linear_forward
        w = weight.to(x.dtype)
        b = None if bias is None else bias.to(x.dtype)
        keep = activation != 0 and any(ctx.needs_input_grad[:3])
        y, z = run(x, w, b, residual, activation, gamma, keep)
        ctx.save_for_backward(x, w, z)
        ctx.args = (activation, gamma)
        ctx.types = (weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            run = torch.ops.vesper_moe.linear_backward
            grad_f32 = torch.float32 in ctx.types
            dx, dw, db = run(x, w, z, dy, *ctx.args, list(need[:3]), grad_f32)
        return (dx if need[0] else None, dw.to(ctx.types[0]) if need[1] else None,
                db.to(ctx.types[1]) if need[2] else None, dy if need[3] else None, None, None)


class _GatedFfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_w, up_w, down_w, gate_b, up_b, down_b, residual, activation, gamma):
        run = torch.ops.vesper_moe.gated_ffn_forward
        params = (gate_w, up_w, down_w, gate_b, up_b, down_b)
        cast = [None if p is None else p.to(x.dtype) for p in params]
        y, saved = run(x, *cast, residual, activation, gamma, any(ctx.needs_input_grad[:7]))
        ctx.save_for_backward(x, *cast[:3], saved)
        ctx.args = (activation, gamma)
        ctx.types = [None if p is None else p.dtype for p in params]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, gate_w, up_w, down_w, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = [None] * 7
        if any(need[:7]):
            run = torch.ops.vesper_moe.gated_ffn_backward
            got = run(x, gate_w, up_w, down_w, saved, dy, *ctx.args, list(need[:7]),
                      torch.float32 in ctx.types)
            grads = [None if not on else g if i == 0 else g.to(ctx.types[i - 1])
                     for i, (g, on) in enumerate(zip(got, need))]
        return (*grads, dy if need[7] else None, None, None)


# ------------------------------------------------------------------------------ the operators
# The eager path checks the same in C++.
def _check_x(name: str, x: torch.Tensor) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: x must be a tensor, not {type(x).__name__}")
    if x.device.type != "cuda":
        raise RuntimeError(f"{name} runs on CUDA tensors only (there is no CPU path)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} supports float32 and bfloat16 inputs, not {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{name}: x must have a feature dimension")


def _check_param(name: str, label: str, p: torch.Tensor, shape: tuple, x: torch.Tensor) -> None:
    if tuple(p.shape) != shape:
        raise ValueError(f"{name}: {label} must have shape {list(shape)}, not {list(p.shape)}")
    if p.device != x.device:
        raise ValueError(f"{name}: {label} is on {p.device}, x on {x.device}")
    if p.dtype not in _DTYPES:
        raise TypeError(f"{name}: {label} must be float32 or bfloat16, not {p.dtype}")


def _check_residual(name: str, r: torch.Tensor, shape: tuple, x: torch.Tensor) -> None:
    if tuple(r.shape) != shape:
        raise ValueError(f"{name}: residual must have shape {list(shape)}, not {list(r.shape)}")
    if r.device != x.device or r.dtype != x.dtype:
        raise TypeError(f"{name}: residual must be {x.dtype} on {x.device}, as x is")


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           residual: torch.Tensor | None = None, activation: str = "none",
           gamma: float = 0.1) -> torch.Tensor:
    """``residual + act(x @ weight.T + bias)``, rounded once, with gradients to all four tensors.

    x ``[..., K]`` (float32 or bfloat16, any strides), weight ``[N, K]``, bias ``[N]``, residual
    ``[..., N]`` of x's type; ``activation`` is one of ``none``, ``relu``, ``silu``,
    ``gelu_tanh`` and ``era`` (``gelu_tanh + gamma * softplus``, python/vesper/model.py:69-76).
    A training call of an activation keeps the pre-activations in x's type.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: activation must be one of {', '.join(ACTIVATIONS)}, "
                         f"not {activation!r}")
    if type(x) in _PLAIN and not torch.compiler.is_compiling():
        y = _native().linear(x, weight, bias, residual, ACTIVATIONS[activation], gamma)
        if y is not None:  # None: a tracer, a dispatch mode or a subclass wants the registered op
            return y
    _check_x("linear", x)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError(f"linear: weight must be [N, {x.shape[-1]}] with N and K at least 1, "
                         f"not {list(weight.shape)}")
    N, K = weight.shape
    _check_param("linear", "weight", weight, (N, K), x)
    if bias is not None:
        _check_param("linear", "bias", bias, (N,), x)
    shape = (*x.shape[:-1], N)
    r2d = None
    if residual is not None:
        _check_residual("linear", residual, shape, x)
        r2d = residual.reshape(-1, N)
    args = (x.reshape(-1, K), weight, bias, r2d)
    act, gamma = ACTIVATIONS[activation], float(gamma)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return _LinearFn.apply(*args, act, gamma).reshape(shape)
    run = torch.ops.vesper_moe.linear_forward
    cast = [None if t is None else _as(t, x) for t in args]
    return run(*cast, act, gamma, False)[0].reshape(shape)


def gated_ffn(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor,
              down_weight: torch.Tensor, gate_bias: torch.Tensor | None = None,
              up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None, *,
              residual: torch.Tensor | None = None, activation: str = "era",
              gamma: float = 0.1) -> torch.Tensor:
    """The gated feed-forward block, with gradients to every tensor:

    ``residual + (act(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)) @
    down_weight.T + down_bias``.

    x and residual ``[..., H]`` (float32 or bfloat16, any strides), gate and up weights
    ``[I, H]``, down weight ``[H, I]``; ``activation`` as for ``linear``, except ``none``.
    """
    if activation == "none" or activation not in ACTIVATIONS:
        raise ValueError(f"gated_ffn: activation must be one of {', '.join(ACTIVATIONS)} but none, "
                         f"not {activation!r}")
    if type(x) in _PLAIN and not torch.compiler.is_compiling():
        y = _native().gated_ffn(x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias,
                                residual, ACTIVATIONS[activation], gamma)
        if y is not None:  # None: a tracer, a dispatch mode or a subclass wants the registered op
            return y
    _check_x("gated_ffn", x)
    H = x.shape[-1]
    if gate_weight.dim() != 2 or gate_weight.shape[1] != H or 0 in gate_weight.shape:
        raise ValueError(f"gated_ffn: gate_weight must be [I, {H}] with I and H at least 1, "
                         f"not {list(gate_weight.shape)}")
    I = gate_weight.shape[0]
    params = (gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias)
    shapes = ((I, H), (I, H), (H, I), (I,), (I,), (H,))
    labels = ("gate_weight", "up_weight", "down_weight", "gate_bias", "up_bias", "down_bias")
    for p, s, n in zip(params, shapes, labels):
        if p is not None:
            _check_param("gated_ffn", n, p, s, x)
    r2d = None
    if residual is not None:
        _check_residual("gated_ffn", residual, tuple(x.shape), x)
        r2d = residual.reshape(-1, H)
    args = (x.reshape(-1, H), *params, r2d)
    act, gamma = ACTIVATIONS[activation], float(gamma)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return _GatedFfnFn.apply(*args, act, gamma).reshape(x.shape)
    run = torch.ops.vesper_moe.gated_ffn_forward
    cast = [None if t is None else _as(t, x) for t in args]
    return run(*cast, act, gamma, False)[0].reshape(x.shape)
