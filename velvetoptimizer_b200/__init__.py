"""B200-native (sm_100a) Mixture-of-Experts FFN forward for VelvetOptimizer.

Public surface:
  * ``MoELayer`` — drop-in for the reference ``vesper.model.MoELayer``;
  * ``FeedForward`` — drop-in for the reference dense ``vesper.model.FeedForward``;
  * ``MoEConfig`` — the MoE knobs of ``VesperConfig``;
  * ``linear``, ``gated_ffn`` — the dense operators with their gradients (dense.py);
  * ``device_status`` — whether one of their kernels gave up a bounded wait;
  * ``clip_grad_norm_``, ``grad_norm`` — the global gradient norm and clipping (grads.py);
  * ``torch.ops.vesper_moe.forward`` — the custom op over the C ABI (include/vesper_moe.h).
"""
from .config import MoEConfig
from .dense import device_status, gated_ffn, linear
from .grads import clip_grad_norm_, grad_norm
from .moe import ExpertFFN, FeedForward, FlyLoRALinear, MoELayer

__all__ = ["MoEConfig", "MoELayer", "FeedForward", "ExpertFFN", "FlyLoRALinear",
           "linear", "gated_ffn", "device_status", "clip_grad_norm_", "grad_norm"]
