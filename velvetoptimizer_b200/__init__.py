"""B200-native (sm_100a) Mixture-of-Experts FFN forward for VelvetOptimizer.

Public surface:
  * ``MoELayer`` — drop-in for the reference ``vesper.model.MoELayer``;
  * ``FeedForward`` — drop-in for the reference dense ``vesper.model.FeedForward``;
  * ``MoEConfig`` — the MoE knobs of ``VesperConfig``;
  * ``linear``, ``gated_ffn`` — the dense operators with their gradients (dense.py);
  * ``clip_grad_norm_``, ``grad_norm`` — the global gradient norm and clipping (grads.py);
  * ``torch.ops.vesper_moe.forward`` — the custom op over the C ABI (include/vesper_moe.h).
"""
from .config import MoEConfig
from .dense import gated_ffn, linear
from .grads import clip_grad_norm_, grad_norm
from .moe import ExpertFFN, FeedForward, FlyLoRALinear, MoELayer

__all__ = ["MoEConfig", "MoELayer", "FeedForward", "ExpertFFN", "FlyLoRALinear",
           "linear", "gated_ffn", "clip_grad_norm_", "grad_norm"]
