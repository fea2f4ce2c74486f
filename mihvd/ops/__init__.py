"""Hand-written CDNA4 (gfx950) HIP kernels, registered as ``torch.ops.mihvd``.

``load()`` loads ``mihvd/_native/libmihvd_kernels.so`` (built in-tree by ``python -m mihvd._build``)
and raises if it is unavailable. Kernels of the MNIST hot path: conv1_fwd, conv2_fwd, fc1_fwd,
head_fwd_bwd, fc1_wgrad, fc1_dgrad, conv2_bwd (+ fused conv1 wgrad), conv2_wgrad_reduce, adam_step,
scale_cast_bf16, bf16_to_f32, segment_dots, adasum_combine, grad_check_, update_scale_; of a
transformer's training step: linear_cross_entropy and gated_ffn with their gradients, newton_schulz
and muon_step behind ``mihvd.optim.orthogonalize`` and ``Muon`` (csrc/kernels/*.hip).
"""
from .. import _native
from .transformer import gated_ffn, linear_cross_entropy  # noqa: F401


def load():
    _native.require_kernels()
    import torch

    return torch.ops.mihvd


def available() -> bool:
    return _native.load_kernels()
