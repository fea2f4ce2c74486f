"""Entry points of the transformer-step kernels (``torch.ops.mihvd.linear_cross_entropy / gated_ffn``, whose
autograd formulas are registered beside them in csrc/kernels/transformer_ops.cpp).

* ``linear_cross_entropy(hidden, weight, labels, bias)`` — the vocabulary projection and its softmax
  cross entropy without materialised logits (csrc/kernels/linear_ce.hip).
* ``gated_ffn(x, w_gate, w_up, w_down)`` — ``(act(x Wg^T) * (x Wu^T)) Wd^T`` with its backward pass
  (csrc/kernels/gated_ffn.hip).

Both run on bf16 or fp16 MFMA operands with fp32 accumulation. Under ``torch.autocast`` fp32, bf16 and
fp16 inputs are cast to the autocast type first, as for ``torch.nn.functional.linear``; otherwise the
inputs must be 16-bit themselves. There is no CPU, fp32 or fp64 form: other inputs raise. Gradients are
reverse-mode and of first order: forward-mode derivatives, gradients of gradients and ``torch.func``'s
gradient transforms raise. Traced (fake tensors, ``torch.compile``), each is one node forward and one
backward.
"""
from __future__ import annotations

import torch

from .. import _native

ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
_ACTIVATION = {name: i for i, name in enumerate(ACTIVATIONS)}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


_ops = {}


def _op(name):
    op = _ops.get(name)
    if op is None:
        _native.require_kernels()
        op = _ops[name] = getattr(torch.ops.mihvd, name).default
    return op


def _on_gpu(op, *tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("%s: every tensor must be on the GPU (got one on %s)" % (op, t.device))


def _autocast(*tensors):
    """Autocast's cast of the floating matrices of a call. Like autocast it leaves float64 alone."""
    dt = torch.get_autocast_dtype("cuda")
    return [t if t is None or t.dtype in (dt, torch.float64) or not t.is_floating_point() else t.to(dt) for t in tensors]


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         bias: torch.Tensor | None = None, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(hidden @ weight.T + bias, labels, ...)`` without keeping the logits.

    ``hidden`` [..., K] and ``weight`` [V, K] in bf16 or fp16 (any strides), ``bias`` [V] in fp32 or
    the same type, ``labels`` [...] int64. The loss is fp32: a scalar for ``reduction="mean"`` (over
    the labelled rows; NaN if there is none) and ``"sum"``, of ``labels``' shape for ``"none"`` (0 where
    the label is ``ignore_index``). Gradients come in the types of their inputs; rows that are ignored
    get exact zeros. A label outside [0, V) that is not ``ignore_index`` makes its row's loss NaN, and
    with it the gradients.

    Ignored rows are dropped before the products, so a head over all positions of a masked-LM batch
    costs what its labelled positions cost. The call never synchronises with the host and can be
    captured in a HIP graph; results repeat bit for bit.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError("linear_cross_entropy: reduction must be one of %s (got %r)" % (tuple(_REDUCTIONS), reduction))
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError("linear_cross_entropy: hidden [..., K] and weight [V, K] are needed (got %s and %s)"
                         % (tuple(hidden.shape), tuple(weight.shape)))
    if labels.shape != hidden.shape[:-1]:
        raise ValueError("linear_cross_entropy: labels must have the shape %s (got %s)"
                         % (tuple(hidden.shape[:-1]), tuple(labels.shape)))
    if labels.dtype != torch.int64:
        raise TypeError("linear_cross_entropy: labels must be int64 (got %s)" % labels.dtype)
    _on_gpu("linear_cross_entropy", hidden, weight, labels, bias)
    if torch.is_autocast_enabled("cuda"):
        if bias is None or bias.dtype == torch.float32:
            hidden, weight = _autocast(hidden, weight)
        else:
            hidden, weight, bias = _autocast(hidden, weight, bias)
    if hidden.dim() != 2:
        hidden = hidden.reshape(-1, hidden.shape[-1])
    flat = labels if labels.dim() == 1 else labels.reshape(-1)
    loss = _op("linear_cross_entropy")(hidden, weight, flat, bias, ignore_index, _REDUCTIONS[reduction])
    return loss.view(labels.shape) if reduction == "none" and labels.dim() != 1 else loss


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``: ``x`` [..., K], ``w_gate`` and ``w_up`` [F, K],
    ``w_down`` [K, F], all bf16 or all fp16, any strides; the result has ``x``'s shape and type.

    ``activation``: "silu" (SwiGLU), "gelu" (GeGLU, the erf form), "gelu_tanh", "relu" or "sigmoid". For
    the backward pass the two projections and their product are kept in 16 bits ([rows, F] each);
    without gradients only the product is written. From one row up; results repeat bit for bit and
    the call can be captured in a HIP graph.
    """
    if activation not in _ACTIVATION:
        raise ValueError("gated_ffn: activation must be one of %s (got %r)" % (ACTIVATIONS, activation))
    k = x.shape[-1] if x.dim() else 0
    if w_gate.dim() != 2 or w_gate.shape[1] != k or w_up.shape != w_gate.shape or w_down.shape != (k, w_gate.shape[0]) or \
            0 in w_gate.shape:
        raise ValueError("gated_ffn: x [..., K], w_gate and w_up [F, K] and w_down [K, F] are needed (got %s, %s, %s, %s)"
                         % tuple(tuple(t.shape) for t in (x, w_gate, w_up, w_down)))
    _on_gpu("gated_ffn", x, w_gate, w_up, w_down)
    if torch.is_autocast_enabled("cuda"):
        x, w_gate, w_up, w_down = _autocast(x, w_gate, w_up, w_down)
    if x.dim() == 2:
        return _op("gated_ffn")(x, w_gate, w_up, w_down, _ACTIVATION[activation])
    return _op("gated_ffn")(x.reshape(-1, k), w_gate, w_up, w_down, _ACTIVATION[activation]).view(x.shape)
