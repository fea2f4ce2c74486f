"""BERT-base encoder + masked-LM head for the "BERT-base synthetic seq=512 on 8×MI355X (large-grad
fusion + fp16 allreduce compression)" stress configuration: 110 M parameters,
440 MB of fp32 gradients per step, one embedding matrix of 94 MB — a fusion-buffer and
compression stress test of the DP engine.

Built from stock PyTorch-ROCm ops (``scaled_dot_product_attention``, hipBLASLt GEMMs) under bf16
autocast; ``BertConfig.ffn_impl`` and ``loss_impl`` choose the framework's own gated feed-forward block
and vocabulary loss (mihvd.ops). Not part of the reference repo (whose only model is the MNIST CNN).
"""
from __future__ import annotations

import dataclasses
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import gated_ffn, linear_cross_entropy


@dataclasses.dataclass
class BertConfig:
    vocab_size: int = 30522
    hidden: int = 768
    layers: int = 12
    heads: int = 12
    ffn: int = 3072
    max_len: int = 512
    type_vocab: int = 2
    dropout: float = 0.1
    attn_dropout: float | None = None  # attention-probability dropout (None: ``dropout``)
    attn_impl: str = "sdpa"  # "sdpa" (F.scaled_dot_product_attention) | "math" (matmul/softmax ops)
    eps: float = 1e-12
    # "gather": lookups as index_select, whose backward is a scatter-add (index_add_); "embedding":
    # F.embedding, whose backward sorts the ids and segments them with rocprim's unique_by_key —
    # that partition kernel faults (memory aperture violation) when a whole BERT step is replayed
    # from a HIP graph on this ROCm build with MLM data (many repeated [MASK] ids)
    embedding_impl: str = "gather"
    # "gelu": fc2(gelu(fc1(x))); "geglu" / "swiglu": the gated block fc_down(act(fc_gate(x)) * fc_up(x)) with
    # ``ffn`` columns and no biases, on the GPU through mihvd.ops.gated_ffn (16-bit: under autocast, or
    # a model in bf16 / fp16)
    ffn_impl: str = "gelu"
    # "torch": logits and F.cross_entropy; "fused": mihvd.ops.linear_cross_entropy on the GPU (16-bit, as
    # above), which keeps no logits and skips the positions without a label
    loss_impl: str = "torch"


class BertLayer(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.c = c
        self.qkv = nn.Linear(c.hidden, 3 * c.hidden)
        self.proj = nn.Linear(c.hidden, c.hidden)
        self.ln1 = nn.LayerNorm(c.hidden, eps=c.eps)
        if c.ffn_impl == "gelu":
            self.fc1 = nn.Linear(c.hidden, c.ffn)
            self.fc2 = nn.Linear(c.ffn, c.hidden)
        elif c.ffn_impl in ("geglu", "swiglu"):
            self.fc_gate = nn.Linear(c.hidden, c.ffn, bias=False)
            self.fc_up = nn.Linear(c.hidden, c.ffn, bias=False)
            self.fc_down = nn.Linear(c.ffn, c.hidden, bias=False)
        else:
            raise ValueError("BertConfig.ffn_impl must be 'gelu', 'geglu' or 'swiglu' (got %r)" % (c.ffn_impl,))
        self.ln2 = nn.LayerNorm(c.hidden, eps=c.eps)
        self.drop = nn.Dropout(c.dropout)

    def _attn_p(self):
        return self.c.dropout if self.c.attn_dropout is None else self.c.attn_dropout

    def _ffn(self, x):
        if self.c.ffn_impl == "gelu":
            return self.fc2(F.gelu(self.fc1(x)))
        act = "gelu" if self.c.ffn_impl == "geglu" else "silu"
        if x.is_cuda:
            return gated_ffn(x, self.fc_gate.weight, self.fc_up.weight, self.fc_down.weight, activation=act)
        return self.fc_down((F.gelu if act == "gelu" else F.silu)(self.fc_gate(x)) * self.fc_up(x))

    def forward(self, x, mask=None):
        B, S, H = x.shape
        nh = self.c.heads
        q, k, v = self.qkv(x).view(B, S, 3, nh, H // nh).permute(2, 0, 3, 1, 4)
        p = self._attn_p() if self.training else 0.0
        if self.c.attn_impl == "math":
            w = (q @ k.transpose(-2, -1)) * (1.0 / math.sqrt(q.size(-1)))
            if mask is not None:
                w = w + mask
            a = F.dropout(w.softmax(-1), p=p, training=p > 0) @ v
        else:
            a = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, dropout_p=p)
        a = a.transpose(1, 2).reshape(B, S, H)
        x = self.ln1(x + self.drop(self.proj(a)))  # post-LN, as in BERT
        return self.ln2(x + self.drop(self._ffn(x)))


class BertForMaskedLM(nn.Module):
    def __init__(self, c: BertConfig | None = None):
        super().__init__()
        c = c or BertConfig()
        if c.loss_impl not in ("torch", "fused"):
            raise ValueError("BertConfig.loss_impl must be 'torch' or 'fused' (got %r)" % (c.loss_impl,))
        self.c = c
        self.tok = nn.Embedding(c.vocab_size, c.hidden)
        self.pos = nn.Embedding(c.max_len, c.hidden)
        self.typ = nn.Embedding(c.type_vocab, c.hidden)
        self.ln = nn.LayerNorm(c.hidden, eps=c.eps)
        self.drop = nn.Dropout(c.dropout)
        self.layers = nn.ModuleList([BertLayer(c) for _ in range(c.layers)])
        self.head_dense = nn.Linear(c.hidden, c.hidden)
        self.head_ln = nn.LayerNorm(c.hidden, eps=c.eps)
        self.head_bias = nn.Parameter(torch.zeros(c.vocab_size))  # decoder weight tied to self.tok
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def _lookup(self, emb: nn.Embedding, ids: torch.Tensor) -> torch.Tensor:
        if self.c.embedding_impl == "embedding":
            return emb(ids)
        return emb.weight.index_select(0, ids.reshape(-1)).view(*ids.shape, emb.weight.shape[1])

    def forward(self, ids, labels=None, masked_positions=None):
        """``masked_positions`` (flat indices into B*S, e.g. from :func:`masked_positions`): apply the
        MLM head only at those positions, as BERT pretraining implementations do — the vocabulary
        projection and its softmax then cost ~15 % of the all-position form. Fixed-size, so the step
        stays free of host synchronisation (HIP-graph capturable)."""
        B, S = ids.shape
        pos = torch.arange(S, device=ids.device)
        x = self._lookup(self.tok, ids) + self._lookup(self.pos, pos)[None] + self._lookup(self.typ, torch.zeros_like(ids))
        x = self.drop(self.ln(x))
        for layer in self.layers:
            x = layer(x)
        if masked_positions is not None:
            x = x.reshape(B * S, -1).index_select(0, masked_positions)
            if labels is not None:
                labels = labels.reshape(-1).index_select(0, masked_positions)
        h = self.head_ln(F.gelu(self.head_dense(x)))
        if labels is not None and self.c.loss_impl == "fused" and h.is_cuda:
            return linear_cross_entropy(h, self.tok.weight, labels.reshape(h.shape[:-1]), self.head_bias)
        logits = h @ self.tok.weight.t() + self.head_bias
        if labels is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.size(-1)), labels.reshape(-1), ignore_index=-100)


def muon_parameters(model: BertForMaskedLM):
    """(matrices, others): the encoder layers' weight matrices, which ``mihvd.optim.Muon`` updates, and the
    embeddings, head, norms and biases, which stay with another optimizer."""
    matrices = [p for layer in model.layers for p in layer.parameters() if p.dim() == 2]
    chosen = {id(p) for p in matrices}
    return matrices, [p for p in model.parameters() if id(p) not in chosen]


def masked_positions(labels: torch.Tensor) -> torch.Tensor:
    """Flat indices of the positions that carry an MLM label (one host sync: call once per batch
    layout, not per step)."""
    return (labels.reshape(-1) != -100).nonzero().squeeze(1)


def synthetic_mlm_batch(batch: int, seq: int, vocab: int, device, generator=None, mask_prob: float = 0.15):
    ids = torch.randint(0, vocab, (batch, seq), device=device, generator=generator)
    labels = torch.full_like(ids, -100)
    m = torch.rand(batch, seq, device=device, generator=generator) < mask_prob
    labels[m] = ids[m]
    ids = ids.masked_fill(m, 103)  # [MASK]
    return ids, labels


def flops_per_token(c: BertConfig, seq: int) -> float:
    """Training FLOPs per token (6·params for the dense parts + attention scores)."""
    mats = 2 if c.ffn_impl == "gelu" else 3
    dense = c.layers * (4 * c.hidden * c.hidden + mats * c.hidden * c.ffn) + c.hidden * c.vocab_size
    attn = c.layers * 2 * seq * c.hidden
    return 6.0 * dense + 6.0 * attn if math.isfinite(seq) else float("nan")
