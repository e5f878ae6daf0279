"""Token embeddings: a table of vectors looked up by number, for models that read discrete tokens (visual tokens, class or text labels)
next to patches.  The reference's models read images only and have no counterpart; the table follows this package's conventions - fp32
masters, bf16 activations, kernels behind ops.py as the only implementation."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import ops
from ._lib import VitkError


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, out_dtype):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.wtype, ctx.scale, ctx.padding_idx = weight.shape[0], weight.dtype, scale, padding_idx
        return ops.embedding_fwd(ids, weight.detach(), scale=scale, out_dtype=out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        grad = ops.embedding_bwd(dout, ids, ctx.rows, scale=ctx.scale, padding_idx=ctx.padding_idx, out_dtype=ctx.wtype)
        return grad, None, None, None, None


def embedding(ids, weight, scale: float = 1.0, padding_idx=None, out_dtype=torch.bfloat16):
    """scale * weight[ids] in out_dtype (bf16 or fp32), differentiable in weight (fp32 or bf16 [V, D], D a multiple of 8); the gradient is summed
    in an order that the ids alone decide, so a step gives the same bits on every run.  Tokens with id padding_idx (negative: counted from the
    end) get their row and give no gradient.  An id outside the table gives a row of NaN."""
    if padding_idx is not None:
        V = weight.shape[0]
        if not -V <= padding_idx < V:
            raise VitkError(f"embedding: padding_idx {padding_idx} outside the table of {V} rows")
        padding_idx = int(padding_idx) % V
    return _Embedding.apply(weight, ids, float(scale), padding_idx, out_dtype)


class TokenEmbedding(nn.Module):
    """A table of num_embeddings vectors of width embedding_dim (fp32 masters, truncated normal with deviation 0.02 like the position table;
    the padding row starts at zero)."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx=None, out_dtype=torch.bfloat16):
        super().__init__()
        if num_embeddings < 1 or embedding_dim < 8 or embedding_dim % 8:
            raise VitkError(f"TokenEmbedding: embedding_dim must be a multiple of 8, num_embeddings positive, got {num_embeddings}, {embedding_dim}")
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise VitkError(f"TokenEmbedding: padding_idx {padding_idx} outside the table of {num_embeddings} rows")
        self.scale, self.padding_idx, self.out_dtype = float(scale), padding_idx, out_dtype
        self.weight = nn.Parameter(torch.empty(num_embeddings, embedding_dim))
        nn.init.trunc_normal_(self.weight, std=0.02)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx, self.out_dtype)
