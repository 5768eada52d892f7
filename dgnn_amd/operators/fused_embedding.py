"""Autograd operator of the node-id embedding (new API surface: the reference looks nothing up)."""
import torch

from ..native import fused_embedding
from ._autograd import differentiated


def NodeEmbeddingFuse(ids, table, scale=1.0):
    """scale * table[ids] as one kernel; [*ids.shape, dim] in table's type.

    ids (int32 or int64, any shape) outside [0, rows) -- padding -- give rows of zeros and no gradient.
    table is [rows, dim], float32, bfloat16 or float16.  Its gradient is dense, summed in float32
    in the order of the ids (sorted, no atomics: the same bits every time)."""
    if not differentiated(table):        # a lookup alone: no graph to build
        return fused_embedding.embedding_forward(ids.contiguous(), table.detach().contiguous(), scale)
    return NodeEmbeddingFunction.apply(ids, table, scale)


class NodeEmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        ids = ids.contiguous()
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.size(0), scale
        return fused_embedding.embedding_forward(ids, table.contiguous(), scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        ids, = ctx.saved_tensors
        return None, fused_embedding.embedding_backward(ids, grad_out.contiguous(), ctx.rows, ctx.scale), None
