"""Autograd operator of packed attention (new API surface: the reference's attention runs over given
edges, dgNN/operators/fused_gatconv.py; this one over all pairs of a graph, a walk or a prompt)."""
import torch

from ..native import fused_attention
from ._autograd import differentiated


def PackedAttentionFuse(q, k, v, row_ptr, col_ptr=None, causal=False, scale=None):
    """softmax(scale q k^T) v inside every sequence of a packed batch; [rows, heads, dim] in q's type.

    q [rows, heads, dim], k and v [keys, key_heads, dim], float32, bfloat16 or float16, dim 1 to 128;
    key_heads divides heads, query head i reads key head i // (heads // key_heads).  Views with
    strides (slices of one projection's output) are read where they lie if their rows are whole
    16-byte chunks, otherwise copied once.
    row_ptr (int32, sequences + 1 ascending offsets) bounds the rows of every sequence, col_ptr (default:
    row_ptr) its keys: one row a sequence and all of its nodes as keys is an attention pooling, or
    the step of a single token.  causal: row i of a sequence sees its keys j <= i + keys - rows.
    scale defaults to dim ** -0.5.

    A row that sees no key (masked, empty sequence, in front of or behind the sequences) gives zeros and no
    gradient, whatever it and the keys hold.  Values do not cross sequences, not even NaN; inside one, a NaN or
    infinity in a key or value may reach rows that the causal mask keeps from it (and one in a row or its
    gradient the gradients of keys that it does not see), as a weight of zero times it does."""
    if scale is None:
        scale = max(q.size(-1), 1) ** -0.5                # (a dim of 0 is refused below)
    if col_ptr is None:
        col_ptr = row_ptr
    if not differentiated(q, k, v):
        return fused_attention.attention_forward(q, k, v, row_ptr, col_ptr, scale, causal)[0]
    return PackedAttentionFunction.apply(q, k, v, row_ptr, col_ptr, causal, scale)


class PackedAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, row_ptr, col_ptr, causal, scale):
        # rest: what rounding took from a 16-bit out (None for float32); the backward's <grad, out> needs it
        out, lse, rest = fused_attention.attention_forward(q, k, v, row_ptr, col_ptr, scale, causal, rest=True)
        ctx.save_for_backward(q, k, v, row_ptr, col_ptr, out, lse, rest)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, v, row_ptr, col_ptr, out, lse, rest = ctx.saved_tensors
        dq, dk, dv = fused_attention.attention_backward(q, k, v, row_ptr, col_ptr, ctx.scale, ctx.causal, out, lse,
                                                        grad_out, out_rest=rest)
        return dq, dk, dv, None, None, None, None
