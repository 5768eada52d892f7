"""What the sequence operators refuse: argument checks of the C ABI and of the Python entry points.  No
kernel is launched, so everything runs without a GPU."""
import ctypes

import pytest
import torch

from dgnn_amd import _lib
from dgnn_amd._lib import DgnnError
from dgnn_amd.operators import LinearCrossEntropyFuse, NodeEmbeddingFuse, PackedAttentionFuse

BAD_ARG, UNSUPPORTED, WORKSPACE, ALIGNMENT = -1, -2, -3, -4
P = 0x10000                      # an aligned address that is never read


def attn(dtype=1, nseq=1, tq=8, tk=8, hq=4, hk=2, d=64, q=P, k=P, v=P, strides=None, row_ptr=P, col_ptr=P, out=P,
         lse=P, rest=None, ws=P, wsb=1 << 30, null_strides=False):
    size = (hq * d, d, hk * d, d, hk * d, d) if strides is None else strides
    arr = None if null_strides else (ctypes.c_longlong * 6)(*size)
    return _lib.lib().dgnn_attn_forward(dtype, nseq, tq, tk, hq, hk, d, 0, 1.0, q, k, v, arr, row_ptr, col_ptr, out, rest, lse, ws, wsb,
                                        None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), BAD_ARG), (dict(dtype=-1), BAD_ARG), (dict(nseq=-1), BAD_ARG), (dict(tq=-1), BAD_ARG),
    (dict(hq=0), BAD_ARG), (dict(hk=3), BAD_ARG), (dict(hk=0), BAD_ARG), (dict(d=0), BAD_ARG),
    (dict(q=None), BAD_ARG), (dict(k=None), BAD_ARG), (dict(v=None), BAD_ARG), (dict(row_ptr=None), BAD_ARG),
    (dict(col_ptr=None), BAD_ARG), (dict(out=None), BAD_ARG), (dict(null_strides=True), BAD_ARG),
    (dict(d=136), UNSUPPORTED), (dict(d=12), UNSUPPORTED), (dict(dtype=0, d=6), UNSUPPORTED),
    (dict(tq=1 << 30), UNSUPPORTED),
    (dict(strides=(32, 64, 128, 64, 128, 64)), UNSUPPORTED),              # token stride under the head dim
    (dict(strides=(260, 64, 128, 64, 128, 64)), UNSUPPORTED),             # rows off 16 bytes
    (dict(strides=(256, 60, 128, 64, 128, 64)), UNSUPPORTED),
    (dict(strides=(256, 64, 0, 64, 128, 64)), UNSUPPORTED),               # expanded keys
    (dict(strides=(1 << 23, 64, 128, 64, 128, 64)), UNSUPPORTED),
    (dict(q=P + 8), ALIGNMENT), (dict(v=P + 2), ALIGNMENT), (dict(out=P + 4), ALIGNMENT), (dict(row_ptr=P + 2), ALIGNMENT),
    (dict(lse=P + 1), ALIGNMENT), (dict(rest=P + 8), ALIGNMENT),
    (dict(tk=4096, tq=2, ws=None), WORKSPACE), (dict(tk=4096, tq=2, wsb=4096), WORKSPACE),
    (dict(tk=4096, tq=2, ws=P + 4), ALIGNMENT),                           # single queries: split over the keys
])
def test_attention_forward_refuses(change, code):
    assert attn(**change) == code


def attn_bwd(dtype=1, tq=8, tk=8, hq=4, hk=2, d=64, out=P, lse=P, grad=P, dq=P, dk=P, dv=P, rest=None, ws=P, wsb=1 << 20):
    arr = (ctypes.c_longlong * 6)(hq * d, d, hk * d, d, hk * d, d)
    return _lib.lib().dgnn_attn_backward(dtype, 1, tq, tk, hq, hk, d, 0, 1.0, P, P, P, arr, P, P, out, rest, lse, grad, dq, dk,
                                         dv, ws, wsb, None)


@pytest.mark.parametrize("change,code", [
    (dict(out=None), BAD_ARG), (dict(lse=None), BAD_ARG), (dict(grad=None), BAD_ARG), (dict(dq=None), BAD_ARG),
    (dict(dk=None), BAD_ARG), (dict(dv=None), BAD_ARG), (dict(ws=None), WORKSPACE), (dict(wsb=255), WORKSPACE),
    (dict(grad=P + 8), ALIGNMENT), (dict(dk=P + 8), ALIGNMENT), (dict(ws=P + 2), ALIGNMENT), (dict(lse=P + 2), ALIGNMENT), (dict(rest=P + 4), ALIGNMENT),
    (dict(d=256), UNSUPPORTED),
])
def test_attention_backward_refuses(change, code):
    assert attn_bwd(**change) == code


def embed(dtype=0, idx=8, n=4, rows=5, dim=6, ids=P, table=P, out=P):
    return _lib.lib().dgnn_embedding_forward(dtype, idx, n, rows, dim, 1.0, ids, table, out, None)


def embed_bwd(dtype=0, idx=8, n=4, rows=5, dim=6, ids=P, grad=P, out=P, ws=P, wsb=1 << 20):
    return _lib.lib().dgnn_embedding_backward(dtype, idx, n, rows, dim, 1.0, ids, grad, out, ws, wsb, None)


@pytest.mark.parametrize("call,change,code", [
    (embed, dict(dtype=5), BAD_ARG), (embed, dict(idx=2), BAD_ARG), (embed, dict(n=-1), BAD_ARG), (embed, dict(rows=-1), BAD_ARG),
    (embed, dict(dim=-1), BAD_ARG), (embed, dict(ids=None), BAD_ARG), (embed, dict(table=None), BAD_ARG),
    (embed, dict(out=None), BAD_ARG), (embed, dict(ids=P + 4), ALIGNMENT), (embed, dict(table=P + 2), ALIGNMENT),
    (embed_bwd, dict(ids=None), BAD_ARG), (embed_bwd, dict(grad=None), BAD_ARG), (embed_bwd, dict(out=None), BAD_ARG),
    (embed_bwd, dict(ws=None), WORKSPACE), (embed_bwd, dict(wsb=100), WORKSPACE), (embed_bwd, dict(ws=P + 4), ALIGNMENT),
    (embed_bwd, dict(grad=P + 1), ALIGNMENT), (embed_bwd, dict(dtype=-1), BAD_ARG),
    (embed_bwd, dict(n=(1 << 30) + 1), UNSUPPORTED),
])
def test_embedding_refuses(call, change, code):
    assert call(**change) == code


def ce(dtype=0, lb=8, n=4, classes=5, d=6, red=1, x=P, w=P, label=P, loss=P, lse=P, ws=P, wsb=1 << 30):
    return _lib.lib().dgnn_linear_ce_forward(dtype, lb, n, classes, d, -100, red, x, w, label, loss, lse, ws, wsb, None)


def ce_bwd(dtype=0, lb=8, n=4, classes=5, d=6, red=1, x=P, w=P, label=P, lse=P, grad=P, dx=P, dw=P, ws=P, wsb=1 << 30):
    return _lib.lib().dgnn_linear_ce_backward(dtype, lb, n, classes, d, -100, red, x, w, label, lse, grad, dx, dw, ws, wsb, None)


@pytest.mark.parametrize("call", [ce, ce_bwd])
@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), BAD_ARG), (dict(lb=1), BAD_ARG), (dict(n=-1), BAD_ARG), (dict(classes=0), BAD_ARG), (dict(d=0), BAD_ARG),
    (dict(red=3), BAD_ARG), (dict(x=None), BAD_ARG), (dict(w=None), BAD_ARG), (dict(label=None), BAD_ARG),
    (dict(lse=None), BAD_ARG), (dict(ws=None), WORKSPACE), (dict(wsb=64), WORKSPACE), (dict(ws=P + 8), ALIGNMENT),
    (dict(label=P + 4), ALIGNMENT), (dict(x=P + 2), ALIGNMENT), (dict(n=(1 << 22) + 1), UNSUPPORTED),
    (dict(d=65537), UNSUPPORTED), (dict(classes=(1 << 30) + 1), UNSUPPORTED),
])
def test_cross_entropy_refuses(call, change, code):
    assert call(**change) == code


def test_workspace_sizes_are_host_functions():
    lib = _lib.lib()
    assert lib.dgnn_attn_backward_workspace_bytes(2, 100, 100, 4, 4, 64) >= 2 * 4 * 400
    assert lib.dgnn_attn_backward_workspace_bytes(2, -1, 100, 4, 4, 64) == 0
    assert lib.dgnn_embedding_backward_workspace_bytes(1000, 50, 64) >= 4 * 4000
    assert lib.dgnn_embedding_backward_workspace_bytes(0, 50, 64) == 0
    assert lib.dgnn_linear_ce_workspace_bytes(1, 100, 50, 64, 0) > 0
    assert lib.dgnn_linear_ce_workspace_bytes(1, 100, 50, 64, 1) > 0
    assert lib.dgnn_linear_ce_workspace_bytes(1, 0, 50, 64, 1) == 0
    # the backward's workspace does not hold all logits
    n, classes = 8192, 1 << 20
    assert lib.dgnn_linear_ce_workspace_bytes(1, n, classes, 64, 1) < n * classes // 4


def test_python_entry_points_refuse_cpu_tensors_and_bad_names():
    ptr = torch.tensor([0, 4], dtype=torch.int32)
    q = torch.zeros(4, 2, 8)
    with pytest.raises(DgnnError, match="GPU"):
        PackedAttentionFuse(q, q, q, ptr)
    with pytest.raises(DgnnError, match="GPU"):
        NodeEmbeddingFuse(torch.zeros(3, dtype=torch.int64), torch.zeros(5, 6))
    with pytest.raises(DgnnError, match="GPU"):
        LinearCrossEntropyFuse(torch.zeros(4, 6), torch.zeros(3, 6), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(DgnnError, match="reduction"):
        LinearCrossEntropyFuse(torch.zeros(4, 6), torch.zeros(3, 6), torch.zeros(4, dtype=torch.int64), reduction="avg")
