"""Limits of the sequence operators: head dims of zero, launches beyond what a dimension of the hardware's grid holds
(2^32 work items), which are refused before anything runs or cut into rows of workgroups."""
import ctypes

import pytest
import torch

from dgnn_amd import _lib
from dgnn_amd._lib import DgnnError
from dgnn_amd.operators import LinearCrossEntropyFuse, NodeEmbeddingFuse, PackedAttentionFuse

UNSUPPORTED = -2
P = 0x10000                      # an aligned address that is never read
DEV = "cuda:0"


def test_head_dim_of_zero_is_refused_as_such():
    q = torch.zeros(4, 2, 0)
    with pytest.raises(DgnnError):
        PackedAttentionFuse(q, q, q, torch.tensor([0, 4], dtype=torch.int32))


@pytest.mark.gpu
def test_head_dim_of_zero_is_refused_on_the_gpu():
    q = torch.zeros(4, 2, 0, device="cuda:0")
    with pytest.raises(DgnnError, match="head dims"):
        PackedAttentionFuse(q, q, q, torch.tensor([0, 4], dtype=torch.int32, device="cuda:0"))


@pytest.mark.parametrize("nseq,tq,tk,h", [(1 << 20, 1 << 28, 1 << 20, 7), (1 << 23, 1 << 28, 1 << 20, 7)])
def test_attention_beyond_the_grid_is_refused(nseq, tq, tk, h):
    """Within 2^31 rows times heads, but more tiles of rows (or, in the backward, of keys) than one launch takes."""
    lib, d = _lib.lib(), 8
    strides = (ctypes.c_longlong * 6)(h * d, d, h * d, d, h * d, d)
    assert lib.dgnn_attn_forward(1, nseq, tq, tk, h, h, d, 0, 1.0, P, P, P, strides, P, P, P, None, P, P, 1 << 60, None) == UNSUPPORTED
    for rows, keys in ((tq, tk), (tk, tq)):
        assert lib.dgnn_attn_backward(1, nseq, rows, keys, h, h, d, 0, 1.0, P, P, P, strides, P, P, P, None, P, P, P, P, P, P,
                                      1 << 60, None) == UNSUPPORTED


@pytest.mark.parametrize("dtype,rows,dim", [(0, 5, 1 << 25), (1, 5, (1 << 22) + 1), (2, 5, (1 << 30) + 1), (0, (1 << 31) - 1, 300)])
def test_embedding_beyond_the_grid_is_refused(dtype, rows, dim):
    lib = _lib.lib()
    assert lib.dgnn_embedding_backward(dtype, 8, 4, rows, dim, 1.0, P, P, P, P, 1 << 60, None) == UNSUPPORTED
    if dim > 1 << 30:
        assert lib.dgnn_embedding_forward(dtype, 8, 4, rows, dim, 1.0, P, P, P, None) == UNSUPPORTED


@pytest.mark.gpu
def test_embedding_of_more_rows_than_a_grid_holds():
    """A workgroup a row: 2^24 of 256 threads are one dimension's end."""
    n, rows, dim = (1 << 24) + 77, 301, 129
    table = torch.randn(rows, dim, device=DEV).bfloat16()
    ids = torch.arange(n, device=DEV, dtype=torch.int32) % (rows + 1)
    out = NodeEmbeddingFuse(ids, table)
    want = torch.cat([table, torch.zeros(1, dim, dtype=table.dtype, device=DEV)])
    whole = n // (rows + 1) * (rows + 1)
    assert bool((out[:whole].view(-1, rows + 1, dim) == want).all()) and torch.equal(out[whole:], want[:n - whole])


@pytest.mark.gpu
def test_loss_of_more_tiles_than_a_grid_holds():
    """2^22 rows and 2^16 classes of floats are 2^24 tiles of 128 x 128.  Rows repeat with an odd period, so that every
    tile's share shows in some row that has to equal the first period's, to the bit."""
    n, classes, dim, period = 1 << 22, 1 << 16, 4, 1021
    gen = torch.Generator(device=DEV).manual_seed(0)
    some = torch.randn(period, dim, device=DEV, generator=gen)
    weight = torch.randn(classes, dim, device=DEV, generator=gen)
    pick = torch.randint(0, classes, (period,), device=DEV, generator=gen)
    at = torch.arange(n, device=DEV) % period
    loss = LinearCrossEntropyFuse(some[at], weight, pick[at], reduction="none")
    z = some.double() @ weight.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, pick[:, None])[:, 0]
    # a score: 4 products of floats; a sum of exponentials: 25 additions in float (16 + 4 + 1 + 4), a term 2 |z| + 8 roundings
    mass = (some.double().abs() @ weight.double().abs().t()).amax(1)
    bound = (2 * 4 * mass + 25 + 4 * z.abs().amax(1) + 16) * 2.0 ** -24
    assert ((loss[:period].double() - want).abs() <= bound).all()
    assert torch.equal(loss, loss[:period][at])
