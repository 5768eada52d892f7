"""Limits of the sequence operators that show without a GPU: head dims of zero."""
import pytest
import torch

from dgnn_amd._lib import DgnnError
from dgnn_amd.operators import PackedAttentionFuse


def test_head_dim_of_zero_is_refused_as_such():
    q = torch.zeros(4, 2, 0)
    with pytest.raises(DgnnError):
        PackedAttentionFuse(q, q, q, torch.tensor([0, 4], dtype=torch.int32))


@pytest.mark.gpu
def test_head_dim_of_zero_is_refused_on_the_gpu():
    q = torch.zeros(4, 2, 0, device="cuda:0")
    with pytest.raises(DgnnError, match="head dims"):
        PackedAttentionFuse(q, q, q, torch.tensor([0, 4], dtype=torch.int32, device="cuda:0"))
