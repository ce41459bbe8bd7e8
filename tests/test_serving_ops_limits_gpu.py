"""Calls of the rotary, tree-attention and logits operators at the edges of what they allow: alignment, aliasing, extreme
values, launch order, autograd's modes, and the kernel forms that only many rows select."""

import pytest
import torch

from comm_opt_b200.ops import kernels as K
from test_serving_ops_gpu import (F32U, check_tree, close, gen, logits_ref, make_tree, norm_rotate64, norm_rotate_grad64, randn,
                                  rotate64, tiny, tree_ref, u)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ alignment
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("off", [1, 2, 4, 7])
def test_tree_attention_of_a_misaligned_contiguous_query(cuda, dtype, off):
    """A contiguous q that starts off a 16-byte boundary is copied; the result is that of the aligned one."""
    g = gen(cuda, off)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, 2, 5, 8, 2, 64, [3, 40], dtype)
    flat = torch.empty(q.numel() + 8, device=cuda, dtype=dtype)
    odd = flat[off:off + q.numel()].view_as(q).copy_(q)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    assert torch.equal(K.tree_attention(odd, kc, vc, bt, cl, bits, 0.125), K.tree_attention(q, kc, vc, bt, cl, bits, 0.125))
