"""CPU tier of the rotary, tree-attention and logits operators' edges: launch order of the tensor-memory kernels."""
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "comm_opt_b200" / "csrc"


@pytest.mark.parametrize("source", ["tree_attention.cu", "gemm_sm100.cu"])
def test_tensor_memory_is_allocated_before_dependents_may_start(source, csrc=CSRC):
    """A dependent kernel's CTA may join an SM once every CTA of this one has triggered. If a warp could trigger before
    its CTA's allocation, that CTA could take the columns that the allocation then waits for, while it waits for this kernel: a
    block barrier stands between the two, and the columns are given back after the last one."""
    text = (csrc / source).read_text()
    at = text.index(" tmem_alloc(tmem_slot")
    first = min(i for i in (text.find(w, at) for w in ("pdl_wait_then_trigger();", "pdl_trigger();")) if i > 0)
    assert "__syncthreads();" in text[at:first]
    assert text.rindex("tmem_dealloc(") > text.rindex("__syncthreads();") > first
