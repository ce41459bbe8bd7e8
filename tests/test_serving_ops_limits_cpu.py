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


def test_tree_attention_reconverges_before_whole_warp_accesses(csrc=CSRC):
    """tcgen05.ld / st are .sync.aligned: after code in which lanes part (a slot's clean-up, one lane's arrival, rows that
    add back or store partials), a __syncwarp or a whole-warp wait stands before the next of them."""
    text = (csrc / "tree_attention.cu").read_text()
    body = text[text.index("// ------------------------------------------------ softmax and epilogue"):text.index("if (!okay) {\n      // a wait gave up")]
    parts = ["*s_odd = 1;", "if (slot >= sl.len) {", "if (lane == 0) mbar_arrive(&turn", "} else if (live) {", "if (odd && live) {"]
    for mark in parts:
        assert body.count(mark) == 1, mark
        at = body.index(mark)
        if mark.startswith(("} else if (live)", "if (odd")):  # the next access is that of the loop's next turn
            at = body.rindex("for (int k = 0; k < D / 32; ++k)", 0, at)
        nxt = min(i for i in (body.find("tmem_ld32(", at), body.find("tmem_st32(", at)) if i > 0)
        assert "__syncwarp();" in body[at:nxt], mark
