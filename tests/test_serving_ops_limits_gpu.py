"""Calls of the rotary, tree-attention and logits operators at the edges of what they allow: alignment, aliasing, extreme
values, launch order, autograd's modes, and the kernel forms that only many rows select."""

import math

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


# ---------------------------------------------------------------------------------------------- launch order
def test_tree_attention_between_gemms_with_programmatic_launch(cuda):
    """Heads of 64 and at most 8 pages a sequence (one kernel, which leaves room for another on its SM) between GEMMs, which
    take tensor memory too: the same bits as launched one after another."""
    from comm_opt_b200.models.gemm import gemm, gemm_error_word

    g = gen(cuda, 3)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, 2, 8, 8, 2, 64, [60, 33], torch.bfloat16)
    w = randn(g, 2048, 512, dtype=torch.bfloat16, std=0.05)
    w2 = randn(g, 512, 2048, dtype=torch.bfloat16, std=0.05)

    def chain():
        x = q
        for _ in range(4):
            o = K.tree_attention(x, kc, vc, bt, cl, bits, 0.125)
            h = gemm(o.view(16, 512), w, pdl=K.native().get_pdl(), small_smem=True)
            x = gemm(h, w2, pdl=K.native().get_pdl(), small_smem=True).view_as(q)
        return x

    assert bt.shape[1] <= 8
    want = chain()
    old = K.set_pdl(True)
    try:
        got = [chain() for _ in range(20)]
        torch.cuda.synchronize()
    finally:
        K.set_pdl(old)
    assert all(torch.equal(x, want) for x in got)
    assert int(gemm_error_word(cuda)) == 0


# --------------------------------------------------------------------------------------------------- lengths
def test_histories_and_biases_past_the_kernel_s_indexes_are_refused(cuda):
    """The kernel steps ahead in 32-bit indexes: rows close to 2^31 entries would wrap and read out of range."""
    x, one = torch.zeros(1, 64, device=cuda), torch.ones(1, device=cuda)
    many = torch.empty(1, 2 ** 30 + 1, dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError, match="at most 2\\^30 ids"):
        K.penalize_logits(x, tokens=many, presence=one)
    with pytest.raises(RuntimeError, match="at most 2\\^30 biases"):
        K.penalize_logits(x, bias_ids=many, bias=many.view(torch.float32))
    # (the longest history that is taken: it ends, and counts what it holds)
    many = many[:, :2 ** 30].fill_(-1)
    many[0, [0, 12345, -1]] = torch.tensor([3, 5, 5], dtype=torch.int32, device=cuda)
    y = K.penalize_logits(x, tokens=many, frequency=one)
    want = torch.zeros_like(x)
    want[0, 3], want[0, 5] = -1, -2
    assert torch.equal(y, want)


# ------------------------------------------------------------------------------------------ lanes that part
@pytest.mark.parametrize("D,T,nq,dtype", [(64, 41, 3, torch.float16), (128, 41, 3, torch.bfloat16), (128, 30, 9, torch.bfloat16)])
def test_tree_attention_rows_that_add_back_beside_rows_that_do_not(cuda, D, T, nq, dtype):
    """Non-finite v of single drafted tokens over a context that is cut between shares: in a warp some rows see them, some
    do not and some are padding. Rows that do not see them keep their bits, the others get the value."""
    g = gen(cuda, T + nq)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, 2, T, nq, 1, D, [5000, 77], dtype)
    tl = torch.tensor([T - 2, T], dtype=torch.int32, device=cuda)
    want = K.tree_attention(q, kc, vc, bt, cl, bits, 0.1, tree_lens=tl)
    bad = vc.clone()
    seen = torch.zeros(2, T, D, dtype=torch.bool, device=cuda)
    for b in range(2):
        for j, d in ((3, 5), (T - 5, 40), (17, D - 1)):
            slot = int(cl[b]) + j
            bad[bt[b, slot // 16].long(), 0, slot % 16, d] = float("inf")
            seen[b, :, d] |= ((bits[b] >> j) & 1).bool()
        seen[b, int(tl[b]):] = False
    got = K.tree_attention(q, kc, bad, bt, cl, bits, 0.1, tree_lens=tl)
    hit = seen[:, :, None].expand_as(got)
    assert bool((got[hit] == float("inf")).all()) and bool(hit.any())
    assert torch.equal(got[~hit], want[~hit])


# ----------------------------------------------------------------------------------------- waits that run out
def test_tree_attention_wait_that_gives_up_is_reported(cuda):
    """With no time to wait every row that the call owes reads as NaN, padding keeps its value, and the device's word is set
    until it is cleared; the next call is a normal one. (Whole pieces and pieces cut between shares, one and two row tiles.)"""
    g = gen(cuda, 12)
    word = K.tree_attention_error_word(cuda)
    assert word.shape == (1,) and word.dtype == torch.int32 and int(word) == 0
    for B, T, nq, nkv, D, ctx in ((2, 5, 8, 2, 64, [40, 3]), (2, 40, 8, 1, 128, [3000, 9]), (3, 9, 2, 1, 128, [0, 700, 64])):
        q, kc, vc, bt, cl, bits = make_tree(g, cuda, B, T, nq, nkv, D, ctx, torch.bfloat16)
        tl = torch.full((B,), T, dtype=torch.int32, device=cuda)
        tl[-1] = 2
        want = K.tree_attention(q, kc, vc, bt, cl, bits, 0.1, tree_lens=tl)
        out = torch.full_like(q, 6.0)
        K.tree_attention(q, kc, vc, bt, cl, bits, 0.1, tree_lens=tl, out=out, timeout_ms=0)
        live = torch.arange(T, device=cuda)[None] < tl[:, None]
        assert bool(out[live].isnan().all()) and bool((out[~live] == 6).all())
        assert int(K.tree_attention_error_word(cuda)) == 1
        word.zero_()
        assert torch.equal(K.tree_attention(q, kc, vc, bt, cl, bits, 0.1, tree_lens=tl), want) and int(word) == 0
    with pytest.raises(RuntimeError, match="timeout_ms"):
        K.tree_attention(q, kc, vc, bt, cl, bits, 0.1, timeout_ms=-1)


# ------------------------------------------------------------------------------------------- shared allocations
def test_disjoint_parts_of_one_allocation_are_taken(cuda):
    """Operands and outputs cut from one arena give what operands of their own give."""
    g = gen(cuda, 6)
    B, S, nq, nkv, D = 2, 3, 4, 2, 64
    n = nq + 2 * nkv
    cos, sin = K.rotary_tables(64, D, device=cuda)
    pos = torch.arange(S, device=cuda, dtype=torch.int32)
    sizes = dict(qkv=(B, S, n * D), q=(B, S, nq, D), k=(8, nkv, 16, D), v=(8, nkv, 16, D), o=(B, S, nq, D))
    arena = randn(g, sum(math.prod(s) for s in sizes.values()), dtype=torch.bfloat16)
    part, at = {}, 0
    for name, s in sizes.items():
        part[name] = arena[at:at + math.prod(s)].view(s)
        at += math.prod(s)
    own = {name: t.clone() for name, t in part.items()}
    bt = torch.arange(8, device=cuda, dtype=torch.int32).view(B, 4)
    at0 = torch.tensor([5, 30], device=cuda, dtype=torch.int32)
    for t in (part, own):
        K.qk_norm_rotary_append_kv(t["qkv"], pos, cos, sin, bt, at0, t["q"], t["k"], t["v"], nq, nkv)
        K.tree_attention(t["q"], t["k"], t["v"], bt, at0, None, 0.125, out=t["o"])
        K.rotary(t["q"], pos, cos, sin, out=t["qkv"].view(-1)[:t["q"].numel()].view(t["q"].shape))
    assert all(torch.equal(part[name], own[name]) for name in sizes)
    two = randn(g, 2, 4, 100)
    want = K.penalize_logits(two[0].clone(), allowed=torch.full((4, 4), 5, dtype=torch.int32, device=cuda))
    assert torch.equal(K.penalize_logits(two[0], allowed=torch.full((4, 4), 5, dtype=torch.int32, device=cuda), out=two[1]), want)
    assert torch.equal(two[1], want)


def test_overlapping_operands_are_refused(cuda):
    """What a call writes lies apart from everything else it reads or writes, whatever the views' types and starts."""
    cos, sin = K.rotary_tables(64, 64, device=cuda)

    def bad(fn, *a, **k):
        with pytest.raises(RuntimeError, match="overlap|memory of"):
            fn(*a, **k)

    raw = torch.zeros(1 << 16, dtype=torch.uint8, device=cuda)

    def cut(dtype, start, *shape):
        n = math.prod(shape) * dtype.itemsize
        return raw[start:start + n].view(dtype).view(shape)

    pos = torch.zeros(2, dtype=torch.int32, device=cuda)
    x = torch.zeros(2, 3, 64, device=cuda)
    bad(K.rotary, x, cut(torch.int32, 0, 2), cos, sin, out=cut(torch.float32, 0, 2, 3, 64))
    c2 = cut(torch.float32, 1024, 4, 32)
    bad(K.rotary, x, pos, c2, sin[:4].clone(), out=cut(torch.float32, 0, 2, 3, 64))
    bad(K.rotary, cut(torch.float32, 256, 2, 3, 64), pos, cos, sin, out=cut(torch.float32, 0, 2, 3, 64))
    # caches that share pages, and an append over what it reads
    kv = torch.zeros(4, 2, 16, 64, device=cuda).half()
    qkv = torch.zeros(1, 2, 8 * 64, device=cuda).half()
    bt, st = torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 2, 4, 64, device=cuda).half()
    ok = dict(positions=pos, cos=cos, sin=sin, block_tables=bt, starts=st, q_out=q, k_cache=kv, v_cache=kv.clone(), nq=4, nkv=2)
    bad(K.qk_norm_rotary_append_kv, qkv, **{**ok, "k_cache": kv[:3], "v_cache": kv[1:]})
    bad(K.qk_norm_rotary_append_kv, qkv, **{**ok, "q_out": kv.view(-1)[100:612].view(1, 2, 4, 64)})
    bad(K.qk_norm_rotary_append_kv, qkv, **{**ok, "q_out": cut(torch.half, 0, 1, 2, 4, 64), "positions": cut(torch.int32, 1016, 2)})
    bad(K.qk_norm_rotary_append_kv, qkv, **{**ok, "q_out": cut(torch.half, 0, 1, 2, 4, 64), "block_tables": cut(torch.int32, 512, 1, 2)})
    bad(K.qk_norm_rotary_append_kv, qkv, **{**ok, "q_out": cut(torch.half, 0, 1, 2, 4, 64)}, bias=cut(torch.half, 1000, 512))
    # tree attention over its own queries' tail, mask and lengths
    o = cut(torch.half, 0, 1, 2, 4, 64)
    bad(K.tree_attention, cut(torch.half, 512, 1, 2, 4, 64), kv, kv.clone(), bt, st, None, 0.1, out=o)
    bad(K.tree_attention, q, kv, kv.clone(), bt, st, cut(torch.int64, 512, 2), 0.1, out=o)
    bad(K.tree_attention, q, kv, kv.clone(), bt, cut(torch.int32, 64, 1), None, 0.1, out=o)
    # logits
    y, L = cut(torch.float32, 0, 2, 64), torch.zeros(2, 64, device=cuda)
    one = torch.ones(2, device=cuda)
    bad(K.penalize_logits, L, tokens=cut(torch.int32, 64, 2, 4), presence=one, out=y)
    bad(K.penalize_logits, L, allowed=cut(torch.int32, 64, 2, 2), out=y)
    bad(K.penalize_logits, L, keys=cut(torch.int64, 64, 2), out=y)
    bad(K.penalize_logits, L, tokens=torch.zeros(2, 4, dtype=torch.int32, device=cuda), presence=cut(torch.float32, 64, 2), out=y)
    bad(K.penalize_logits, y, keys=cut(torch.int64, 64, 2))
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------- autograd
def _calls(dev, dtype=torch.float32):
    """name -> (call, tensors that it writes in place)."""
    cos, sin = K.rotary_tables(64, 64, device=dev)
    pos = torch.arange(2, dtype=torch.int32, device=dev)
    x, y = torch.randn(2, 3, 64, device=dev), torch.empty(2, 3, 64, device=dev)
    h = torch.randn(1, 2, 4, 64, device=dev).half()
    kc, vc = torch.randn(3, 2, 16, 64, device=dev).half(), torch.randn(3, 2, 16, 64, device=dev).half()
    bt, cl = torch.arange(2, dtype=torch.int32, device=dev).view(1, 2), torch.zeros(1, dtype=torch.int32, device=dev)
    qkv, o = torch.randn(1, 2, 8 * 64, device=dev).half(), torch.empty_like(h)
    L, M = torch.randn(2, 64, device=dev), torch.empty(2, 64, device=dev)
    keys = torch.zeros(2, dtype=torch.int64, device=dev)
    return dict(
        rotary_in_place=(lambda: K.rotary(x, pos, cos, sin, out=x), [x]),
        rotary_out=(lambda: K.rotary(x, pos, cos, sin, out=y), [y]),
        append=(lambda: K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, cl, o, kc, vc, 4, 2), [o, kc, vc]),
        tree=(lambda: K.tree_attention(h, kc, vc, bt, cl, None, 0.1, out=o), [o]),
        logits_in_place=(lambda: K.penalize_logits(L, out=L, keys=keys), [L, keys]),
        logits_out=(lambda: K.penalize_logits(L, out=M), [M]))


def test_outputs_written_in_place_raise_their_version(cuda):
    for name, (call, written) in _calls(cuda).items():
        before = [t._version for t in written]
        call()
        assert all(t._version > v for t, v in zip(written, before)), name
    # a value that a backward pass needs, overwritten before it: refused, as for torch's own operators
    cos, sin = K.rotary_tables(8, 64, device=cuda)
    pos, w = torch.arange(3, device=cuda, dtype=torch.int32), torch.ones(64, device=cuda)
    q = torch.randn(3, 2, 64, device=cuda, requires_grad=True)
    k = torch.randn(3, 1, 64, device=cuda)
    p = q * 1.0
    y, _ = K.qk_norm_rotary(p, k, w, w, pos, cos, sin)
    with torch.no_grad():
        K.rotary(p, pos, cos, sin, out=p)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    # tensors made in inference mode have no version: written as before, inside and outside of it
    with torch.inference_mode():
        for call, _ in _calls(cuda).values():
            call()
        late = _calls(cuda)
    for call, _ in late.values():
        call()


def test_gradients_that_are_not_formed_are_refused(cuda):
    """Operators without a backward pass, and forward-mode tangents, raise where a derivative would be lost."""
    import torch.autograd.forward_ad as fwd

    cos, sin = K.rotary_tables(64, 64, device=cuda)
    pos = torch.arange(2, dtype=torch.int32, device=cuda)
    h = torch.randn(1, 2, 4, 64, device=cuda).half()
    kc, vc = torch.randn(3, 2, 16, 64, device=cuda).half(), torch.randn(3, 2, 16, 64, device=cuda).half()
    bt, cl = torch.arange(2, dtype=torch.int32, device=cuda).view(1, 2), torch.zeros(1, dtype=torch.int32, device=cuda)
    qkv, w = torch.randn(1, 2, 8 * 64, device=cuda).half(), torch.ones(64, device=cuda).half()
    L, one = torch.randn(2, 64, device=cuda), torch.ones(2, device=cuda)
    tok = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    ids, bias = torch.zeros(2, 1, dtype=torch.int32, device=cuda), torch.ones(2, 1, device=cuda)
    x, x1, wf = torch.randn(2, 3, 64, device=cuda), torch.randn(2, 1, 64, device=cuda), torch.ones(64, device=cuda)

    def tree(q=h, k=kc, v=vc):
        return K.tree_attention(q, k, v, bt, cl, None, 0.1)

    def append(qkv=qkv, wq=w, wk=w, b=qkv[0, 0].clone()):
        return K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, cl, torch.empty_like(h), kc.clone(), vc.clone(), 4, 2,
                                          q_weight=wq, k_weight=wk, bias=b)

    def logits(x=L, rep=one, freq=one, pres=one, bias=bias):
        return K.penalize_logits(x, tokens=tok, repetition=rep, frequency=freq, presence=pres, bias_ids=ids, bias=bias)

    def back(dq=x, dk=x1, q=x, k=x1, wq=wf, wk=wf):
        return K.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, pos, cos, sin)

    plain = [(tree, dict(q=h, k=kc, v=vc)), (append, dict(qkv=qkv, wq=w, wk=w, b=qkv[0, 0].clone())),
             (logits, dict(x=L, rep=one, freq=one, pres=one, bias=bias))]
    for fn, args in plain:
        want = fn()
        for name, t in args.items():
            leaf = t.clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient"):
                fn(**{name: leaf})
            with torch.no_grad():
                got = fn(**{name: leaf})
            for a, b in zip(*((r if isinstance(r, tuple) else (r,)) for r in (got, want))):
                assert torch.equal(a, b), (fn.__name__, name)
    outs = dict(rotary=lambda x: K.rotary(x, pos, cos, sin), rotary_out=lambda x: K.rotary(x, pos, cos, sin, out=torch.empty(2, 3, 64, device=cuda)),
                q=lambda x: K.qk_norm_rotary(x, x1, wf, wf, pos, cos, sin), k=lambda x: K.qk_norm_rotary(x1, x, wf, wf, pos, cos, sin),
                w=lambda w: K.qk_norm_rotary(x, x1, w, wf, pos, cos, sin), logits=lambda x: logits(x=x), back=lambda q: back(q=q),
                tree=lambda q: tree(q=q), append=lambda t: append(qkv=t))
    give = dict(w=wf, logits=L, tree=h, append=qkv)
    with fwd.dual_level():
        for grad in (False, True):
            for name, fn in outs.items():
                t = give.get(name, x).clone().requires_grad_(grad)
                dual = fwd.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward-mode|no gradient"):
                    fn(dual)


# ------------------------------------------------------------------------------------------------ arguments
def test_append_takes_positions_by_batch_and_sequence_only(cuda):
    """[seq, batch] positions hold as many numbers and would rotate every row by another's."""
    cos, sin = K.rotary_tables(64, 64, device=cuda)
    B, S, nq, nkv = 2, 3, 2, 1
    qkv = torch.randn(B, S, 4 * 64, device=cuda)
    bt, st = torch.arange(4, dtype=torch.int32, device=cuda).view(B, 2), torch.zeros(B, dtype=torch.int32, device=cuda)
    pos = torch.arange(6, dtype=torch.int32, device=cuda).view(B, S)

    def call(p, x=qkv):
        q, k, v = (torch.zeros(s, device=cuda) for s in ((B, S, nq, 64), (4, nkv, 16, 64), (4, nkv, 16, 64)))
        K.qk_norm_rotary_append_kv(x, p, cos, sin, bt, st, q, k, v, nq, nkv)
        return q, k, v

    want = call(pos)
    for same in (call(pos.flatten()), call(pos, qkv.flatten(0, 1)), call(pos.flatten(), qkv.flatten(0, 1))):
        assert all(torch.equal(a, b) for a, b in zip(same, want))
    row = torch.arange(S, dtype=torch.int32, device=cuda)
    assert all(torch.equal(a, b) for a, b in zip(call(row), call(row.expand(B, S).contiguous())))
    for p in (pos.t().contiguous(), pos[None], pos[:, :, None], pos[:, None], row[None], pos.flatten()[:, None]):
        with pytest.raises(RuntimeError, match="positions"):
            call(p)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e60])
def test_tree_attention_refuses_a_scale_that_is_not_finite(cuda, scale):
    q, kc, vc, bt, cl, bits = make_tree(gen(cuda, 1), cuda, 1, 3, 2, 1, 64, [20], torch.float16)
    with pytest.raises(RuntimeError, match="scale"):
        K.tree_attention(q, kc, vc, bt, cl, bits, scale)


# --------------------------------------------------------------------------------------------- small weights
@pytest.mark.parametrize("D,T,G", [(64, 1, 1), (128, 3, 2), (64, 64, 4)])
@pytest.mark.parametrize("bits", [12, 20, 26, 30])
def test_tree_attention_weights_behind_one_strong_token(cuda, D, T, G, bits):
    """One token with weight 1 and v = 0, 4000 tokens with weights of 2^-bits and v = 1 (fp16), heads enough for each to be
    walked whole by one CTA: the many are what the row says, although each weight is far below the strong one's step.

    A weight is held as fp16(2^11 w), w relative to the row's reference maximum, which is at most 2^4 below the true one:
    normal numbers (half a step of the type) down to w = 2^-25, below that off by at most 2^-25 / 2^11 = 2^-36 each."""
    B, nkv, n, dtype = 6, 64, 4001, torch.float16
    pages = (n + T + 15) // 16
    kc = torch.zeros(B * pages, nkv, 16, D, device=cuda, dtype=dtype)
    vc = torch.ones(B * pages, nkv, 16, D, device=cuda, dtype=dtype)
    bt = torch.arange(B * pages, device=cuda, dtype=torch.int32).view(B, pages)
    kc[bt[:, 0].long(), :, 5, 0], vc[bt[:, 0].long(), :, 5] = bits, 0.0  # exact in the type; the score is bits * ln 2
    q = torch.zeros(B, T, nkv * G, D, device=cuda, dtype=dtype)
    q[..., 0] = 1.0
    cl = torch.full((B,), n, device=cuda, dtype=torch.int32)
    mask = torch.zeros(T, dtype=torch.int64, device=cuda)  # no drafted token sees another or itself
    y = K.tree_attention(q, kc, vc, bt, cl, mask, math.log(2.0))
    many = (n - 1) * 2.0 ** -bits
    ref = torch.full_like(y, many / (1 + many), dtype=torch.float64)
    # the score's error: one rounding of the scale and of the product, each of bits * ln 2; sums over n slots in fp32;
    # each weight's rounding, and the absolute one below the normal numbers
    err = ref * (2 * (D + 8) * F32U * bits + (n + 32) * F32U + u(dtype)) + (n - 1) * 2.0 ** -36
    close(y, ref, err)


# --------------------------------------------------------------------------------------------- greedy choice
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_greedy_choice_takes_the_lowest_of_equal_zeros(cuda, dtype):
    """-0 and +0 are equal: the lowest id wins, in argmax_local and in the penalties' keys."""
    x = torch.full((3, 300), -1.0, device=cuda, dtype=dtype)
    x[0, 7], x[0, 8], x[0, 290] = -0.0, 0.0, 0.0
    x[1, 100], x[1, 101] = 0.0, -0.0
    x[2, 299], x[2, 298] = 0.0, -0.0
    keys = torch.zeros(3, dtype=torch.int64, device=cuda)
    y = K.penalize_logits(x, keys=keys)
    assert torch.equal(y, x) and torch.equal(keys, K.argmax_local(x, 0))
    assert K.argmax_combine(keys.view(1, 3), 1).tolist() == [7, 100, 298] == x.float().argmax(-1).tolist()


# -------------------------------------------------------------------------------------------------- transposes
@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_transpose_also_of_scaled_tables(cuda, interleaved):
    """YaRN tables carry a factor m: rotating and rotating back multiplies by m^2; the gradient is the transpose."""
    g = gen(cuda, 13)
    cos, sin = K.rotary_tables(40, 32, 1e4, dict(type="yarn", factor=16.0, original=20), device=cuda)
    m2 = (0.1 * math.log(16.0) + 1.0) ** 2
    pos = torch.arange(9, device=cuda, dtype=torch.int32)
    x = randn(g, 2, 9, 3, 64).requires_grad_()
    y = K.rotary(x, pos, cos, sin, interleaved=interleaved)
    dy = randn(g, 2, 9, 3, 64)
    (dx,) = torch.autograd.grad(y, x, dy)
    back = K.rotary(dy, pos, cos, sin, interleaved=interleaved, inverse=True)
    assert torch.equal(dx, back)
    ref, mag = rotate64(dy.double(), cos[:9], sin[:9], interleaved, -1.0)
    close(back, ref, 3 * F32U * mag)
    round_trip = K.rotary(y.detach(), pos, cos, sin, interleaved=interleaved, inverse=True).double()
    want = x.detach().double().clone()
    a, b = ((slice(0, 32, 2), slice(1, 32, 2)) if interleaved else (slice(0, 16), slice(16, 32)))
    want[..., a] *= m2
    want[..., b] *= m2
    big = float(x.detach().abs().max()) * 2 * m2
    assert float((round_trip - want).abs().max()) <= 12 * F32U * big


# -------------------------------------------------------------- forms that only many rows select (rotary.cu's launchers)
SMS = 148


def _lanes(D, V):
    gl = 1
    while gl < 32 and gl < D // (2 * V):
        gl *= 2
    return gl


def _forward_form(rows, heads, D, steps):
    """(several heads a lane, head blocks that a warp takes, whether the last step of the widest operand is partial)"""
    per = 32 // _lanes(D, 8)
    many = rows * sum(heads) >= SMS * 64 * per
    blocks = [-(-h // (per * steps)) for h in heads]
    inner = max(1, min(sum(blocks), rows * sum(blocks) // (SMS * 32)))
    return many, inner, heads[0] % (per * steps) != 0


def _dw_chain(rows, heads, other, D, V, hpt):
    """The longest chain of additions behind a weight's gradient: a lane's rows and heads, lanes, warps, blocks."""
    cost = (heads + 12, other + 12)
    nb = max(1, min(SMS * 3 * cost[0] // sum(cost), rows * ((heads + 7) // 8)))
    per = 32 // _lanes(D, V)
    inner = 4 if rows >= SMS * 24 else 1
    groups = -(-(-(-heads // (per * hpt))) // inner)
    units = -(-rows * groups // (nb * 4))
    return units * inner * hpt + 5 + 4 + -(-nb // 32) + 5


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,H,D,rot", [(8, 512, 40, 128, 64), (3, 1111, 37, 128, 128), (1, 4001, 50, 64, 64), (2, 2000, 21, 256, 64)])
def test_rotary_of_many_rows(cuda, interleaved, dtype, B, S, H, D, rot):
    many, inner, partial = _forward_form(B * S, (H,), D, 3)
    assert many and inner > 1 and partial
    g = gen(cuda, S)
    cos, sin = K.rotary_tables(300, rot, 1e4, device=cuda)
    pos = torch.randint(0, 300, (B, S), generator=g, device=cuda, dtype=torch.int32)
    pos[0, 5], pos[-1, -1] = -1, 300
    wide = randn(g, B, S, H + 2, D, dtype=dtype)
    x = wide[:, :, 1:H + 1]
    p = pos.long().clamp(0, 299)
    pad = (pos < 0) | (pos >= 300)
    for inverse in (False, True):
        ref, mag = rotate64(x.double(), cos[p], sin[p], interleaved, -1.0 if inverse else 1.0)
        ref[pad], mag[pad] = 0, 0
        y = K.rotary(x, pos, cos, sin, interleaved=interleaved, inverse=inverse)
        close(y, ref, 3 * F32U * mag)
        z = wide.clone()
        K.rotary(z[:, :, 1:H + 1], pos, cos, sin, interleaved=interleaved, inverse=inverse, out=z[:, :, 1:H + 1])
        assert torch.equal(z[:, :, 1:H + 1], y) and torch.equal(z[:, :, 0], wide[:, :, 0]) and torch.equal(z[:, :, -1], wide[:, :, -1])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,nq,nk,D,rot", [(4, 2048, 37, 5, 128, 128), (2, 1000, 37, 5, 128, 64), (1, 3553, 40, 8, 128, 128),
                                             (2, 4100, 5, 1, 64, 64), (3, 1300, 21, 3, 64, 32)])
def test_qk_norm_rotary_of_many_rows(cuda, interleaved, dtype, B, S, nq, nk, D, rot):
    rows = B * S
    many, inner, _ = _forward_form(rows, (nq, nk), D, 2)
    assert many == (nq > 5) and (not many or inner > 1)
    g = gen(cuda, S + nq)
    cos, sin = K.rotary_tables(300, rot, 1e4, device=cuda)
    pos = torch.randint(0, 300, (B, S), generator=g, device=cuda, dtype=torch.int32)
    pos[0, 3], pos[-1, S // 2] = -1, 300
    pad = (pos < 0) | (pos >= 300)
    live = ~pad
    p = pos.long().clamp(0, 299)
    c, s = cos[p][live], sin[p][live]
    qkv = randn(g, B, S, nq + 2 * nk, D, dtype=dtype, std=2.0)
    qkv[pad] = float("nan")  # what padding may hold
    q, k = qkv[:, :, :nq].detach().requires_grad_(), qkv[:, :, nq:nq + nk].detach().requires_grad_()
    wq, wk = (1 + 0.2 * randn(g, D)).requires_grad_(), (1 + 0.2 * randn(g, D)).requires_grad_()
    ys = K.qk_norm_rotary(q, k, wq, wk, pos, cos, sin, 1e-6, interleaved=interleaved)
    for y, x, w in zip(ys, (q, k), (wq, wk)):
        ref, mag = norm_rotate64(x.detach()[live], w.detach(), c, s, 1e-6, interleaved)
        close(y.detach()[live], ref, (D + 10) * F32U * torch.maximum(mag, ref.abs()))
        assert not bool(y[pad].any())
    for sparse in (False, True):  # all rows; then a few rows and heads only, so that none of them can be missing from dw
        dys = [randn(g, *y.shape, dtype=dtype) for y in ys]
        if sparse:
            dys = [d * (torch.rand(d.shape[:3], generator=g, device=cuda) < 40 / (rows * d.shape[2]))[..., None] for d in dys]
        for d in dys:
            d[pad] = float("nan")
        grads = torch.autograd.grad(ys, (q, k, wq, wk), dys, retain_graph=True)
        again = K.qk_norm_rotary_backward(*dys, q, k, wq, wk, pos, cos, sin, 1e-6, interleaved=interleaved)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))  # a fixed order of the sums
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            dx, mag, dw, wmag = norm_rotate_grad64(x.detach()[live], w.detach(), dys[i][live], c, s, 1e-6, interleaved)
            close(grads[i][live], dx, (3 * D + 20) * F32U * mag)
            assert not bool(grads[i][pad].any())
            n = _dw_chain(rows, x.shape[2], (nk, nq)[i], D, 8, 2)
            close(grads[2 + i], dw, (n + D + 20) * F32U * wmag)


@pytest.mark.parametrize("dtype,D,rot,off", [(torch.bfloat16, 80, 20, 0), (torch.float16, 96, 24, 0), (torch.float32, 80, 20, 0),
                                             (torch.bfloat16, 64, 64, 1)])
def test_qk_norm_rotary_of_many_narrow_rows(cuda, dtype, D, rot, off):
    """Vectors that the layout or the alignment keeps narrow, with rows enough for four head blocks a warp."""
    B, S, nq, nk = 2, 1900, 5, 2
    assert B * S >= SMS * 24
    g = gen(cuda, D + off)
    cos, sin = K.rotary_tables(S, rot, 1e4, device=cuda)
    pos = torch.arange(S, device=cuda, dtype=torch.int32)

    def operand(h):
        flat = torch.empty(B * S * h * D + off, device=cuda, dtype=dtype)
        return flat[off:].view(B, S, h, D).copy_(randn(g, B, S, h, D, dtype=dtype))

    q, k, dq, dk = operand(nq), operand(nk), operand(nq), operand(nk)
    wq, wk = 1 + 0.2 * randn(g, D), 1 + 0.2 * randn(g, D)
    ys = K.qk_norm_rotary(q, k, wq, wk, pos, cos, sin)
    grads = K.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, pos, cos, sin)
    for i, (x, w, d) in enumerate(((q, wq, dq), (k, wk, dk))):
        ref, mag = norm_rotate64(x, w, cos[None, :S], sin[None, :S], 1e-6, False)
        close(ys[i], ref, (D + 10) * F32U * torch.maximum(mag, ref.abs()))
        dx, mag, dw, wmag = norm_rotate_grad64(x, w, d, cos[None, :S], sin[None, :S], 1e-6, False)
        close(grads[i], dx, (3 * D + 20) * F32U * mag)
        close(grads[2 + i], dw, (_dw_chain(B * S, x.shape[2], (nk, nq)[i], D, 1, 1) + D + 20) * F32U * wmag)


@pytest.mark.parametrize("interleaved,norm,bias", [(False, True, True), (True, True, False), (False, False, True), (True, False, False)])
@pytest.mark.parametrize("dtype,B,S,nq,nkv,D,rot", [(torch.bfloat16, 4, 2048, 40, 8, 128, 128), (torch.float16, 3, 1111, 37, 5, 128, 64),
                                                    (torch.bfloat16, 5, 901, 21, 7, 64, 64)])
def test_append_of_many_rows(cuda, interleaved, norm, bias, dtype, B, S, nq, nkv, D, rot):
    many, inner, partial = _forward_form(B * S, (nq, nkv, nkv), D, 2 if norm else 3)
    assert many and inner > 1 and partial == (nq != 40 or not norm)
    g = gen(cuda, S + D)
    n, pages = nq + 2 * nkv, (S + 40 + 15) // 16
    cos, sin = K.rotary_tables(S + 60, rot, 1e4, device=cuda)
    qkv = randn(g, B, S, n * D + 16, dtype=dtype)[..., :n * D]
    starts = torch.randint(0, 41, (B,), generator=g, device=cuda, dtype=torch.int32)
    lens = torch.randint(1, S + 1, (B,), generator=g, device=cuda, dtype=torch.int32)
    lens[0], lens[1] = S, 0
    pos = torch.randint(0, S + 60, (B, S), generator=g, device=cuda, dtype=torch.int32)
    pos[0, 7] = -1
    bt = torch.randperm(B * pages, generator=g, device=cuda).to(torch.int32).view(B, pages)
    kc, vc = (randn(g, B * pages, nkv, 16, D, dtype=dtype) for _ in range(2))
    wq, wk = (1 + 0.1 * randn(g, D)).to(dtype), (1 + 0.1 * randn(g, D)).to(dtype)
    bv = randn(g, n * D, dtype=dtype) if bias else None
    q_out = torch.full((B, S, nq, D), 3.0, device=cuda, dtype=dtype)
    k1, v1 = kc.clone(), vc.clone()
    K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, starts, q_out, k1, v1, nq, nkv, q_weight=wq if norm else None,
                               k_weight=wk if norm else None, eps=1e-5, lens=lens, bias=bv, interleaved=interleaved)
    live = (torch.arange(S, device=cuda)[None] < lens[:, None]) & (pos >= 0)
    x = (qkv.double() + (bv.double() if bias else 0)).view(B, S, n, D)[live]
    c, s = cos[pos[live].long()], sin[pos[live].long()]
    b, row = live.nonzero().T
    slot = starts.long()[b] + row
    page, at = bt[b, slot // 16].long(), slot % 16
    # a bias enters with one more rounding, of terms as large as |x| + |bias| <= 2 max
    extra = 12 * F32U * (float(x.abs().max()) + 1) if bias else 0
    n32 = ((D + 14) if norm else 4) * F32U
    for got, part, w in ((q_out[live], x[:, :nq], wq), (k1[page, :, at], x[:, nq:nq + nkv], wk)):
        ref, mag = norm_rotate64(part, w, c, s, 1e-5, interleaved) if norm else rotate64(part, c, s, interleaved)
        close(got, ref, n32 * torch.maximum(mag, ref.abs()) + extra)
    close(v1[page, :, at], x[:, nq + nkv:], extra)
    assert bool((q_out[~live] == 3).all())
    rest = torch.ones(B * pages, 16, dtype=torch.bool, device=cuda)
    rest[page, at] = False
    rest = rest[:, None].expand(-1, nkv, -1)
    assert torch.equal(k1[rest], kc[rest]) and torch.equal(v1[rest], vc[rest])


def test_qk_norm_rotary_gradients_of_one_output(cuda):
    """Only one of the two outputs used: the other's gradients are zeros."""
    g = gen(cuda, 2)
    cos, sin = K.rotary_tables(9, 64, device=cuda)
    pos = torch.arange(9, device=cuda, dtype=torch.int32)
    t = [randn(g, 2, 9, 4, 64), randn(g, 2, 9, 2, 64), 1 + randn(g, 64), 1 + randn(g, 64)]
    dys = [randn(g, 2, 9, 4, 64), randn(g, 2, 9, 2, 64)]
    whole = K.qk_norm_rotary_backward(*dys, *t, pos, cos, sin)
    for one in (0, 1):
        leaves = [v.clone().requires_grad_() for v in t]
        y = K.qk_norm_rotary(*leaves, pos, cos, sin)[one]
        grads = torch.autograd.grad(y, leaves, dys[one])
        for i in range(4):
            assert torch.equal(grads[i], whole[i] if i % 2 == one else torch.zeros_like(whole[i])), (one, i)


# -------------------------------------------------------------------------------------- large tree attentions
def test_tree_attention_of_several_launches(cuda):
    """300 sequences are three launches that share one workspace; contexts long enough that pieces are cut in each. Every
    row against its 64-bit statement, and the same bits under programmatic launch, where they follow closely."""
    g = gen(cuda, 31)
    B, T, nq, nkv, D = 300, 3, 8, 2, 64
    q, kc, vc, bt, _, bits = make_tree(g, cuda, B, T, nq, nkv, D, [900], torch.bfloat16)
    ctx = torch.randint(0, 900, (B,), generator=g, device=cuda, dtype=torch.int32)
    tl = torch.randint(0, T + 1, (B,), generator=g, device=cuda, dtype=torch.int32)
    out = torch.full_like(q, 4.0)
    K.tree_attention(q, kc, vc, bt, ctx, bits, 0.2, tree_lens=tl, out=out)
    ref, mag, sm = tree_ref(q, kc, vc, bt, ctx, bits.tolist(), 0.2, tl)
    check_tree(out, ref, mag, sm, 903, D)
    dead = torch.arange(T, device=cuda)[None] >= tl[:, None]
    assert bool((out[dead] == 4).all())
    old = K.set_pdl(True)
    try:
        outs = [torch.full_like(q, 4.0) for _ in range(10)]
        for o in outs:
            K.tree_attention(q, kc, vc, bt, ctx, bits, 0.2, tree_lens=tl, out=o)
        torch.cuda.synchronize()
    finally:
        K.set_pdl(old)
    assert all(torch.equal(o, out) for o in outs)


@pytest.mark.parametrize("T,nq,nkv,D,ctx", [(64, 64, 1, 128, [900, 5]), (64, 64, 1, 64, [300]), (4, 8, 1, 128, [20011]),
                                            (16, 16, 2, 64, [9000, 70])])
def test_tree_attention_of_many_rows_and_long_contexts(cuda, T, nq, nkv, D, ctx):
    """Up to sixteen row blocks of a KV head, and contexts far beyond one tile per share; the same bits every time."""
    g = gen(cuda, T + D)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, len(ctx), T, nq, nkv, D, ctx, torch.float16)
    y = K.tree_attention(q, kc, vc, bt, cl, bits, D ** -0.5)
    ref, mag, sm = tree_ref(q, kc, vc, bt, cl, bits.tolist(), D ** -0.5)
    check_tree(y, ref, mag, sm, max(ctx) + T, D)
    for _ in range(10):
        assert torch.equal(K.tree_attention(q, kc, vc, bt, cl, bits, D ** -0.5), y)


def test_tensors_that_are_not_their_memory_are_refused(cuda):
    """Lazily negated views, tensors whose storage was given back or never was, sparse ones: every operand."""
    cos, sin = K.rotary_tables(64, 64, device=cuda)
    pos = torch.arange(2, dtype=torch.int32, device=cuda)
    x, w = torch.randn(2, 3, 64, device=cuda), torch.ones(64, device=cuda)
    h = torch.randn(1, 2, 4, 64, device=cuda).half()
    kc, vc = (torch.randn(3, 2, 16, 64, device=cuda).half() for _ in range(2))
    bt, cl = torch.arange(2, dtype=torch.int32, device=cuda).view(1, 2), torch.zeros(1, dtype=torch.int32, device=cuda)
    qkv, wh, b = torch.randn(1, 2, 512, device=cuda).half(), w.half(), torch.randn(512, device=cuda).half()
    L, one = torch.randn(2, 64, device=cuda), torch.ones(2, device=cuda)
    tok, bits = torch.zeros(2, 4, dtype=torch.int32, device=cuda), torch.full((2, 2), -1, dtype=torch.int32, device=cuda)
    ids, bias = torch.zeros(2, 1, dtype=torch.int32, device=cuda), torch.ones(2, 1, device=cuda)
    keys, mask = torch.zeros(2, dtype=torch.int64, device=cuda), torch.ones(2, dtype=torch.int64, device=cuda)
    calls = [
        (K.rotary, dict(x=x, positions=pos, cos=cos, sin=sin)),
        (K.rotary, dict(x=x, positions=pos, cos=cos, sin=sin, out=torch.empty_like(x))),
        (K.qk_norm_rotary, dict(q=x, k=x[:, :1].clone(), q_weight=w, k_weight=w.clone(), positions=pos, cos=cos, sin=sin)),
        (K.qk_norm_rotary_backward, dict(dq=x.clone(), dk=x[:, :1].clone(), q=x, k=x[:, :1].clone(), q_weight=w, k_weight=w.clone(),
                                         positions=pos, cos=cos, sin=sin)),
        (K.qk_norm_rotary_append_kv, dict(qkv=qkv, positions=pos, cos=cos, sin=sin, block_tables=bt, starts=cl, q_out=h.clone(),
                                          k_cache=kc, v_cache=vc, nq=4, nkv=2, q_weight=wh, k_weight=wh.clone(), lens=cl + 2, bias=b)),
        (K.tree_attention, dict(q=h, k_cache=kc, v_cache=vc, block_tables=bt, ctx_lens=cl, tree_mask=mask, scale=1.0,
                                tree_lens=cl + 2, out=torch.empty_like(h))),
        (K.penalize_logits, dict(logits=L, tokens=tok, lens=tok[:, 0].clone(), prompt_lens=tok[:, 0].clone(), repetition=one,
                                 frequency=one.clone(), presence=one.clone(), bias_ids=ids, bias=bias, allowed=bits, keys=keys,
                                 out=torch.empty_like(L))),
    ]
    n = 0
    for fn, kw in calls:
        fn(**kw)
        for name, t in kw.items():
            if not torch.is_tensor(t):
                continue
            gone = t.clone()
            gone.untyped_storage().resize_(0)
            odd = [gone]
            if t.is_floating_point():
                odd += [torch._neg_view(t.clone()), t.to_sparse(), torch._efficientzerotensor(t.shape, dtype=t.dtype, device=cuda)]
            for o in odd:
                with pytest.raises(RuntimeError, match="memory|strided"):
                    fn(**{**kw, name: o})
                n += 1
    assert n > 100
    torch.cuda.synchronize()


@pytest.mark.parametrize("offset", [2 ** 31 - 64, 2 ** 31, 2 ** 63 - 1, 2 ** 63 - 64, -1])
def test_vocabulary_offsets_that_wrap_are_refused(cuda, offset):
    """Sums with 64-bit offsets do not wrap past the check (the mask would be read in front of its start)."""
    x, bits = torch.zeros(1, 64, device=cuda), torch.full((1, 4), -1, dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError, match="vocab_offset"):
        K.penalize_logits(x, allowed=bits, vocab_offset=offset)


@pytest.mark.parametrize("nq,nkv", [(2 ** 63 - 2, 2 ** 62 + 1), (2 ** 62, 2 ** 61), (2 ** 40, 1), (0, 1), (1, -1)])
def test_append_refuses_head_counts_that_wrap(cuda, nq, nkv):
    """(the first sums to zero in 64 bits, which would divide the process to its end)"""
    cos, sin = K.rotary_tables(8, 64, device=cuda)
    z = torch.zeros(1, dtype=torch.int32, device=cuda)
    kc = torch.zeros(2, 1, 16, 64, device=cuda)
    with pytest.raises(RuntimeError, match="nq and nkv"):
        K.qk_norm_rotary_append_kv(torch.zeros(1, 1, 256, device=cuda), z, cos, sin, z[None], z.clone(), torch.zeros(1, 1, 2, 64, device=cuda),
                                   kc, kc.clone(), nq, nkv)


def test_rotary_refuses_heads_whose_sums_wrap(cuda):
    cos, sin = K.rotary_tables(8, 2, device=cuda)
    pos, w = torch.zeros(1, dtype=torch.int32, device=cuda), torch.ones(2, device=cuda)
    x = torch.zeros(1, 1, 2, device=cuda)
    many = x.expand(1, 2 ** 31 - 1, 2)
    with pytest.raises(RuntimeError, match="heads"):
        K.rotary(many, pos, cos, sin)
    for q, k in ((many, x), (x, many)):
        with pytest.raises(RuntimeError, match="heads"):
            K.qk_norm_rotary(q, k, w, w, pos, cos, sin)


# ----------------------------------------------------------------------------------------------- huge scores
@pytest.mark.parametrize("dtype,mag", [(torch.float16, 2.0 ** 12), (torch.float16, 2.0 ** 15), (torch.bfloat16, 2.0 ** 13),
                                       (torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** 63)])
@pytest.mark.parametrize("D,T,G,ctx", [(64, 3, 2, [200]), (128, 40, 8, [3000, 130])])
def test_tree_attention_of_huge_scores(cuda, dtype, mag, D, T, G, ctx):
    """Scores up to 2^127, far past where fp32 resolves a unit: every row is the mean of the values of its largest keys.

    q has one component `mag`, keys one component 0.75, 1 or (two tokens a sequence) 1.5 times mag: scores of three values
    exact in fp32, at least mag^2 / 8 apart, so every weight but those of the largest is zero or one, exactly."""
    g = gen(cuda, D)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, len(ctx), T, G, 1, D, ctx, dtype)
    B = len(ctx)
    q.zero_()
    q[..., 7] = mag
    kc.zero_()
    n = max(ctx)
    level = 0.75 + 0.25 * (torch.rand(B, n, generator=g, device=cuda) < 0.5)
    want = torch.empty(B, D, dtype=torch.float64, device=cuda)
    for b in range(B):
        level[b, [3, ctx[b] - 2]] = 1.5
        at = torch.arange(ctx[b], device=cuda)
        kc[bt[b, at // 16].long(), 0, at % 16, 7] = (mag * level[b, :ctx[b]]).to(dtype)
        want[b] = (vc[bt[b, 0].long(), 0, 3].double() + vc[bt[b, (ctx[b] - 2) // 16].long(), 0, (ctx[b] - 2) % 16].double()) / 2
    for scale in (1.0, 0.125):
        y = K.tree_attention(q, kc, vc, bt, cl, bits, scale)
        ref = want[:, None, None].expand(y.shape)
        close(y, ref, 4 * F32U * (ref.abs() + float(vc.abs().max())))
