"""Numerics and refusals of the rotary, tree-attention and logits operators against 64-bit statements.

Tolerances count roundings: u(T) = half a step of the output type for the one rounding at the store, and multiples of
2^-24 of the terms' magnitudes for the fp32 arithmetic before it.
"""
import math

import pytest
import torch

from comm_opt_b200.ops import kernels as K

pytestmark = pytest.mark.gpu

F32U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):  # half a step of the subnormals
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def close(got, ref, fp32_err, scale=1.0):
    """|got - ref| <= one rounding to got's type + the fp32 error, elementwise; NaN and infinities in the same places."""
    d = got.dtype
    got, ref = got.double(), ref.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin) or bool((torch.isfinite(got) == fin).all())
    assert torch.equal(got[~fin].isnan(), ref[~fin].isnan())
    err = (got - ref).abs()
    tol = scale * (u(d) * ref.abs() + fp32_err * (1 + u(d)) + tiny(d))
    bad = fin & (err > tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off; worst {float((err / tol)[fin].max()):.3g} x tolerance"


def pairs(rot, interleaved, dev):
    j = torch.arange(rot // 2, device=dev)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)


def rotate64(x, cos, sin, interleaved, sign=1.0):
    """(rotated, magnitude of the terms) of x [.., H, D] float64; cos / sin [.., rot / 2] of its rows."""
    a, b = pairs(2 * cos.shape[-1], interleaved, x.device)
    c, s = cos.double().unsqueeze(-2), sign * sin.double().unsqueeze(-2)
    y, m = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    m[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    m[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, m


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, std=1.0):
    return (std * torch.randn(*shape, generator=g, device=g.device)).to(dtype)


# ---------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,H,D,rot", [(1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (3, 7, 4, 128, 64), (1, 33, 3, 80, 20),
                                         (2, 5, 2, 96, 24), (1, 4, 6, 256, 256), (2, 2, 1, 512, 128), (1, 9, 2, 130, 66),
                                         (4, 129, 40, 128, 128), (1, 3, 17, 64, 2), (64, 20, 64, 128, 128)])
def test_rotary(cuda, interleaved, dtype, B, S, H, D, rot):
    g = gen(cuda, D + rot)
    cos, sin = K.rotary_tables(50, rot, 1e4, device=cuda)
    x = randn(g, B, S, H, D, dtype=dtype)
    pos = torch.randint(0, 50, (B, S), generator=g, device=cuda, dtype=torch.int32)
    ref, mag = rotate64(x.double(), cos[pos.long()], sin[pos.long()], interleaved)
    y = K.rotary(x, pos, cos, sin, interleaved=interleaved)
    close(y, ref, 3 * F32U * mag)
    # views: heads of a wider row, a transposed batch, an unaligned start, an expanded operand
    wide = randn(g, B, S, H + 3, D, dtype=dtype)
    wide[:, :, 1:H + 1] = x
    assert torch.equal(K.rotary(wide[:, :, 1:H + 1], pos, cos, sin, interleaved=interleaved), y)
    tr = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(K.rotary(tr, pos, cos, sin, interleaved=interleaved), y)
    flat = torch.empty(x.numel() + 1, device=cuda, dtype=dtype)
    odd = flat[1:].view_as(x).copy_(x)
    assert torch.equal(K.rotary(odd, pos, cos, sin, interleaved=interleaved), y)
    ex = x[:, :, :1].expand(B, S, H, D)
    assert torch.equal(K.rotary(ex, pos, cos, sin, interleaved=interleaved), y[:, :, :1].expand(B, S, H, D))
    assert torch.equal(K.rotary(x.flatten(0, 1), pos.flatten(), cos, sin, interleaved=interleaved).view_as(y), y)
    # in place, into a view, back again
    z = x.clone()
    assert K.rotary(z, pos, cos, sin, interleaved=interleaved, out=z) is not None and torch.equal(z, y)
    o = torch.full((B, S, H + 1, D), 7.0, device=cuda, dtype=dtype)
    K.rotary(x, pos, cos, sin, interleaved=interleaved, out=o[:, :, 1:])
    assert torch.equal(o[:, :, 1:], y) and bool((o[:, :, 0] == 7).all())
    back = K.rotary(y, pos, cos, sin, interleaved=interleaved, inverse=True)
    rb, mb = rotate64(y.double(), cos[pos.long()], sin[pos.long()], interleaved, -1.0)
    close(back, rb, 3 * F32U * mb)


def test_rotary_rows_outside_the_tables_and_empty(cuda):
    cos, sin = K.rotary_tables(4, 64, device=cuda)
    x = torch.randn(6, 2, 64, device=cuda, requires_grad=True)
    pos = torch.tensor([0, -1, 3, 4, 2 ** 31 - 1, -2 ** 31], device=cuda, dtype=torch.int32)
    y = K.rotary(x, pos, cos, sin)
    y.sum().backward()
    for r in (1, 3, 4, 5):
        assert not bool(y[r].any()) and not bool(x.grad[r].any())
    assert bool(y[2].any()) and bool(x.grad[2].any())
    for shape in ((0, 2, 64), (3, 0, 64), (0, 4, 2, 64), (2, 0, 2, 64)):
        e = torch.zeros(shape, device=cuda)
        n = shape[0] if len(shape) == 3 else shape[1]
        assert K.rotary(e, torch.zeros(n, dtype=torch.int32, device=cuda), cos, sin).shape == shape


def test_rotary_passes_infinities_through(cuda):
    """Components that do not rotate are copies, and an infinity reaches its own pair only."""
    cos, sin = K.rotary_tables(9, 32, device=cuda)
    for inter in (False, True):
        x = torch.randn(3, 2, 64, device=cuda).bfloat16()
        x[0, 0, 40], x[1, 1, 63], x[2, 0, 3] = float("inf"), float("nan"), float("inf")
        y = K.rotary(x, torch.tensor([5, 6, 7], device=cuda, dtype=torch.int32), cos, sin, interleaved=inter)
        assert torch.equal(y[..., 32:].isnan(), x[..., 32:].isnan()) and y[0, 0, 40] == float("inf")
        odd = ~torch.isfinite(y[..., :32].float())
        mate = 2 if inter else 19
        assert odd.nonzero().tolist() == sorted([[2, 0, 3], [2, 0, mate]])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradients(cuda, interleaved):
    g = gen(cuda, 3)
    cos, sin = K.rotary_tables(40, 32, device=cuda)
    for dtype in DTYPES:
        x = randn(g, 2, 9, 3, 64, dtype=dtype).requires_grad_()
        pos = torch.arange(9, device=cuda, dtype=torch.int32)  # one row of positions for the batch
        dy = randn(g, 2, 9, 3, 64, dtype=dtype)
        (dx,) = torch.autograd.grad(K.rotary(x, pos, cos, sin, interleaved=interleaved), x, dy)
        ref, mag = rotate64(dy.double(), cos[:9], sin[:9], interleaved, -1.0)
        close(dx, ref, 3 * F32U * mag)
    # gradients that are expanded (a sum's) or transposed, an expanded operand, a gradient of the gradient
    x = randn(g, 2, 9, 1, 64).requires_grad_()
    K.rotary(x.expand(2, 9, 5, 64), pos, cos, sin, interleaved=interleaved).sum().backward()
    one, _ = rotate64(torch.ones(9, 1, 64, device=cuda, dtype=torch.float64), cos[:9], sin[:9], interleaved, -1.0)
    assert torch.allclose(x.grad.double(), 5 * one.expand(2, 9, 1, 64), atol=5 * 4 * F32U * 2)
    w = randn(g, 2, 9, 5, 64).requires_grad_()
    v = randn(g, 2, 9, 5, 64).requires_grad_()
    (d1,) = torch.autograd.grad(K.rotary(w, pos, cos, sin, interleaved=interleaved), w, v, create_graph=True)
    (d2,) = torch.autograd.grad(d1, v, torch.ones_like(d1))
    assert torch.equal(d2, K.rotary(torch.ones_like(w), pos, cos, sin, interleaved=interleaved).detach())


# ------------------------------------------------------------------------------------------- QK norm + rotary
def norm_rotate64(x, w, cos, sin, eps, interleaved):
    x, w = x.double(), w.double()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return rotate64(n, cos, sin, interleaved)


def norm_rotate_grad64(x, w, dy, cos, sin, eps, interleaved):
    """(dx, its terms' magnitude, dw, its terms' magnitude) by the formula."""
    x, w = x.double(), w.double()
    g, gm = rotate64(dy.double(), cos, sin, interleaved, -1.0)
    gm = torch.maximum(gm, g.abs())
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    h = x * r
    dx = r * (w * g - h * (w * g * h).mean(-1, keepdim=True))
    mag = r * (w.abs() * gm + h.abs() * (w.abs() * gm * h.abs()).mean(-1, keepdim=True))
    dims = tuple(range(x.dim() - 1))
    return dx, mag, (g * h).sum(dims), (gm * h.abs()).sum(dims)


SHAPES = [(1, 1, 1, 1, 64, 64), (2, 3, 8, 2, 128, 128), (2, 17, 5, 1, 128, 64), (3, 5, 4, 4, 80, 20), (1, 40, 6, 2, 96, 96),
          (2, 300, 32, 8, 128, 128), (1, 2, 3, 1, 256, 256), (1, 3, 2, 2, 6, 4), (2, 2, 2, 1, 512, 512)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,nq,nk,D,rot", SHAPES)
def test_qk_norm_rotary_and_gradients(cuda, interleaved, dtype, B, S, nq, nk, D, rot):
    g = gen(cuda, S + D)
    cos, sin = K.rotary_tables(S + 3, rot, 1e4, device=cuda)
    for wdtype in {dtype, torch.float32}:
        qkv = randn(g, B, S, nq + 2 * nk, D, dtype=dtype, std=2.0)
        q, k = qkv[:, :, :nq].detach().requires_grad_(), qkv[:, :, nq:nq + nk].detach().requires_grad_()
        wq, wk = (randn(g, D, dtype=wdtype) + 1).requires_grad_(), (randn(g, D, dtype=wdtype) + 1).requires_grad_()
        pos = torch.randint(0, S + 3, (B, S), generator=g, device=cuda, dtype=torch.int32)
        c, s = cos[pos.long()], sin[pos.long()]
        ys = K.qk_norm_rotary(q, k, wq, wk, pos, cos, sin, 1e-6, interleaved=interleaved)
        # relative error of a normalised component: the sum of D squares, the root, three products
        n32 = (D + 10) * F32U
        for y, x, w in zip(ys, (q, k), (wq, wk)):
            ref, mag = norm_rotate64(x.detach(), w.detach(), c, s, 1e-6, interleaved)
            close(y.detach(), ref, n32 * torch.maximum(mag, ref.abs()))
        dys = [randn(g, *y.shape, dtype=dtype) for y in ys]
        grads = torch.autograd.grad(ys, (q, k, wq, wk), dys)
        again = K.qk_norm_rotary_backward(*dys, q, k, wq, wk, pos, cos, sin, 1e-6, interleaved=interleaved)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))  # a fixed order of the sums
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            dx, mag, dw, wmag = norm_rotate_grad64(x.detach(), w.detach(), dys[i], c, s, 1e-6, interleaved)
            close(grads[i], dx, (3 * D + 20) * F32U * mag)
            rows = x.numel() // D
            close(grads[2 + i], dw, (rows + D + 20) * F32U * wmag)


def test_qk_norm_rotary_gradient_by_differences(cuda):
    """The kernel's gradient against central differences of the 64-bit formula."""
    g = gen(cuda, 9)
    D, eps = 64, 1e-5
    cos, sin = K.rotary_tables(8, D, device=cuda)
    q, k = randn(g, 1, 4, 2, D), randn(g, 1, 4, 1, D)
    wq, wk = randn(g, D) + 1, randn(g, D) + 1
    pos = torch.tensor([0, 3, 5, 7], device=cuda, dtype=torch.int32)
    c, s = cos[pos.long()], sin[pos.long()]
    dq, dk = randn(g, *q.shape), randn(g, *k.shape)
    gq, gk, gwq, gwk = K.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, pos, cos, sin, eps)

    def f(x, w, dy):
        return float((norm_rotate64(x, w, c, s, eps, False)[0] * dy.double()).sum())

    h = 1e-5
    for x, w, dy, gx, gw in ((q, wq, dq, gq, gwq), (k, wk, dk, gk, gwk)):
        for _ in range(3):
            e = torch.randn(x.shape, generator=g, device=cuda, dtype=torch.float64)
            num = (f(x.double() + h * e, w, dy) - f(x.double() - h * e, w, dy)) / (2 * h)
            # the differences' own error is h^2; the kernel's is fp32
            assert abs(num - float((gx.double() * e).sum())) <= 1e-4 * float((gx.double() * e).abs().sum())
            e = torch.randn(D, generator=g, device=cuda, dtype=torch.float64)
            num = (f(x, w.double() + h * e, dy) - f(x, w.double() - h * e, dy)) / (2 * h)
            assert abs(num - float((gw.double() * e).sum())) <= 1e-4 * float((gw.double() * e).abs().sum())


def test_qk_norm_rotary_zero_rows_and_padding(cuda):
    """A row of zeros stays finite (eps), a padded row (position -1) gives zeros and adds nothing to any gradient."""
    g = gen(cuda, 1)
    cos, sin = K.rotary_tables(4, 64, device=cuda)
    q, k = randn(g, 3, 2, 64), randn(g, 3, 1, 64)
    q[1], k[1] = 0, 0
    q[2], k[2] = float("nan"), float("inf")  # what padding may hold
    w = torch.ones(64, device=cuda)
    pos = torch.tensor([1, 2, -1], device=cuda, dtype=torch.int32)
    yq, yk = K.qk_norm_rotary(q, k, w, w, pos, cos, sin, 1e-6)
    assert not bool(yq[1:].any()) and not bool(yk[1:].any())
    dq, dk = randn(g, 3, 2, 64), randn(g, 3, 1, 64)
    dq[2] = float("nan")
    got = K.qk_norm_rotary_backward(dq, dk, q, k, w, w, pos, cos, sin, 1e-6)
    want = K.qk_norm_rotary_backward(dq[:2], dk[:2], q[:2], k[:2], w, w, pos[:2], cos, sin, 1e-6)
    assert torch.equal(got[0][:2], want[0]) and not bool(got[0][2].any()) and not bool(got[1][2].any())
    for a, b in zip(got[2:], want[2:]):
        assert bool(torch.isfinite(a).all())
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("interleaved,norm,bias", [(False, True, False), (True, True, True), (False, False, True), (True, False, False)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,nq,nkv,D,rot", [(1, 1, 8, 1, 128, 128), (8, 1, 32, 8, 128, 64), (3, 37, 5, 1, 128, 128),
                                              (2, 20, 4, 4, 64, 64), (2, 6, 3, 1, 80, 20)])
def test_append(cuda, interleaved, norm, bias, dtype, B, S, nq, nkv, D, rot):
    g = gen(cuda, B * S + D)
    n, pages = nq + 2 * nkv, (S + 40 + 15) // 16
    cos, sin = K.rotary_tables(S + 60, rot, 1e4, device=cuda)
    wide = randn(g, B, S, n * D + 16, dtype=dtype)
    qkv = wide[..., :n * D]
    starts = torch.randint(0, 41, (B,), generator=g, device=cuda, dtype=torch.int32)
    lens = torch.randint(0, S + 1, (B,), generator=g, device=cuda, dtype=torch.int32)
    lens[0] = S
    pos = torch.randint(0, S + 60, (B, S), generator=g, device=cuda, dtype=torch.int32)
    bt = torch.randperm(B * pages, generator=g, device=cuda).to(torch.int32).view(B, pages)
    kc = randn(g, B * pages, nkv, 16, D, dtype=dtype)
    vc = randn(g, B * pages, nkv, 16, D, dtype=dtype)
    wq, wk = (1 + 0.1 * randn(g, D)).to(dtype), (1 + 0.1 * randn(g, D)).to(dtype)
    bv = randn(g, n * D, dtype=dtype) if bias else None
    q_out = torch.full((B, S, nq, D), 3.0, device=cuda, dtype=dtype)
    k1, v1 = kc.clone(), vc.clone()
    K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, starts, q_out, k1, v1, nq, nkv, q_weight=wq if norm else None,
                               k_weight=wk if norm else None, eps=1e-5, lens=lens, bias=bv, interleaved=interleaved)
    x = qkv.double() + (bv.double() if bias else 0)
    x = x.view(B, S, n, D)
    c, s = cos[pos.long()], sin[pos.long()]
    parts = []
    for t, w in ((x[:, :, :nq], wq), (x[:, :, nq:nq + nkv], wk)):
        if norm:
            r, m = norm_rotate64(t, w, c, s, 1e-5, interleaved)
        else:
            r, m = rotate64(t, c, s, interleaved)
        # a bias enters with one more rounding, of terms as large as |x| + |bias| <= 2 max
        parts.append((r, torch.maximum(m, r.abs())))
    extra = 4 * F32U * (float(x.abs().max()) + 1) * 3
    n32 = ((D + 14) if norm else 4) * F32U
    live = torch.arange(S, device=cuda)[None] < lens[:, None]
    close(q_out[live], parts[0][0][live], n32 * parts[0][1][live] + (extra if bias else 0))
    assert bool((q_out[~live] == 3).all())
    touched = torch.zeros(B * pages, 16, dtype=torch.bool, device=cuda)
    for b in range(B):
        at = int(starts[b]) + torch.arange(int(lens[b]), device=cuda)
        pg, off = bt[b].long()[at // 16], at % 16
        close(k1[pg, :, off], parts[1][0][b, :int(lens[b])], n32 * parts[1][1][b, :int(lens[b])] + (extra if bias else 0))
        close(v1[pg, :, off], x[b, :int(lens[b]), nq + nkv:], extra if bias else 0)
        touched[pg, off] = True
    rest = ~touched[:, None].expand(-1, nkv, -1)
    assert torch.equal(k1[rest], kc[rest]) and torch.equal(v1[rest], vc[rest])


def test_append_equals_the_decode_append(cuda):
    """Without norms, half layout, one token: rope_append_kv up to the fp32 roundings before the store (at most one
    step of the type apart); v and the places are the same bits."""
    g = gen(cuda, 5)
    B, nq, nkv, D = 5, 8, 2, 128
    cos, sin = K.rotary_tables(64, D, 500000.0, device=cuda)
    qkv = randn(g, B, (nq + 2 * nkv) * D, dtype=torch.bfloat16)
    pos = torch.tensor([0, 17, 33, 63, 48], device=cuda, dtype=torch.int32)
    bt = torch.randperm(20, generator=g, device=cuda).to(torch.int32).view(5, 4)
    c = [torch.zeros(20, nkv, 16, D, device=cuda, dtype=torch.bfloat16) for _ in range(4)]
    qa, qb = (torch.empty(B, nq, D, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    K.rope_append_kv(qkv, pos, cos, sin, bt, qa, c[0], c[1], nq, nkv)
    K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, pos, qb, c[2], c[3], nq, nkv)
    assert torch.equal(c[1], c[3])
    big = 3 * F32U * float(qkv.float().abs().max())  # of either side's terms
    for a, b in ((qa, qb), (c[0], c[2])):
        a, b = a.double(), b.double()
        assert bool(((a - b).abs() <= 2 * u(torch.bfloat16) * a.abs() * (1 + u(torch.bfloat16)) + 2 * big).all())


def test_append_bad_slots_and_pages(cuda):
    """Rows whose slot lies past the table, before the cache or on a page that does not exist write nothing."""
    D, nq, nkv = 64, 2, 1
    cos, sin = K.rotary_tables(100, D, device=cuda)
    qkv = torch.randn(5, 3, 4 * D, device=cuda).half()
    bt = torch.tensor([[0, 1], [2, 99], [-1, 3], [4, 5], [6, 7]], device=cuda, dtype=torch.int32)
    starts = torch.tensor([30, 15, 0, -2, 2 ** 31 - 2], device=cuda, dtype=torch.int32)
    pos = torch.tensor([[0, 1, 2]] * 5, device=cuda, dtype=torch.int32)
    pos[0, 0] = 100  # outside the tables
    kc, vc = torch.zeros(8, nkv, 16, D, device=cuda).half(), torch.zeros(8, nkv, 16, D, device=cuda).half()
    q = torch.zeros(5, 3, nq, D, device=cuda).half()
    K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, starts, q, kc, vc, nq, nkv)
    used = vc.abs().sum((1, 3)).nonzero().tolist()
    assert used == [[1, 15], [2, 15]]  # slot 31 of sequence 0 (30 lost its position), slot 15 of sequence 1
    assert not bool(q[0, 0].any()) and bool(q[4].any()) and bool(q[3].any())


# ------------------------------------------------------------------------------------------- tree attention
def tree_ref(q, kc, vc, bt, ctx, bits, scale, tree_lens=None):
    """(output, sum p |v| / sum p, largest |q k| sum) in 64 bits; rows past tree_lens are NaN."""
    B, T, nq, D = q.shape
    nkv = kc.shape[1]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    mag, sm = torch.zeros_like(out), torch.zeros(B, T, nq, 1, dtype=torch.float64, device=q.device)
    for b in range(B):
        tl = T if tree_lens is None else min(T, int(tree_lens[b]))
        cap = bt.shape[1] * 16
        n = min(int(ctx[b]), cap)
        L = min(n + tl, cap)
        at = torch.arange(L, device=q.device)
        pg = bt[b].long()[at // 16]
        bad = (pg < 0) | (pg >= kc.shape[0])
        pg = pg.clamp(0, kc.shape[0] - 1)
        k, v = kc[pg, :, at % 16].double(), vc[pg, :, at % 16].double()
        k[bad], v[bad] = 0, 0
        for t in range(tl):
            see = torch.tensor([s < n or bool((bits[b][t] >> (s - n)) & 1) for s in range(max(L - 80, 0), L)],
                               dtype=torch.bool, device=q.device)
            idx = torch.cat([torch.arange(max(L - 80, 0), device=q.device), max(L - 80, 0) + see.nonzero()[:, 0]])
            kk = k[idx].repeat_interleave(nq // nkv, 1)
            vv = v[idx].repeat_interleave(nq // nkv, 1)
            qq = q[b, t].double()
            s = torch.einsum("hd,shd->hs", qq, kk) * scale
            if len(idx) == 0:
                out[b, t] = 0
                continue
            p = torch.softmax(s, -1)
            out[b, t] = torch.einsum("hs,shd->hd", p, vv)
            mag[b, t] = torch.einsum("hs,shd->hd", p, vv.abs())
            sm[b, t] = (torch.einsum("hd,shd->hs", qq.abs(), kk.abs()) * scale).max(-1).values[:, None]
    return out, mag, sm


def check_tree(got, ref, mag, sm, n, D):
    """The weights are rounded to the cache's type before their product with v (u of them, in the numerator only);
    a score is off by (D + 8) roundings of its terms, its weight by twice that; sums over n slots are fp32."""
    d = got.dtype
    live = ~ref.isnan()
    err32 = (2 * (D + 8) * F32U * sm + (n + 32) * F32U + u(d)) * mag
    close(got[live], ref[live], err32[live])


def make_tree(g, dev, B, T, nq, nkv, D, ctx, dtype, bits=None):
    pages = (max(ctx) + T + 15) // 16 + 1
    kc = randn(g, B * pages + 2, nkv, 16, D, dtype=dtype)
    vc = randn(g, B * pages + 2, nkv, 16, D, dtype=dtype)
    bt = torch.randperm(B * pages + 2, generator=g, device=dev)[:B * pages].to(torch.int32).view(B, pages)
    q = randn(g, B, T, nq, D, dtype=dtype)
    par = (torch.rand(B, T, generator=g, device=dev) * (torch.arange(T, device=dev) + 1)).long() - 1
    return q, kc, vc, bt, torch.tensor(ctx, dtype=torch.int32, device=dev), K.tree_mask(par)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,nq,nkv,D,ctx", [
    (1, 1, 1, 1, 64, [0]), (1, 1, 8, 1, 128, [1]), (3, 5, 8, 2, 128, [0, 15, 16]), (2, 8, 5, 1, 128, [127, 300]),
    (2, 64, 8, 1, 128, [113, 64]), (1, 63, 4, 4, 64, [1000]), (4, 17, 16, 2, 64, [5, 128, 129, 2500]),
    (2, 33, 16, 1, 128, [700, 3]), (1, 64, 64, 8, 128, [513]), (2, 9, 64, 1, 128, [4100, 77]), (9, 3, 4, 1, 128, [50 * i for i in range(9)])])
def test_tree_attention(cuda, dtype, B, T, nq, nkv, D, ctx):
    g = gen(cuda, B + T + D)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, B, T, nq, nkv, D, ctx, dtype)
    scale = 1 / math.sqrt(D)
    host = bits.tolist()
    ref, mag, sm = tree_ref(q, kc, vc, bt, cl, host, scale)
    y = K.tree_attention(q, kc, vc, bt, cl, bits, scale)
    check_tree(y, ref, mag, sm, max(ctx) + T, D)
    assert torch.equal(K.tree_attention(q, kc, vc, bt, cl, bits, scale), y)  # a fixed order of the sums
    # q as heads of a wider projection row; an output view; one mask for all
    wide = torch.zeros(B, T, nq + 2 * nkv, D, device=cuda, dtype=dtype)
    wide[:, :, :nq] = q
    o = torch.full((B, T, nq + 1, D), 5.0, device=cuda, dtype=dtype)
    K.tree_attention(wide[:, :, :nq], kc, vc, bt, cl, bits, scale, out=o[:, :, 1:])
    assert torch.equal(o[:, :, 1:], y) and bool((o[:, :, 0] == 5).all())
    ch = K.tree_attention(q, kc, vc, bt, cl, None, scale)
    one = K.tree_mask(torch.arange(T, device=cuda) - 1)
    assert torch.equal(ch, K.tree_attention(q, kc, vc, bt, cl, one, scale))
    ref, mag, sm = tree_ref(q, kc, vc, bt, cl, [one.tolist()] * B, scale)
    check_tree(ch, ref, mag, sm, max(ctx) + T, D)


def test_tree_attention_padding_empty_rows_and_garbage(cuda):
    """Rows past tree_lens keep what out held; rows that see nothing are zeros; stale, infinite and NaN contents of
    slots that are not seen (pages behind the last token, siblings, padding tokens) reach nothing."""
    for D, T, nq, dtype in ((128, 12, 8, torch.bfloat16), (64, 40, 4, torch.float16), (128, 30, 16, torch.float16)):
        g = gen(cuda, D + T)
        ctx = [0, 0, 37, 250, 128]
        q, kc, vc, bt, cl, bits = make_tree(g, cuda, 5, T, nq, 1, D, ctx, dtype)
        tl = torch.tensor([T, 3, 0, T - 1, 1], dtype=torch.int32, device=cuda)
        bits[0, 2] = 0  # sees nothing at all
        bits[3, 4] = 0  # sees the cache only
        want = K.tree_attention(q, kc, vc, bt, cl, bits, 0.1, tree_lens=tl)
        ref, mag, sm = tree_ref(q, kc, vc, bt, cl, bits.tolist(), 0.1, tl)
        check_tree(want, ref, mag, sm, 250 + T, D)
        assert not bool(want[0, 2].any())
        for fill in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
            k2, v2 = kc.clone(), vc.clone()
            live = torch.zeros(kc.shape[0], 16, dtype=torch.bool, device=cuda)
            for b in range(5):
                at = torch.arange(ctx[b] + int(tl[b]), device=cuda)
                live[bt[b].long()[at // 16], at % 16] = True
            dead = ~live[:, None].expand(-1, 1, -1)
            k2[dead], v2[dead] = fill, fill
            out = torch.full_like(q, 9.0)
            K.tree_attention(q, k2, v2, bt, cl, bits, 0.1, tree_lens=tl, out=out)
            for b in range(5):
                assert torch.equal(out[b, :int(tl[b])], want[b, :int(tl[b])]), (fill, b)
                assert bool((out[b, int(tl[b]):] == 9).all())
            # one drafted token's own k or v is not finite: rows that do not see it keep their bits
            for which in (0, 1):
                k3, v3 = kc.clone(), vc.clone()
                slot = ctx[3] + 2
                (k3 if which == 0 else v3)[bt[3].long()[slot // 16], :, slot % 16] = fill
                got = K.tree_attention(q, k3, v3, bt, cl, bits, 0.1, tree_lens=tl)
                sees = ((bits[3] >> 2) & 1).bool()
                sees[int(tl[3]):] = False
                keep = ~sees
                assert torch.equal(got[3][keep], want[3][keep]), (fill, which)
                if math.isnan(fill):
                    assert bool(got[3][sees].isnan().all())
                if math.isinf(fill) and which == 1:
                    assert bool((got[3][sees] == fill).all())


def test_tree_attention_bad_pages_and_lengths(cuda):
    """Page indexes outside the cache read as zeros, lengths past the table are cut, negative ones are zero."""
    g = gen(cuda, 2)
    D, T, nq = 64, 6, 4
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, 4, T, nq, 2, D, [40, 200, 100, 90], torch.float16)
    bt[0, 1], bt[1, 3], bt[1, 4] = -1, kc.shape[0], 2 ** 31 - 1
    cl[2], cl[3] = 10 ** 9, -5
    y = K.tree_attention(q, kc, vc, bt, cl, bits, 0.125)
    assert bool(torch.isfinite(y).all())
    fixed = cl.clone()
    fixed[2], fixed[3] = bt.shape[1] * 16, 0
    ref, mag, sm = tree_ref(q, kc, vc, bt, fixed, bits.tolist(), 0.125)
    check_tree(y, ref, mag, sm, 300, D)


def test_tree_attention_large_scores(cuda):
    """Scores that rise along the cache by far more than the type's range of exponentials."""
    g = gen(cuda, 4)
    q, kc, vc, bt, cl, bits = make_tree(g, cuda, 1, 24, 8, 1, 128, [900], torch.bfloat16)
    at = torch.arange(924, device=cuda)
    kc[bt[0].long()[at // 16], 0, at % 16] = (at[:, None] / 924 * q[0, 3, 2].float()).to(torch.bfloat16)
    for scale in (1.0, -1.0):
        ref, mag, sm = tree_ref(q, kc, vc, bt, cl, bits.tolist(), scale)
        check_tree(K.tree_attention(q, kc, vc, bt, cl, bits, scale), ref, mag, sm, 924, 128)


# -------------------------------------------------------------------------------------------------- logits
def logits_ref(x, off, tokens=None, lens=None, plens=None, rep=None, freq=None, pres=None, ids=None, bias=None, allowed=None,
               dtype=torch.float64):
    """(result, magnitude of its terms), each step rounded to `dtype`; entry by entry on the host."""
    B, V = x.shape
    dev = x.device
    y = x.to(dtype).cpu()
    mag = y.abs().double()
    one = torch.ones((), dtype=dtype)
    for b in range(B):
        seen, count = {}, {}
        if tokens is not None:
            n = tokens.shape[1] if lens is None else max(0, min(int(lens[b]), tokens.shape[1]))
            p = 0 if plens is None else int(plens[b])
            for i, t in enumerate(tokens[b, :n].tolist()):
                v = t - off
                if 0 <= v < V:
                    seen[v] = True
                    if i >= p:
                        count[v] = count.get(v, 0) + 1
        for v in seen:
            if rep is not None:
                r = rep[b].cpu().to(dtype)
                y[b, v] = y[b, v] / r if y[b, v] > 0 else y[b, v] * r
                mag[b, v] = torch.maximum(mag[b, v], y[b, v].abs().double())
            c = count.get(v, 0)
            if c and freq is not None:
                d = freq[b].cpu().to(dtype) * (c * one)
                y[b, v] = y[b, v] - d
                mag[b, v] += d.abs().double()
            if c and pres is not None:
                y[b, v] = y[b, v] - pres[b].cpu().to(dtype)
                mag[b, v] += pres[b].cpu().abs().double()
        if ids is not None:
            add = {}
            for t, w in zip(ids[b].tolist(), bias[b].cpu().to(dtype)):
                v = t - off
                if 0 <= v < V:
                    add[v] = add.get(v, torch.zeros((), dtype=dtype)) + w
                    mag[b, v] += w.abs().double()
            for v, w in add.items():
                y[b, v] = y[b, v] + w
        if allowed is not None:
            words = allowed[b].cpu().to(torch.int64) & 0xFFFFFFFF
            gi = torch.arange(V) + off
            y[b, ((words[gi // 32] >> (gi % 32)) & 1) == 0] = float("-inf")
    return y.to(dev), mag.to(dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V,L,nb,off", [(1, 1, 3, 1, 0), (3, 7, 20, 5, 0), (2, 1000, 300, 40, 0), (5, 4097, 64, 70, 33),
                                          (4, 16032, 2000, 300, 16032), (2, 50257, 500, 0, 0), (1, 33, 0, 2, 5)])
def test_penalize_logits(cuda, dtype, B, V, L, nb, off):
    g = gen(cuda, V + B)
    x = randn(g, B, V, dtype=dtype, std=3.0)
    total = off + V + 10
    words = (total + 31) // 32

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=cuda, dtype=torch.int32)

    tokens = ri(-2, min(total, off + 400), B, L + 3)[:, 1:L + 1]  # a view with a longer row, ids of other shards, padding
    lens, plens = ri(0, L + 1, B), ri(0, L + 1, B)
    rep, freq, pres = (1 + torch.rand(B, generator=g, device=cuda) for _ in range(3))
    ids, bias = ri(-1, total, B, nb), randn(g, B, nb)
    if nb > 2:
        ids[:, 1:3] = ids[:, :1]  # one id three times
        bias[0, 0] = float("-inf")
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, words + 1), generator=g, device=cuda).to(torch.int32)[:, :words]
    forms = [dict(), dict(tokens=tokens, repetition=rep), dict(tokens=tokens, lens=lens, prompt_lens=plens, repetition=rep,
             frequency=freq, presence=pres), dict(bias_ids=ids, bias=bias), dict(allowed=allowed),
             dict(tokens=tokens, lens=lens, frequency=freq, presence=pres, bias_ids=ids, bias=bias, allowed=allowed)]
    names = dict(prompt_lens="plens", repetition="rep", frequency="freq", presence="pres", bias_ids="ids")
    for f in forms:
        y = K.penalize_logits(x, vocab_offset=off, **f)
        kw = {names.get(k, k): v for k, v in f.items()}
        ref, mag = logits_ref(x, off, **kw)
        close(y, ref, 6 * F32U * mag)
        same, _ = logits_ref(x, off, dtype=torch.float32, **kw)  # the same steps in fp32, rounded once: the same bits
        assert torch.equal(y, same.to(dtype))
        keys = torch.zeros(B, dtype=torch.int64, device=cuda)
        z = x.clone()
        K.penalize_logits(z, vocab_offset=off, out=z, keys=keys, **f)  # in place, with the greedy keys
        assert torch.equal(z, y)
        assert torch.equal(keys, K.argmax_local(y, off))
        pad = torch.full((B, V + 3), 7.0, device=cuda, dtype=dtype)
        src = torch.full((B, V + 5), 1.0, device=cuda, dtype=dtype)
        src[:, 2:V + 2] = x
        K.penalize_logits(src[:, 2:V + 2], vocab_offset=off, out=pad[:, 1:V + 1], **f)
        assert torch.equal(pad[:, 1:V + 1], y) and bool((pad[:, 0] == 7).all()) and bool((pad[:, V + 1:] == 7).all())


def test_penalize_logits_last_ids(cuda):
    """Ids up to 2^31 - 2: the mask's last word is the row's last, and ids below zero do not wrap into the shard."""
    V, words = 101, 1 << 26
    off = 2 ** 31 - 1 - V
    g = gen(cuda, 9)
    x = randn(g, 1, V, dtype=torch.float32)
    allowed = torch.zeros(1, words, dtype=torch.int32, device=cuda)
    bits = torch.rand(V, generator=g, device=cuda) < 0.6
    bits[-2:] = torch.tensor([True, False], device=cuda)
    for v in bits.nonzero()[:, 0].tolist():
        one = 1 << ((off + v) % 32)
        allowed[0, (off + v) // 32] |= one - (1 << 32) if one >> 31 else one
    tokens = torch.tensor([[off + V - 2, off, off - 1, -1, -2 ** 31, 2 ** 31 - 1, 0]], dtype=torch.int32, device=cuda)
    pres = torch.ones(1, device=cuda)
    keys = torch.zeros(1, dtype=torch.int64, device=cuda)
    y = K.penalize_logits(x, vocab_offset=off, allowed=allowed, tokens=tokens, presence=pres, bias_ids=tokens,
                          bias=torch.full((1, 7), 0.5, device=cuda), keys=keys)
    ref = x.clone()
    ref[0, [0, V - 2]] = ref[0, [0, V - 2]] - 1.0 + 0.5
    ref[0, ~bits] = float("-inf")
    assert torch.equal(y, ref)
    assert torch.equal(keys, K.argmax_local(y, off))
    # the mask as the last row of a tensor that ends with it, at every alignment of the shard in its words
    for v0 in range(33):
        y = K.penalize_logits(x[:, v0:], vocab_offset=off + v0, allowed=allowed)
        assert torch.equal(y[0], torch.where(bits, x[0], float("-inf"))[v0:])


def test_penalize_logits_special_values(cuda):
    x = torch.tensor([[float("inf"), -float("inf"), float("nan"), 0.0, -0.0, torch.finfo(torch.bfloat16).min]], device=cuda).bfloat16()
    t = torch.tensor([[0, 1, 2, 3, 4, 5]], device=cuda, dtype=torch.int32)
    r = torch.tensor([2.0], device=cuda)
    y = K.penalize_logits(x, tokens=t, repetition=r, frequency=r, presence=r)[0].float().tolist()
    assert y[0] == float("inf") and y[1] == -float("inf") and math.isnan(y[2]) and y[3] == y[4] == -4.0
    assert y[5] == -float("inf")  # past the type's lowest value
    # a grammar that allows nothing, and one that allows one id
    none = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    none[1] = 16
    keys = torch.zeros(2, dtype=torch.int64, device=cuda)
    z = K.penalize_logits(x.expand(2, 6), allowed=none, keys=keys)
    assert bool((z[0] == -float("inf")).all()) and z[1, 4] == 0
    assert K.argmax_combine(keys.view(1, 2), 1).tolist() == [0, 4]


# ------------------------------------------------------------------------------- a run of them together, graphs
def _step_inputs(dev, dtype=torch.bfloat16, seed=0):
    g = gen(dev, seed)
    B, T, nq, nkv, D, V = 3, 7, 8, 2, 128, 4096
    ctx = [5, 60, 130]
    q, kc, vc, bt, cl, _ = make_tree(g, dev, B, T, nq, nkv, D, ctx, dtype)
    par = torch.tensor([[-1, 0, 0, 1, 1, 2, 5]] * B, device=dev)
    depth = torch.tensor([0, 1, 1, 2, 2, 2, 3], device=dev, dtype=torch.int32)
    st = dict(qkv=randn(g, B, T, (nq + 2 * nkv) * D, dtype=dtype), kc=kc, vc=vc, bt=bt, cl=cl, mask=K.tree_mask(par),
              pos=(cl[:, None] + depth).contiguous(), tl=torch.tensor([7, 4, 6], dtype=torch.int32, device=dev),
              wq=(1 + 0.1 * randn(g, D)).to(dtype), wk=(1 + 0.1 * randn(g, D)).to(dtype), q=torch.zeros(B, T, nq, D, device=dev, dtype=dtype),
              o=torch.zeros(B, T, nq, D, device=dev, dtype=dtype), head=randn(g, V, nq * D, dtype=dtype, std=0.05),
              tok=torch.randint(0, V, (B * T, 50), generator=g, device=dev, dtype=torch.int32),
              rep=1 + torch.rand(B * T, generator=g, device=dev),
              allowed=torch.randint(-2 ** 31, 2 ** 31, (B * T, V // 32), generator=g, device=dev).to(torch.int32),
              keys=torch.zeros(B * T, dtype=torch.int64, device=dev), ids=torch.zeros(B * T, dtype=torch.int32, device=dev),
              logits=torch.empty(B * T, V, device=dev, dtype=dtype))
    st["cos"], st["sin"] = K.rotary_tables(300, D, 500000.0, device=dev)
    return st


def _verify_step(s):
    """One verification step of drafted trees: append, attention, head, logits, greedy choice."""
    K.qk_norm_rotary_append_kv(s["qkv"], s["pos"], s["cos"], s["sin"], s["bt"], s["cl"], s["q"], s["kc"], s["vc"], 8, 2,
                               q_weight=s["wq"], k_weight=s["wk"], lens=s["tl"])
    K.tree_attention(s["q"], s["kc"], s["vc"], s["bt"], s["cl"], s["mask"], 128 ** -0.5, tree_lens=s["tl"], out=s["o"])
    torch.matmul(s["o"].view(21, -1), s["head"].t(), out=s["logits"])
    K.penalize_logits(s["logits"], tokens=s["tok"], repetition=s["rep"], allowed=s["allowed"], out=s["logits"], keys=s["keys"])
    K.argmax_combine(s["keys"].view(1, -1), 1, ids=s["ids"], local_keys=s["keys"])


def test_verification_step(cuda):
    """Append, tree attention, logits and greedy choice in sequence equal their statements in sequence, each tree path
    equals decoding its tokens one by one, and a captured step replays to the same bits."""
    s = _step_inputs(cuda)
    k0, v0 = s["kc"].clone(), s["vc"].clone()
    _verify_step(s)
    ids, out = s["ids"].clone(), s["o"].clone()
    ref, mag, sm = tree_ref(s["q"], s["kc"], s["vc"], s["bt"], s["cl"], s["mask"].tolist(), 128 ** -0.5, s["tl"])
    check_tree(out, torch.where(ref.isnan(), ref, ref), mag, sm, 140, 128)
    live = (torch.arange(7, device=cuda)[None] < s["tl"][:, None]).flatten()
    x = torch.matmul(s["o"].view(21, -1), s["head"].t())
    want, _ = logits_ref(x, 0, tokens=s["tok"], rep=s["rep"], allowed=s["allowed"], dtype=torch.float32)
    assert torch.equal(want.bfloat16(), s["logits"])
    assert torch.equal(ids, s["logits"].float().argmax(-1).to(torch.int32)) and not bool(s["keys"].any())
    # the path 0 -> 1 -> 4 of sequence 2, token by token through the single-token forms
    kc, vc = k0.clone(), v0.clone()
    for step, node in enumerate((0, 1, 4)):
        q1 = torch.zeros(1, 1, 8, 128, device=cuda, dtype=torch.bfloat16)
        at = (s["cl"][2:] + step).to(torch.int32)
        K.qk_norm_rotary_append_kv(s["qkv"][2:, node:node + 1], at, s["cos"], s["sin"], s["bt"][2:], at, q1, kc, vc, 8, 2,
                                   q_weight=s["wq"], k_weight=s["wk"])
        assert torch.equal(q1[0, 0], s["q"][2, node])
        o1 = torch.empty(1, 8, 128, device=cuda, dtype=torch.bfloat16)
        K.DecodeAttention(1, 8, 2, 128, s["bt"].shape[1], cuda)(q1[0], kc, vc, s["bt"][2:], at + 1, o1, 128 ** -0.5)
        o2 = K.tree_attention(q1, kc, vc, s["bt"][2:], at, None, 128 ** -0.5)
        for o in (o1[0], o2[0, 0]):
            r, m, z = ref[2, node], mag[2, node], sm[2, node]
            check_tree(o, r, m, z, 140, 128)
    # graph
    s2 = _step_inputs(cuda)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _verify_step(s2)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _verify_step(s2)
    for _ in range(3):
        s2["kc"].copy_(k0)
        s2["vc"].copy_(v0)
        s2["o"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s2["ids"], ids) and torch.equal(s2["o"], out)
        assert torch.equal(s2["kc"], s["kc"]) and torch.equal(s2["vc"], s["vc"])
    assert bool(live.any())


def test_two_streams_and_two_graphs(cuda):
    """Calls in flight at once on two streams, and two captured graphs replayed together, share nothing."""
    g = gen(cuda, 8)
    a = make_tree(g, cuda, 2, 16, 16, 2, 128, [3000, 2000], torch.bfloat16)
    b = make_tree(g, cuda, 2, 16, 16, 2, 128, [2500, 3500], torch.bfloat16)
    qa, ka = randn(g, 2, 200, 8, 128), randn(g, 2, 200, 2, 128)
    w = torch.ones(128, device=cuda)
    cos, sin = K.rotary_tables(200, 128, device=cuda)
    pos = torch.arange(200, device=cuda, dtype=torch.int32)

    def work(t):
        return (K.tree_attention(*t, 0.09), *K.qk_norm_rotary_backward(qa, ka, qa, ka, w, w, pos, cos, sin))

    want = work(a), work(b)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in (a, b):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(t))
        graphs.append(gr)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        for st, gr in ((s1, graphs[0]), (s2, graphs[1])):
            with torch.cuda.stream(st):
                gr.replay()
    got = []
    for st, t in ((s1, a), (s2, b)):
        with torch.cuda.stream(st):
            got.append([work(t) for _ in range(5)])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for x, y in zip(outs[i], want[i]))
        for r in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[i]))


def test_programmatic_launch_keeps_the_results(cuda):
    s = _step_inputs(cuda, seed=3)
    k0, v0 = s["kc"].clone(), s["vc"].clone()
    _verify_step(s)
    want = [s[n].clone() for n in ("ids", "o", "kc", "vc")]
    old = K.set_pdl(True)
    try:
        for _ in range(10):
            s["kc"].copy_(k0)
            s["vc"].copy_(v0)
            _verify_step(s)
        torch.cuda.synchronize()
    finally:
        K.set_pdl(old)
    assert all(torch.equal(s[n], w) for n, w in zip(("ids", "o", "kc", "vc"), want))


def test_caches_past_32_bit_offsets(cuda):
    """Pages whose elements lie beyond 2^31: appended to and attended like the same pages of a small cache."""
    g = gen(cuda, 21)
    nkv, D, B, T = 8, 128, 2, 5
    blocks = 2 ** 31 // (nkv * 16 * D) + 40
    kc = torch.zeros(blocks, nkv, 16, D, device=cuda, dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    far = torch.arange(blocks - 32, blocks, device=cuda).view(B, 16).to(torch.int32)
    near = torch.arange(32, device=cuda).view(B, 16).to(torch.int32)
    ks, vs = kc[:32].clone(), vc[:32].clone()
    rand = randn(g, 32, nkv, 16, D, dtype=torch.bfloat16)
    kc[-32:], vc[-32:], ks[:], vs[:] = rand, rand.flip(0), rand, rand.flip(0)
    ctx = torch.tensor([200, 97], device=cuda, dtype=torch.int32)
    qkv = randn(g, B, T, (16 + 2 * nkv) * D, dtype=torch.bfloat16)
    cos, sin = K.rotary_tables(300, D, device=cuda)
    pos = (ctx[:, None] + torch.arange(T, device=cuda, dtype=torch.int32)).contiguous()
    outs = []
    for bt, k, v in ((far, kc, vc), (near, ks, vs)):
        q = torch.zeros(B, T, 16, D, device=cuda, dtype=torch.bfloat16)
        K.qk_norm_rotary_append_kv(qkv, pos, cos, sin, bt, ctx, q, k, v, 16, nkv)
        outs.append((q, K.tree_attention(q, k, v, bt, ctx, None, 0.1), k[-32:].clone(), v[-32:].clone()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert not bool(kc[:-32:1000].any())


def test_many_sequences_and_rows(cuda):
    """More sequences than one launch's lengths hold; every (batch, head) of them equals the call on its own."""
    g = gen(cuda, 30)
    B, T, nq, nkv, D = 300, 3, 8, 2, 64
    ctx = torch.randint(0, 200, (B,), generator=g, device=cuda, dtype=torch.int32)
    q, kc, vc, bt, _, bits = make_tree(g, cuda, B, T, nq, nkv, D, [200], torch.bfloat16)
    tl = torch.randint(0, T + 1, (B,), generator=g, device=cuda, dtype=torch.int32)
    out = torch.full_like(q, 4.0)
    K.tree_attention(q, kc, vc, bt, ctx, bits, 0.2, tree_lens=tl, out=out)
    pick = [0, 1, 127, 128, 129, 255, 256, 299]
    ref, mag, sm = tree_ref(q[pick], kc, vc, bt[pick], ctx[pick], [bits.tolist()[i] for i in pick], 0.2, tl[pick])
    got = out[pick]
    check_tree(got, ref, mag, sm, 203, D)
    dead = torch.arange(T, device=cuda)[None] >= tl[:, None]
    assert bool((out[dead] == 4).all())


def test_gradients_in_a_graph(cuda):
    """Forward and backward captured through autograd (no eager graph of the leaves alive: torch ties their accumulation
    nodes to its stream), and as plain calls while one is alive."""
    g = gen(cuda, 17)
    q, k = randn(g, 2, 9, 4, 64).requires_grad_(), randn(g, 2, 9, 2, 64).requires_grad_()
    wq, wk = torch.ones(64, device=cuda).requires_grad_(), torch.ones(64, device=cuda).requires_grad_()
    cos, sin = K.rotary_tables(9, 64, device=cuda)
    pos = torch.arange(9, device=cuda, dtype=torch.int32)
    dq, dk = randn(g, 2, 9, 4, 64), randn(g, 2, 9, 2, 64)

    def step():
        y = K.qk_norm_rotary(q, k, wq, wk, pos, cos, sin)
        z = K.rotary(y[0], pos, cos, sin)
        return torch.autograd.grad((z, y[1]), (q, k, wq, wk), (dq, dk))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    alive = K.qk_norm_rotary(q, k, wq, wk, pos, cos, sin)
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2), torch.no_grad():
        plain = K.qk_norm_rotary_backward(K.rotary(dq, pos, cos, sin, inverse=True), dk, q, k, wq, wk, pos, cos, sin)
    graph2.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(plain, want)) and alive[0].requires_grad


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(cuda):
    cos, sin = K.rotary_tables(8, 64, device=cuda)
    pos = torch.zeros(2, dtype=torch.int32, device=cuda)
    x = torch.zeros(2, 3, 64, device=cuda)

    def bad(match, fn, *a, **k):
        with pytest.raises(RuntimeError, match=match):
            fn(*a, **k)

    bad("dtype", K.rotary, x.double(), pos, cos, sin)
    bad("head_dim", K.rotary, torch.zeros(2, 3, 514, device=cuda), pos, cos, sin)
    bad("rotary_dim", K.rotary, x[..., :32], pos, cos, sin)
    bad("int32", K.rotary, x, pos.long(), cos, sin)
    bad("positions", K.rotary, x, pos[:1], cos, sin)
    bad("Float", K.rotary, x, pos, cos.double(), sin.double())
    buf = torch.zeros(4, 3, 64, device=cuda)
    bad("memory of its own", K.rotary, buf[:2], pos, cos, sin, out=buf[1:3])
    bad("overlaps itself", K.rotary, x, pos, cos, sin, out=torch.zeros(2, 1, 64, device=cuda).expand(2, 3, 64))
    bad("no gradient", K.rotary, x.clone().requires_grad_(), pos, cos, sin, out=x)
    bad("constants", K.rotary, x, pos, cos.clone().requires_grad_(), sin)
    off = torch.zeros(8 * 32 + 1, device=cuda)[1:].view(8, 32)
    bad("16-byte aligned", K.rotary, x, pos, off, sin)
    bad("no gradient|not formed", lambda: torch.autograd.grad(torch.autograd.grad(K.qk_norm_rotary(
        v := x.clone().requires_grad_(), x, torch.ones(64, device=cuda), torch.ones(64, device=cuda), pos, cos, sin)[0].sum(),
        v, create_graph=True)[0].sum(), v))
    w = torch.ones(64, device=cuda)
    bad("norm weights", K.qk_norm_rotary, x, x, w, w.half(), pos, cos, sin)
    bad("agree", K.qk_norm_rotary, x, x[:1], w, w, pos, cos, sin)
    h = torch.zeros(1, 2, 4, 64, device=cuda).half()
    kc = torch.zeros(3, 2, 16, 64, device=cuda).half()
    bt, cl = torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    bad("float16 or bfloat16", K.tree_attention, h.float(), kc.float(), kc.float(), bt, cl, None, 1.0)
    bad("1 to 64", K.tree_attention, h.expand(1, 2, 4, 64).repeat(1, 33, 1, 1), kc, kc, bt, cl, None, 1.0)
    bad("head_dim", K.tree_attention, h[..., :32], kc[..., :32], kc[..., :32], bt, cl, None, 1.0)
    bad("multiple of nkv", K.tree_attention, h[:, :, :3], kc, kc, bt, cl, None, 1.0)
    bad("tree_mask", K.tree_attention, h, kc, kc, bt, cl, torch.zeros(1, 3, dtype=torch.int64, device=cuda), 1.0)
    bad("block_tables", K.tree_attention, h, kc, kc, bt.long(), cl, None, 1.0)
    bad("ctx_lens", K.tree_attention, h, kc, kc, bt, torch.zeros(2, dtype=torch.int32, device=cuda), None, 1.0)
    bad("memory of its own", K.tree_attention, h, kc, kc, bt, cl, None, 1.0, out=h)
    qkv = torch.zeros(1, 2, 8 * 64, device=cuda).half()
    app = dict(positions=pos, cos=cos, sin=sin, block_tables=bt, starts=cl, q_out=h.clone(), k_cache=kc, v_cache=kc.clone(), nq=4, nkv=2)
    bad("heads", K.qk_norm_rotary_append_kv, qkv, **{**app, "nq": 5})
    bad("both norm weights", K.qk_norm_rotary_append_kv, qkv, **app, q_weight=w.half())
    bad("q_out", K.qk_norm_rotary_append_kv, qkv, **{**app, "q_out": h[:, :1].clone()})
    bad("caches must be", K.qk_norm_rotary_append_kv, qkv, **{**app, "k_cache": kc[:, :1].contiguous()})
    bad("memory of their own", K.qk_norm_rotary_append_kv, qkv, **{**app, "v_cache": kc})
    L = torch.zeros(2, 64, device=cuda)
    t = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    bad("need the rows' tokens", K.penalize_logits, L, repetition=torch.ones(2, device=cuda))
    bad("together", K.penalize_logits, L, bias_ids=t)
    bad("allowed", K.penalize_logits, L, allowed=torch.zeros(2, 2, dtype=torch.int32, device=cuda), vocab_offset=1)
    bad("tokens", K.penalize_logits, L, tokens=t.long(), repetition=torch.ones(2, device=cuda))
    bad("repetition", K.penalize_logits, L, tokens=t, repetition=torch.ones(3, device=cuda))
    bad("memory of its own", K.penalize_logits, L[:, :32], out=L[:, 32:])
    bad("keys", K.penalize_logits, L, keys=torch.zeros(3, dtype=torch.int64, device=cuda))
    torch.cuda.synchronize()
