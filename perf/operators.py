"""Cases of the speculative-decoding and rotary-position operators, with plain forms of each.

Four operators of `comm_opt_b200.ops.kernels`:

- ``rotary``         rotary positions: half or interleaved layout, whole head or its first part, tables scaled
                     for long contexts; forward, and forward with backward.
- ``qk_norm_rotary`` RMSNorm of every query and key head with the rotation in the same pass: the training form
                     (forward and backward, gradients of the norm weights among them) and the serving form that
                     also appends k and v to the paged cache.
- ``tree_attention`` grouped-query attention of a tree of drafted tokens over a paged cache.
- ``penalize_logits`` repetition / frequency / presence penalties, sparse biases and grammar masks on logits,
                     with the greedy choice of the result.

`run` is the plain form where `own` is false and the calls of the package where it is true. Model shapes
(heads, head sizes, vocabularies) are those of `comm_opt_b200.models.llama` and its tensor-parallel shards.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE = 16  # tokens per cache page


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 8 sequences, 8B-shaped query heads
        dict(name="rotary_decode", op="rotary", batch=8, seq=1, heads=32, dim=128, rot=128, dtype="bf16",
             inter=False, train=False, strided=True, far=2048, scaling="none"),
        # one training micro-batch of the 1B shape: head size 64, forward and backward
        dict(name="rotary_train", op="rotary", batch=4, seq=2048, heads=32, dim=64, rot=64, dtype="bf16",
             inter=False, train=True, strided=False, far=0, scaling="none"),
        # a long prompt, first half of each head rotated, neighbouring pairs, tables scaled for 128k positions
        dict(name="rotary_long_partial", op="rotary", batch=1, seq=32763, heads=64, dim=128, rot=64, dtype="f16",
             inter=True, train=False, strided=True, far=98304, scaling="yarn"),
        # decode append of 8 sequences, 8B heads
        dict(name="qk_norm_decode", op="qk_norm_rotary", batch=8, seq=1, nq=32, nkv=8, dim=128, rot=128,
             dtype="bf16", wdtype="bf16", inter=False, train=False, norm=True, bias=False, ctx=2047, ragged=True,
             strided=False),
        # prompts of unequal lengths entering the cache, Qwen2.5-32B heads with the QKV bias
        dict(name="qk_norm_prompts", op="qk_norm_rotary", batch=4, seq=2048, nq=40, nkv=8, dim=128, rot=128,
             dtype="bf16", wdtype="bf16", inter=False, train=False, norm=True, bias=True, ctx=0, ragged=True,
             strided=False),
        # the training batch of 8 sequences x 2048 tokens, 8B heads, fp32 norm weights, q and k views of one tensor
        dict(name="qk_norm_train", op="qk_norm_rotary", batch=8, seq=2048, nq=32, nkv=8, dim=128, rot=128,
             dtype="bf16", wdtype="f32", inter=False, train=True, norm=True, bias=False, ctx=0, ragged=False,
             strided=True),
        # one sequence, a draft of 8 tokens over a short cache
        dict(name="tree_short", op="tree_attention", batch=1, tree=8, nq=32, nkv=8, dim=128, dtype="bf16", ctx=1021,
             ragged=False, padded=False),
        # 8 sequences of the 70B heads with 16 drafted tokens over 2k-token caches of unequal lengths
        dict(name="tree_batch", op="tree_attention", batch=8, tree=16, nq=64, nkv=8, dim=128, dtype="bf16",
             ctx=2048, ragged=True, padded=True),
        # wide trees over long caches: the arithmetic of attention, not the cache's bytes, is what counts
        dict(name="tree_long_wide", op="tree_attention", batch=4, tree=64, nq=64, nkv=8, dim=128, dtype="f16",
             ctx=32749, ragged=False, padded=False),
        # one request, bf16 logits of a 128256-token vocabulary, a short history
        dict(name="logits_one", op="penalize_logits", batch=1, vocab=128256, dtype="bf16", history=211, penalties=True,
             bias=16, mask=False, greedy=True, offset=0),
        # a serving batch of one vocabulary shard's rows with grammar masks, long histories
        dict(name="logits_shard", op="penalize_logits", batch=32, vocab=19008, dtype="bf16", history=4096,
             penalties=True, bias=300, mask=True, greedy=True, offset=38016),
        # the largest batch, fp32 logits, every feature
        dict(name="logits_batch", op="penalize_logits", batch=128, vocab=152064, dtype="f32", history=2048,
             penalties=True, bias=64, mask=True, greedy=False, offset=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm_rotary", "tree_attention", "penalize_logits"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim // 2, dim // 4 // 2 * 2])
        heads = rng.choice([1, 4, 8, 32, 40, 64])
        seq = max(1, min(_log(rng, 1, 32768), 268000000 // (heads * dim) // 2))
        train = rng.random() < 0.4
        batch = max(1, min(_log(rng, 1, 64), (80000000 if train else 130000000) // (heads * dim * seq)))
        return dict(op=op, batch=batch, seq=seq, heads=heads, dim=dim, rot=rot, dtype=rng.choice(["bf16", "f16", "f32"]),
                    inter=rng.random() < 0.5, train=train, strided=rng.random() < 0.5, far=rng.choice([0, 4000, 98304]),
                    scaling=rng.choice(["none", "linear", "llama3", "yarn"]))
    if op == "qk_norm_rotary":
        nq, nkv, dim = rng.choice([(32, 8, 128), (64, 8, 128), (40, 8, 128), (8, 1, 128), (5, 1, 128), (32, 4, 64),
                                   (16, 2, 64)])
        train = rng.random() < 0.5
        seq = _log(rng, 1, 2048)
        batch = max(1, min(_log(rng, 1, 64), 16384 * 5120 // (seq * (nq + nkv) * dim)))
        return dict(op=op, batch=batch, seq=seq, nq=nq, nkv=nkv, dim=dim, rot=rng.choice([dim, dim // 2]),
                    dtype=rng.choice(["bf16", "f16"] + (["f32"] if train else [])),
                    wdtype=rng.choice(["same", "f32"]), inter=rng.random() < 0.5, train=train,
                    norm=True if train else rng.random() < 0.7, bias=(not train) and rng.random() < 0.3,
                    ctx=0 if train else rng.choice([0, _log(rng, 1, 8192)]), ragged=rng.random() < 0.5,
                    strided=rng.random() < 0.5)
    if op == "tree_attention":
        nq, nkv, dim = rng.choice([(32, 8, 128), (64, 8, 128), (40, 8, 128), (8, 1, 128), (5, 1, 128), (32, 4, 64),
                                   (4, 4, 64), (16, 1, 128)])
        tree = _log(rng, 1, 64)
        ctx = rng.choice([0, _log(rng, 1, 32768), _log(rng, 256, 32768)])
        cap = 4 * 64 * 64 * 128 * 32000
        batch = max(1, min(_log(rng, 1, 64), cap // (tree * nq * dim * (ctx + tree)), (131072 * 8 * 128) // ((ctx + tree) * nkv * dim)))
        return dict(op=op, batch=batch, tree=tree, nq=nq, nkv=nkv, dim=dim, dtype=rng.choice(["bf16", "f16"]), ctx=ctx,
                    ragged=rng.random() < 0.5, padded=rng.random() < 0.4)
    vocab, offset = rng.choice([(128256, 0), (152064, 0), (32000, 0), (16032, 16032), (19008, 38016), (50257, 0),
                                (_log(rng, 1000, 200000), 0)])
    dtype = rng.choice(["bf16", "f16", "f32"])
    batch = max(1, min(_log(rng, 1, 256), 19000000 // vocab))
    return dict(op=op, batch=batch, vocab=vocab, dtype=dtype, history=rng.choice([0, _log(rng, 1, 8192)]),
                penalties=rng.random() < 0.8, bias=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5,
                greedy=rng.random() < 0.5, offset=offset)


# --------------------------------------------------------------------------------------------- preparing
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + salt)


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _tables(n, rot, scaling):
    """cos / sin [n, rot / 2] in fp32 of angles formed in 64 bits; theta and scalings as models publish them."""
    half = rot // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    inv = 500000.0 ** (-2.0 * i / rot)
    mul = 1.0
    if scaling == "linear":
        inv = inv / 4.0
    elif scaling == "llama3":
        wave = 2 * math.pi / inv
        smooth = ((8192 / wave - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        inv = (1 - smooth) * inv / 8.0 + smooth * inv
    elif scaling == "yarn":
        def at(turns):
            return rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        inv = inv / 16.0 * ramp + inv * (1 - ramp)
        mul = 0.1 * math.log(16.0) + 1.0
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return (ang.cos() * mul).float(), (ang.sin() * mul).float()


def _lens(gen, batch, full, ragged, low=0):
    if not ragged or full <= low:
        return torch.full((batch,), full, dtype=torch.int32, device="cuda")
    n = torch.randint(low, full + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    n[0] = full
    return n


def _pages(gen, batch, pages):
    return torch.randperm(batch * pages, generator=gen, device="cuda").to(torch.int32).view(batch, pages)


def prepare(case, seed):
    torch.cuda.current_device()
    return {"rotary": _prep_rotary, "qk_norm_rotary": _prep_qk, "tree_attention": _prep_tree,
            "penalize_logits": _prep_logits}[case["op"]](case, seed)


def _prep_rotary(c, seed):
    g, dt = _gen(seed, 1), DT[c["dtype"]]
    B, S, H, D = c["batch"], c["seq"], c["heads"], c["dim"]
    if c["strided"]:  # the query heads of a projection output that also holds two more heads
        x = _randn(g, B, S, (H + 2) * D, dtype=dt).view(B, S, H + 2, D)[:, :, :H]
    else:
        x = _randn(g, B, S, H, D, dtype=dt)
    cos, sin = _tables(c["far"] + S, c["rot"], c["scaling"])
    start = torch.randint(0, c["far"] + 1, (B, 1), generator=g, device="cuda")
    pos = (start + torch.arange(S, device="cuda")[None, :]).to(torch.int32)
    st = dict(case=c, x=x.requires_grad_() if c["train"] else x, pos=pos, cos=cos, sin=sin)
    if c["train"]:
        st["dy"] = _randn(g, B, S, H, D, dtype=dt)
    return st


def _prep_qk(c, seed):
    g, dt = _gen(seed, 2), DT[c["dtype"]]
    B, S, nq, nkv, D = c["batch"], c["seq"], c["nq"], c["nkv"], c["dim"]
    wdt = dt if c["wdtype"] == "same" else DT[c["wdtype"]]
    n = nq + 2 * nkv
    wq = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(wdt) if c["norm"] else None
    wk = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(wdt) if c["norm"] else None
    cos, sin = _tables(c["ctx"] + S, c["rot"], "none")
    st = dict(case=c, wq=wq, wk=wk, cos=cos, sin=sin, eps=1e-6)
    if c["train"]:
        if c["strided"]:
            qkv = _randn(g, B, S, n * D, dtype=dt).view(B, S, n, D)
            q, k = qkv[:, :, :nq], qkv[:, :, nq:nq + nkv]
        else:
            q, k = _randn(g, B, S, nq, D, dtype=dt), _randn(g, B, S, nkv, D, dtype=dt)
        st.update(q=q.detach().requires_grad_(), k=k.detach().requires_grad_(), wq=wq.requires_grad_(),
                  wk=wk.requires_grad_(), dq=_randn(g, B, S, nq, D, dtype=dt), dk=_randn(g, B, S, nkv, D, dtype=dt),
                  pos=torch.arange(S, device="cuda", dtype=torch.int32))
        return st
    width = n * D + (64 if c["strided"] else 0)  # a projection output with a wider row
    qkv = _randn(g, B, S, width, dtype=dt)[..., :n * D]
    lens = _lens(g, B, S, c["ragged"], 1) if S > 1 else None
    starts = _lens(g, B, c["ctx"], c["ragged"])
    pages = (c["ctx"] + S + PAGE - 1) // PAGE
    pos = (starts[:, None] + torch.arange(S, device="cuda", dtype=torch.int32)[None, :]).contiguous()
    st.update(qkv=qkv, lens=lens, starts=starts, pos=pos, bt=_pages(g, B, pages),
              bias=_randn(g, n * D, dtype=dt) if c["bias"] else None,
              kc=torch.zeros(B * pages, nkv, PAGE, D, device="cuda", dtype=dt),
              vc=torch.zeros(B * pages, nkv, PAGE, D, device="cuda", dtype=dt),
              q_out=torch.zeros(B, S, nq, D, device="cuda", dtype=dt))
    return st


def _prep_tree(c, seed):
    g, dt = _gen(seed, 3), DT[c["dtype"]]
    B, T, nq, nkv, D = c["batch"], c["tree"], c["nq"], c["nkv"], c["dim"]
    pages = (c["ctx"] + T + PAGE - 1) // PAGE
    kc = _randn(g, B * pages, nkv, PAGE, D, dtype=dt)
    vc = _randn(g, B * pages, nkv, PAGE, D, dtype=dt)
    q = _randn(g, B, T, nq, D, dtype=dt)
    # every node hangs from a random earlier one, the first from the cache's last token; ancestors as bits
    par = (torch.rand(B, T, generator=g, device="cuda") * torch.arange(T, device="cuda")).long()
    bits = torch.ones(B, T, dtype=torch.int64, device="cuda")
    for t in range(1, T):
        own_bit = 1 << t if t < 63 else -(1 << 63)
        bits[:, t] = bits.gather(1, par[:, t:t + 1])[:, 0] | own_bit
    return dict(case=c, kc=kc, vc=vc, q=q, bits=bits, bt=_pages(g, B, pages), ctx=_lens(g, B, c["ctx"], c["ragged"]),
                tlens=_lens(g, B, T, True, 1) if c["padded"] else None, scale=1 / math.sqrt(D),
                out=torch.zeros(B, T, nq, D, device="cuda", dtype=dt))


def _prep_logits(c, seed):
    g, dt = _gen(seed, 4), DT[c["dtype"]]
    B, V, L, off = c["batch"], c["vocab"], c["history"], c["offset"]
    total = off + V
    st = dict(case=c, logits=_randn(g, B, V, dtype=torch.float32).mul_(3).to(dt), out=torch.zeros(B, V, device="cuda", dtype=dt),
              keys=torch.zeros(B, dtype=torch.int64, device="cuda"),
              ids=torch.zeros(B, dtype=torch.int32, device="cuda"))
    # text repeats itself: ids follow a skewed distribution
    u = torch.rand(B, max(L, 1), generator=g, device="cuda", dtype=torch.float64)
    st["tokens"] = (u ** 3 * total).long().clamp_(max=total - 1).to(torch.int32)
    st["lens"] = _lens(g, B, L, True)
    st["plens"] = (st["lens"].float() * torch.rand(B, generator=g, device="cuda")).to(torch.int32)

    def per_row(lo, hi):
        return lo + (hi - lo) * torch.rand(B, generator=g, device="cuda")
    st["rep"], st["freq"], st["pres"] = per_row(1.0, 1.5), per_row(0.0, 0.5), per_row(0.0, 1.0)
    if c["bias"]:
        st["bias_ids"] = torch.randint(0, total, (B, c["bias"]), generator=g, device="cuda", dtype=torch.int32)
        st["bias_ids"][:, c["bias"] * 3 // 4 + 1:] = -1  # requests with fewer entries end in padding
        st["bias_vals"] = 4 * torch.randn(B, c["bias"], generator=g, device="cuda")
    if c["mask"]:  # grammars allow anything from a few tokens to nearly all
        words = (total + 31) // 32
        r = torch.randint(-2**31, 2**31, (B, words), generator=g, device="cuda", dtype=torch.int64)
        r2 = torch.randint(-2**31, 2**31, (B, words), generator=g, device="cuda", dtype=torch.int64)
        few = torch.arange(B, device="cuda")[:, None] % 2 == 0
        st["mask"] = torch.where(few, r & r2, r | r2).to(torch.int32)
    return st


# ------------------------------------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, inter, sign=1.0):
    """x [..., H, D] in fp32, cos / sin [..., rot / 2] of its rows."""
    h = cos.shape[-1]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2) * sign
    y = x.clone()
    if inter:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y[..., 0:2 * h:2] = a * c - b * s
        y[..., 1:2 * h:2] = b * c + a * s
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        y[..., :h] = a * c - b * s
        y[..., h:2 * h] = b * c + a * s
    return y


def _plain_rotary(st):
    c, x = st["case"], st["x"].detach()
    p = st["pos"].long()
    cos, sin = st["cos"][p], st["sin"][p]
    y = _rotate(x.float(), cos, sin, c["inter"]).to(x.dtype)
    if not c["train"]:
        return y
    return y, _rotate(st["dy"].float(), cos, sin, c["inter"], -1.0).to(x.dtype)


def _norm_rot_train(x, w, dy, cos, sin, eps, inter):
    """(y, dx, dw) of y = rotate(x * rstd * w) in fp32, rounded at the end."""
    xf, wf = x.float(), w.float()
    rstd = (xf.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = xf * rstd
    y = _rotate(xh * wf, cos, sin, inter).to(x.dtype)
    g = _rotate(dy.float(), cos, sin, inter, -1.0)
    dw = (g * xh).sum((0, 1, 2)).to(w.dtype)
    g = g * wf
    return y, ((g - xh * (g * xh).mean(-1, keepdim=True)) * rstd).to(x.dtype), dw


def _plain_qk(st):
    c = st["case"]
    if c["train"]:
        p = st["pos"].long()
        cos, sin = st["cos"][p][None], st["sin"][p][None]
        yq, dq, dwq = _norm_rot_train(st["q"].detach(), st["wq"].detach(), st["dq"], cos, sin, st["eps"], c["inter"])
        yk, dk, dwk = _norm_rot_train(st["k"].detach(), st["wk"].detach(), st["dk"], cos, sin, st["eps"], c["inter"])
        return yq, yk, dq, dk, dwq, dwk
    B, S, nq, nkv, D = c["batch"], c["seq"], c["nq"], c["nkv"], c["dim"]
    x = st["qkv"].float()
    if st["bias"] is not None:
        x = x + st["bias"].float()
    x = x.view(B, S, nq + 2 * nkv, D)
    p = st["pos"].long()
    cos, sin = st["cos"][p], st["sin"][p]
    q, k, v = x.split([nq, nkv, nkv], 2)
    if c["norm"]:
        q = q * (q.square().mean(-1, keepdim=True) + st["eps"]).rsqrt() * st["wq"].float()
        k = k * (k.square().mean(-1, keepdim=True) + st["eps"]).rsqrt() * st["wk"].float()
    q, k = _rotate(q, cos, sin, c["inter"]), _rotate(k, cos, sin, c["inter"])
    dt = st["qkv"].dtype
    slot = st["starts"].long()[:, None] + torch.arange(S, device="cuda")[None]
    live = torch.ones_like(slot, dtype=torch.bool) if st["lens"] is None else \
        torch.arange(S, device="cuda")[None] < st["lens"].long()[:, None]
    page = st["bt"].long().gather(1, slot // PAGE)[live]
    off = (slot % PAGE)[live]
    q_out = torch.where(live[:, :, None, None], q.to(dt), st["q_out"])
    st["kc"][page, :, off] = k.to(dt)[live]
    st["vc"][page, :, off] = v.to(dt)[live]
    return q_out, st["kc"], st["vc"]


def _plain_tree(st):
    c = st["case"]
    B, T, nq, nkv, D = c["batch"], c["tree"], c["nq"], c["nkv"], c["dim"]
    G, n = nq // nkv, st["bt"].shape[1] * PAGE
    slot = torch.arange(n, device="cuda")
    node = slot[None] - st["ctx"].long()[:, None]  # [B, n]: drafted token at this slot, negative in the cache
    shift = node.clamp(0, 63)[:, None, :].expand(B, T, n)
    see = (node[:, None] < 0) | ((node[:, None] < T) & ((st["bits"][:, :, None] >> shift) & 1).bool())  # [B, T, n]
    if st["tlens"] is not None:
        tl = st["tlens"].long()
        see = see & (node < tl[:, None])[:, None]
    see = see.unsqueeze(2)[:, None]  # [B, 1, T, 1, n]
    bt = st["bt"].long()
    k = st["kc"][bt].permute(0, 2, 1, 3, 4).reshape(B, nkv, n, D).float()
    q = st["q"].float().view(B, T, nkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, D)
    s = (q @ k.transpose(-1, -2)) * st["scale"]
    del k
    s = s.view(B, nkv, T, G, n).masked_fill(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = (s - m).exp()
    del s
    p = torch.where(m == float("-inf"), torch.zeros_like(p), p)
    z = p.sum(-1, keepdim=True)
    v = st["vc"][bt].permute(0, 2, 1, 3, 4).reshape(B, nkv, n, D).float()
    o = (p.view(B, nkv, T * G, n) @ v).view(B, nkv, T, G, D)
    o = torch.where(z > 0, o / z, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(B, T, nq, D).to(st["q"].dtype)
    if st["tlens"] is None:
        return o
    live = torch.arange(T, device="cuda")[None] < st["tlens"].long()[:, None]
    return torch.where(live[:, :, None, None], o, st["out"])


def _history(st, dtype):
    """(seen in prompt or output, count in the output) [B, V] of this shard's vocabulary."""
    c = st["case"]
    B, V, L, off = c["batch"], c["vocab"], c["history"], c["offset"]
    seen = torch.zeros(B, V + 1, dtype=dtype, device="cuda")
    count = torch.zeros(B, V + 1, dtype=dtype, device="cuda")
    if L:
        i = torch.arange(L, device="cuda")[None]
        live, outp = i < st["lens"][:, None], i >= st["plens"][:, None]
        idx = st["tokens"][:, :L].long() - off
        idx = torch.where(live & (idx >= 0) & (idx < V), idx, V)
        seen.scatter_(1, idx, 1.0)
        count.scatter_add_(1, idx, outp.to(dtype))
    return seen[:, :V] > 0, count[:, :V]


def _add_bias(st, x):
    c = st["case"]
    V = c["vocab"]
    idx = st["bias_ids"].long() - c["offset"]
    idx = torch.where((idx >= 0) & (idx < V), idx, V)
    b = torch.zeros(c["batch"], V + 1, dtype=torch.float64, device="cuda")  # entries of one id add up
    b.scatter_add_(1, idx, st["bias_vals"].double())
    b = b.to(x.dtype)
    return x + b[:, :V]


def _allowed(st):
    c = st["case"]
    i = torch.arange(c["vocab"], device="cuda") + c["offset"]
    return ((st["mask"][:, i // 32] >> (i % 32)) & 1).bool()


def _plain_logits(st):
    c = st["case"]
    x = st["logits"].float()
    if c["penalties"]:
        seen, count = _history(st, torch.float32)
        x = torch.where(seen, torch.where(x > 0, x / st["rep"][:, None], x * st["rep"][:, None]), x)
        x = x - st["freq"][:, None] * count
        x = x - st["pres"][:, None] * (count > 0)
    if c["bias"]:
        x = _add_bias(st, x)
    if c["mask"]:
        x = x.masked_fill(~_allowed(st), float("-inf"))
    x = x.to(st["logits"].dtype)
    if not c["greedy"]:
        return x
    top = x.amax(-1, keepdim=True)
    i = torch.arange(c["vocab"], device="cuda")
    return x, torch.where(x == top, i, c["vocab"]).amin(-1).add(c["offset"]).to(torch.int32)


# ------------------------------------------------------------------------------------- the package's calls
def _own_rotary(st):
    from comm_opt_b200.ops import kernels as K

    c = st["case"]
    y = K.rotary(st["x"], st["pos"], st["cos"], st["sin"], interleaved=c["inter"])
    if not c["train"]:
        return y
    return y.detach(), torch.autograd.grad(y, st["x"], st["dy"])[0]


def _own_qk(st):
    from comm_opt_b200.ops import kernels as K

    c = st["case"]
    if c["train"]:
        yq, yk = K.qk_norm_rotary(st["q"], st["k"], st["wq"], st["wk"], st["pos"], st["cos"], st["sin"], st["eps"],
                                  interleaved=c["inter"])
        grads = torch.autograd.grad((yq, yk), (st["q"], st["k"], st["wq"], st["wk"]), (st["dq"], st["dk"]))
        return (yq.detach(), yk.detach(), *grads)
    K.qk_norm_rotary_append_kv(st["qkv"], st["pos"], st["cos"], st["sin"], st["bt"], st["starts"], st["q_out"],
                               st["kc"], st["vc"], c["nq"], c["nkv"], q_weight=st["wq"], k_weight=st["wk"],
                               eps=st["eps"], lens=st["lens"], bias=st["bias"], interleaved=c["inter"])
    return st["q_out"], st["kc"], st["vc"]


def _own_tree(st):
    from comm_opt_b200.ops import kernels as K

    return K.tree_attention(st["q"], st["kc"], st["vc"], st["bt"], st["ctx"], st["bits"], st["scale"],
                            tree_lens=st["tlens"], out=st["out"])


def _own_logits(st):
    from comm_opt_b200.ops import kernels as K

    c = st["case"]
    a = {}
    if c["penalties"]:
        a.update(tokens=st["tokens"], lens=st["lens"], prompt_lens=st["plens"], repetition=st["rep"],
                 frequency=st["freq"], presence=st["pres"])
    if c["bias"]:
        a.update(bias_ids=st["bias_ids"], bias=st["bias_vals"])
    if c["mask"]:
        a.update(allowed=st["mask"])
    if not c["greedy"]:
        return K.penalize_logits(st["logits"], vocab_offset=c["offset"], out=st["out"], **a)
    out = K.penalize_logits(st["logits"], vocab_offset=c["offset"], out=st["out"], keys=st["keys"], **a)
    ids = K.argmax_combine(st["keys"].view(1, -1), 1, ids=st["ids"], local_keys=st["keys"])
    return out, ids


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "qk_norm_rotary": _own_qk, "tree_attention": _own_tree,
                "penalize_logits": _own_logits}[op](state)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "qk_norm_rotary": _plain_qk, "tree_attention": _plain_tree,
                "penalize_logits": _plain_logits}[op](state)


# ----------------------------------------------------------------------------------------------- the work
def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rotary":
        n = c["batch"] * c["seq"] * c["heads"]
        tab = min(c["batch"] * c["seq"], c["far"] + c["seq"]) * c["rot"] * 4 + c["batch"] * c["seq"] * 4
        passes = 2 if c["train"] else 1
        return {"bytes": passes * (2 * n * c["dim"] * e + tab), "flops": passes * 3 * n * c["rot"]}
    if c["op"] == "qk_norm_rotary":
        rows, D = c["batch"] * c["seq"], c["dim"]
        heads = c["nq"] + c["nkv"]
        if c["train"]:
            # forward reads and writes every head, backward reads the heads and their gradients, writes gradients
            return {"bytes": 5 * rows * heads * D * e + 2 * c["seq"] * c["rot"] * 4,
                    "flops": rows * heads * (4 * D + 3 * c["rot"] + 10 * D + 3 * c["rot"])}
        return {"bytes": 2 * rows * (heads + c["nkv"]) * D * e + rows * (c["rot"] * 4 + 8),
                "flops": rows * heads * (4 * D * c["norm"] + 3 * c["rot"])}
    if c["op"] == "tree_attention":
        B, T, nq, nkv, D = c["batch"], c["tree"], c["nq"], c["nkv"], c["dim"]
        ctx = c["ctx"] * (0.5 if c["ragged"] and B > 1 else 1.0)  # ragged: uniform lengths up to ctx
        return {"bytes": int(2 * B * (ctx + T) * nkv * D * e + 2 * B * T * nq * D * e + B * T * 8),
                "flops": int(4 * B * T * nq * D * (ctx + T))}
    B, V = c["batch"], c["vocab"]
    b = 2 * B * V * e + (B * V // 8 if c["mask"] else 0) + B * c["bias"] * 8
    if c["penalties"]:
        b += B * c["history"] // 2 * 4
    return {"bytes": b, "flops": B * V * 4}


# ------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "qk_norm_rotary": _exact_qk, "tree_attention": _exact_tree,
                "penalize_logits": _exact_logits}[case["op"]](st)


def _pair_index(rot, inter):
    j = torch.arange(rot // 2, device="cuda")
    return (2 * j, 2 * j + 1) if inter else (j, j + rot // 2)


def _turn(x, cos, sin, inter, back=False):
    """Each pair of the first `rot` components as a complex number, times cos + i sin (or its conjugate)."""
    a, b = _pair_index(2 * cos.shape[-1], inter)
    z = torch.complex(x[..., a], x[..., b])
    w = torch.complex(cos, -sin if back else sin).unsqueeze(-2)
    z = z * w
    y = x.clone()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_rotary(st):
    c = st["case"]
    p = st["pos"].long()
    ys, gs = [], []
    for b in range(c["batch"]):
        cos, sin = st["cos"].double()[p[b]], st["sin"].double()[p[b]]
        ys.append(_turn(st["x"].detach()[b].double(), cos, sin, c["inter"]))
        if c["train"]:
            gs.append(_turn(st["dy"][b].double(), cos, sin, c["inter"], back=True))
    return (torch.stack(ys), torch.stack(gs)) if c["train"] else torch.stack(ys)


def _exact_qk(st):
    c = st["case"]
    if c["train"]:
        p = st["pos"].long()
        cos, sin = st["cos"].double()[p], st["sin"].double()[p]
        res = []
        for x, w, dy in ((st["q"], st["wq"], st["dq"]), (st["k"], st["wk"], st["dk"])):
            w64 = w.detach().double()
            ys, dxs, dw = [], [], torch.zeros_like(w64)
            for b in range(c["batch"]):
                xb = x.detach()[b].double()
                r = 1.0 / torch.sqrt((xb * xb).sum(-1, keepdim=True) / c["dim"] + st["eps"])
                ys.append(_turn(xb * r * w64, cos, sin, c["inter"]))
                g = _turn(dy[b].double(), cos, sin, c["inter"], back=True)
                dw += (g * xb * r).sum((0, 1))
                g = g * w64
                dxs.append(r * g - xb * r ** 3 * (g * xb).sum(-1, keepdim=True) / c["dim"])
            res.append((torch.stack(ys), torch.stack(dxs), dw))
        (yq, dq, dwq), (yk, dk, dwk) = res
        return yq, yk, dq, dk, dwq, dwk
    B, S, nq, nkv, D = c["batch"], c["seq"], c["nq"], c["nkv"], c["dim"]
    q_out, kc, vc = st["q_out"].double(), st["kc"].double(), st["vc"].double()
    for b in range(B):
        n = S if st["lens"] is None else int(st["lens"][b])
        x = st["qkv"][b, :n].double()
        if st["bias"] is not None:
            x = x + st["bias"].double()
        x = x.reshape(n, nq + 2 * nkv, D)
        p = st["pos"][b, :n].long()
        cos, sin = st["cos"].double()[p], st["sin"].double()[p]
        parts = []
        for h, w in ((x[:, :nq], st["wq"]), (x[:, nq:nq + nkv], st["wk"])):
            if c["norm"]:
                h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / D + st["eps"]) * w.double()
            parts.append(_turn(h, cos, sin, c["inter"]))
        q_out[b, :n] = parts[0]
        at = int(st["starts"][b]) + torch.arange(n, device="cuda")
        page = st["bt"][b].long()[at // PAGE]
        kc[page, :, at % PAGE] = parts[1]
        vc[page, :, at % PAGE] = x[:, nq + nkv:]
    return q_out, kc, vc


def _exact_tree(st):
    c = st["case"]
    B, T, nq, nkv, D = c["batch"], c["tree"], c["nq"], c["nkv"], c["dim"]
    out = st["out"].double()
    nodes = torch.arange(T, device="cuda")
    for b in range(B):
        n, t = int(st["ctx"][b]), T if st["tlens"] is None else int(st["tlens"][b])
        at = torch.arange(n + t, device="cuda")
        page = st["bt"][b].long()[at // PAGE]
        k, v = st["kc"][page, :, at % PAGE], st["vc"][page, :, at % PAGE]  # [n + t, nkv, D]
        hide = torch.zeros(t, n + t, dtype=torch.bool, device="cuda")
        hide[:, n:] = ((st["bits"][b, :t, None] >> nodes[None, :t]) & 1) == 0
        for h in range(nkv):
            q = st["q"][b, :t, h * (nq // nkv):(h + 1) * (nq // nkv)].double()  # [t, G, D]
            s = torch.matmul(q, k[:, h].double().t()) * st["scale"]
            s.masked_fill_(hide[:, None], float("-inf"))
            w = torch.softmax(s, -1)
            out[b, :t, h * (nq // nkv):(h + 1) * (nq // nkv)] = torch.matmul(w, v[:, h].double())
    return out


def _exact_logits(st):
    c = st["case"]
    x = st["logits"].double()
    if c["penalties"]:
        seen, count = _history(st, torch.float64)
        r = st["rep"].double()[:, None]
        x = torch.where(seen & (x > 0), x / r, torch.where(seen, x * r, x))
        x = x - count * st["freq"].double()[:, None] - (count > 0).double() * st["pres"].double()[:, None]
    if c["bias"]:
        x = _add_bias(st, x)
    if c["mask"]:
        x = torch.where(_allowed(st), x, torch.full_like(x, float("-inf")))
    return (x, None) if c["greedy"] else x
