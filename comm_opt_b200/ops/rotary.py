"""Rotary positions and per-head norms of queries and keys: table builder, autograd, paged append.

Layouts: ``interleaved=False`` rotates components (j, j + rotary_dim / 2), as the decode kernels and the models
of this package do; ``interleaved=True`` rotates neighbours (2j, 2j + 1). ``rotary_dim`` is twice the tables' column
count and may be smaller than the head: the components past it pass through.
"""
from __future__ import annotations

import math

import torch

from .._ext import native


def rotary_tables(max_pos: int, rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, device=None):
    """cos, sin [max_pos, rotary_dim / 2] fp32 of angles formed in 64 bits (a far position times a frequency needs
    more than 24 bits).

    ``scaling`` stretches the positions of a model beyond its training length ``original``: dict(type=...) of

    - ``linear``: factor - every frequency divided by it;
    - ``ntk``: factor - theta raised so that the lowest frequency is divided by it and the highest kept;
    - ``llama3``: factor, original, low_freq_factor = 1, high_freq_factor = 4 - wavelengths above original /
      low are divided, those below original / high kept, a linear blend between;
    - ``yarn``: factor, original, beta_fast = 32, beta_slow = 1, attention_factor = 0.1 ln(factor) + 1 - components
      that turn fewer than beta_slow times in original positions are divided, those that turn more than beta_fast
      times kept, a ramp between; cos and sin are multiplied by attention_factor.
    """
    if max_pos < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"need max_pos >= 1 and an even rotary_dim >= 2, got {max_pos}, {rotary_dim}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    mul = 1.0
    sc = dict(scaling or {"type": "none"})
    kind = sc.pop("type")
    factor = float(sc.pop("factor", 1.0))
    if factor <= 0:
        raise ValueError(f"rotary scaling factor must be positive, got {factor}")
    if kind == "ntk":
        if rotary_dim > 2:
            theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** (-i / rotary_dim)
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        orig, low, high = sc.pop("original"), sc.pop("low_freq_factor", 1.0), sc.pop("high_freq_factor", 4.0)
        turns = orig * inv / (2 * math.pi)  # in the original length
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        inv = keep * inv + (1 - keep) * inv / factor
    elif kind == "yarn":
        orig, fast, slow = sc.pop("original"), sc.pop("beta_fast", 32.0), sc.pop("beta_slow", 1.0)
        mul = sc.pop("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)

        def index(turns):  # component that turns this often in the original length
            return rotary_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1 - ramp) + inv / factor * ramp
    elif kind not in ("none", "ntk"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    if sc:
        raise ValueError(f"unknown rotary scaling arguments for {kind!r}: {sorted(sc)}")
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    return (ang.cos() * mul).float().to(device), (ang.sin() * mul).float().to(device)


def rotary(x: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, interleaved: bool = False,
           inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate x [tokens, heads, D] or [batch, seq, heads, D] (fp32, fp16, bf16; any strides) by its positions
    (int32 [seq] or [batch, seq]) and the tables cos, sin (fp32 [max_pos, rotary_dim / 2], see `rotary_tables`).

    Differentiable in x (reverse mode). ``inverse`` applies the transpose, the gradient's rotation: it rotates back where
    cos^2 + sin^2 = 1, and with tables that carry a factor m (YaRN's attention_factor) leaves m^2 x. ``out`` may be x (in
    place, no gradient) or other memory. A row whose position lies outside the tables becomes zeros (and has a zero
    gradient): padded rows carry position -1."""
    if out is None and x.requires_grad and torch.is_grad_enabled():
        return native().rotary_autograd(x, positions, cos, sin, bool(interleaved), bool(inverse))
    if out is not None and torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
        raise RuntimeError("rotary with out= forms no gradient: call it without out, or under torch.no_grad()")
    return native().rotary(x, positions, cos, sin, bool(interleaved), bool(inverse), out)


def qk_norm_rotary(q, k, q_weight, k_weight, positions, cos, sin, eps: float = 1e-6, *, interleaved: bool = False):
    """(rotate(RMSNorm(q) * q_weight), rotate(RMSNorm(k) * k_weight)) in one pass over q [.., nq, D] and k [.., nkv, D]
    (shapes, positions and tables as in `rotary`); the norms are over each head's D components, their weights [D] of
    the operands' type or fp32. fp32 inside, one rounding at the end.

    Differentiable in q, k and both weights (reverse mode, once). `qk_norm_rotary_backward` is the same gradient as a plain call: it can be
    captured in a CUDA graph whatever else is alive, which torch allows for autograd only while no eager graph of the same
    leaves is."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or
                                    k_weight.requires_grad):
        return native().qk_norm_rotary_autograd(q, k, q_weight, k_weight, positions, cos, sin, float(eps), bool(interleaved))
    return native().qk_norm_rotary(q, k, q_weight, k_weight, positions, cos, sin, float(eps), bool(interleaved))


def qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, positions, cos, sin, eps: float = 1e-6, *,
                            interleaved: bool = False):
    """Gradients (q, k, q_weight, k_weight) of `qk_norm_rotary` from those of its outputs. The weights' gradients are
    summed in fp32 in a fixed order (equal inputs give equal bits) and rounded to the weights' type. The results are
    constants: what requires a gradient is taken as its value."""
    return native().qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, positions, cos, sin, float(eps),
                                            bool(interleaved))


def qk_norm_rotary_append_kv(qkv, positions, cos, sin, block_tables, starts, q_out, k_cache, v_cache, nq: int, nkv: int, *,
                             q_weight=None, k_weight=None, eps: float = 1e-6, lens=None, bias=None,
                             interleaved: bool = False):
    """Projection rows into queries and the paged cache: bias, per-head RMSNorm of q and k (with the weights; none
    without), rotation, k and v appended. For prompts, single tokens and drafted trees alike.

    qkv [batch, seq, (nq + 2 nkv) D] (or [batch * seq, ..]; any row stride): row s of sequence b goes to cache slot
    starts[b] + s (int32 [batch]) and is rotated by positions[b, s] (int32; a drafted token's position is its depth, not
    its slot). q_out [batch, seq, nq, D]; caches [num_blocks, nkv, 16, D] (fp32, fp16, bf16) paged by block_tables
    [batch, max_blocks]. Rows s >= lens[b], and rows whose position lies outside the tables, are left out: q_out and the
    caches keep what they held. k and v of rows whose slot or page does not exist are dropped; the rows of a call have
    slots of their own. No gradient is formed."""
    native().qk_norm_rotary_append(qkv, positions, cos, sin, block_tables, starts, q_out, k_cache, v_cache, int(nq),
                                   int(nkv), q_weight, k_weight, float(eps), lens, bias, bool(interleaved))
    return q_out
