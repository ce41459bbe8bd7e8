"""Speculative-decoding attention over the paged cache, and penalties and masks on logits."""
from __future__ import annotations

import torch

from .._ext import native

MAX_TREE = 64


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """Ancestor bits (int64, bit j: drafted token j is seen) of drafted trees given as parents [.., tree]: each token's
    parent is an earlier token's index, or -1 for a token that follows the cache directly. A token sees itself."""
    T = parents.shape[-1]
    if not 1 <= T <= MAX_TREE:
        raise ValueError(f"a tree has 1 to {MAX_TREE} drafted tokens, got {T}")
    p = parents.long()
    bits = torch.zeros(*p.shape[:-1], T + 1, dtype=torch.int64, device=p.device)  # the last column: no parent
    for t in range(T):
        own = 1 << t if t < 63 else -(1 << 63)
        src = torch.where((p[..., t:t + 1] >= 0) & (p[..., t:t + 1] < t), p[..., t:t + 1], T)
        bits[..., t:t + 1] = bits.gather(-1, src) | own
    return bits[..., :T].contiguous()


def tree_attention_error_word(device) -> torch.Tensor:
    """Per-device int32 that `tree_attention` sets when one of its bounded waits runs out (zero it to go on)."""
    dev = torch.device(device)
    return native().tree_attention_error_word(dev.index if dev.index is not None else torch.cuda.current_device())


def tree_attention(q, k_cache, v_cache, block_tables, ctx_lens, tree_mask, scale: float, *, tree_lens=None, out=None,
                   timeout_ms: float = 1000.0):
    """Grouped-query attention of drafted tokens over a paged cache that already holds their k and v.

    q [batch, tree, nq, D] (fp16 / bf16, D 64 or 128, any strides, tree <= 64); caches [num_blocks, nkv, 16, D];
    block_tables int32 [batch, max_blocks]; ctx_lens int32 [batch]: tokens before the tree. Row t of sequence b sees
    the slots [0, ctx_lens[b]) and the drafted tokens j (slot ctx_lens[b] + j) with bit j of tree_mask (int64 [batch,
    tree] or [tree], see `tree_mask`; None: a chain, token t sees 0..t). A row that sees nothing gives zeros; whatever a
    slot that a row does not see holds, infinities and NaN included, does not reach it. With tree_lens (int32 [batch])
    rows t >= tree_lens[b] are padding: nothing sees them and `out` keeps what it held there (zeros without `out`). Slots
    past the block table are not seen; a page index outside the cache reads as zeros. Every wait inside the kernel is
    bounded by `timeout_ms` (0: it gives up before the first): where one runs out, rows become NaN and
    `tree_attention_error_word` is set. No gradient is formed."""
    return native().tree_attention(q, k_cache, v_cache, block_tables, ctx_lens, tree_mask, float(scale), tree_lens, out,
                                   int(timeout_ms * 1e6))


def penalize_logits(logits, *, tokens=None, lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
                    bias_ids=None, bias=None, allowed=None, vocab_offset: int = 0, out=None, keys=None):
    """Penalties, biases and grammar masks on logits [rows, vocab] (fp32, fp16, bf16), in this order:

    - id seen in the row's tokens: x / repetition where x > 0, else x * repetition;
    - seen c > 0 times in its output: x - frequency * c - presence;
    - x + the sum of its entries in bias_ids / bias;
    - -inf where its bit of `allowed` is 0.

    tokens int32 [rows, history]: the first lens[row] (default all) count, of them the first prompt_lens[row] (default
    none) are the prompt's. repetition, frequency, presence: fp32 [rows] each, None for none. bias_ids int32 and bias fp32
    [rows, entries]; at most 2^30 ids and entries a row. allowed int32 [rows, words], bit i % 32 of word i / 32 for id i.
    All ids are global: logits column v is id vocab_offset + v of a vocabulary shard; ids elsewhere (or negative: padding)
    are skipped. Computed in fp32, rounded once. `out` may be the logits themselves. With `keys` (int64 [rows], zero
    before use) the stored values' greedy keys are folded in as `argmax_local` does, for `argmax_combine`. No gradient is
    formed."""
    return native().penalize_logits(logits, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias,
                                    allowed, int(vocab_offset), out, keys)
