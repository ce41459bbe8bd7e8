"""CPU tier of the rotary, tree-attention and logits operators: tables, tree masks, refusals of host tensors."""
import math

import pytest
import torch

from comm_opt_b200._ext import available
from comm_opt_b200.ops import kernels as K
from comm_opt_b200.ops.reference import rope_tables

needs_ext = pytest.mark.skipif(not available(), reason="native extension not built")


def test_plain_tables_are_the_framework_tables():
    for a, b in zip(K.rotary_tables(300, 64, 500000.0), rope_tables(300, 64, 500000.0)):
        assert torch.equal(a, b)


def _angles(pos, dim, theta):
    return [pos * theta ** (-2 * j / dim) for j in range(dim // 2)]


def test_far_positions_keep_their_angle():
    """fp32 tables hold the cosine of the exact angle even at a million positions (an fp32 product would not)."""
    cos, sin = K.rotary_tables(1_000_001, 8, 10000.0)
    for j, a in enumerate(_angles(1_000_000, 8, 10000.0)):
        assert abs(float(cos[-1, j]) - math.cos(a)) <= 2 ** -24 + 1e-9
        assert abs(float(sin[-1, j]) - math.sin(a)) <= 2 ** -24 + 1e-9


def test_linear_and_ntk_scaling():
    a, _ = K.rotary_tables(33, 16, 1e4, dict(type="linear", factor=4.0))
    b, _ = K.rotary_tables(9, 16, 1e4)
    assert torch.allclose(a[::4], b, atol=2 ** -23)
    c, _ = K.rotary_tables(5, 16, 1e4, dict(type="ntk", factor=8.0))
    assert torch.allclose(c[:, 0], b[:5, 0], atol=2 ** -23)  # the highest frequency is kept
    low = 1e4 ** (-14 / 16) / 8.0  # the lowest is divided by the factor
    assert abs(float(c[4, 7]) - math.cos(4 * low)) <= 2 ** -23


def test_llama3_scaling_bands():
    dim, theta, orig = 128, 500000.0, 8192
    cos, sin = K.rotary_tables(2, dim, theta, dict(type="llama3", factor=8.0, original=orig))
    ang = torch.atan2(sin[1].double(), cos[1].double())
    for j in range(dim // 2):
        inv = theta ** (-2 * j / dim)
        wave = 2 * math.pi / inv
        if wave < orig / 4:
            want = inv
        elif wave > orig:
            want = inv / 8
        else:
            s = (orig / wave - 1) / 3
            want = (1 - s) * inv / 8 + s * inv
        assert abs(float(ang[j]) - want) <= 2 ** -22, j


def test_yarn_scaling_bands():
    dim, theta, orig, f = 64, 1e4, 4096, 16.0
    cos, sin = K.rotary_tables(2, dim, theta, dict(type="yarn", factor=f, original=orig))
    mul = 0.1 * math.log(f) + 1
    r = torch.sqrt(cos[1].double() ** 2 + sin[1].double() ** 2)
    assert torch.allclose(r, torch.full_like(r, mul), atol=1e-6)
    ang = torch.atan2(sin[1].double(), cos[1].double())
    assert abs(float(ang[0]) - 1.0) <= 1e-6  # fast components are kept, slow ones divided
    assert abs(float(ang[-1]) - theta ** (-62 / 64) / f) <= 1e-9


def test_table_refusals():
    for bad in (dict(type="spiral"), dict(type="linear", factor=2.0, original=3), dict(type="linear", factor=0.0)):
        with pytest.raises(ValueError):
            K.rotary_tables(4, 8, 1e4, bad)
    with pytest.raises(ValueError):
        K.rotary_tables(4, 7)
    with pytest.raises(ValueError):
        K.rotary_tables(0, 8)


def test_tree_mask_bits():
    #      0        1        2 (under 0)  3 (under 2)  4 (under 1)
    p = torch.tensor([[-1, -1, 0, 2, 1], [-1, 0, 1, 2, 3]])
    m = K.tree_mask(p)
    assert m.tolist() == [[0b1, 0b10, 0b101, 0b1101, 0b10010], [0b1, 0b11, 0b111, 0b1111, 0b11111]]
    chain = K.tree_mask(torch.arange(64) - 1)
    assert chain[63].item() == -1 and chain[62].item() == 2 ** 63 - 1 and chain[0].item() == 1
    # a parent that is not earlier counts as none
    assert K.tree_mask(torch.tensor([5, 1, 0])).tolist() == [1, 2, 5]
    with pytest.raises(ValueError):
        K.tree_mask(torch.zeros(2, 65))


@needs_ext
def test_host_tensors_are_refused():
    cos, sin = K.rotary_tables(8, 8)
    pos = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rotary(torch.zeros(2, 3, 8), pos, cos, sin)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.qk_norm_rotary(torch.zeros(2, 3, 8), torch.zeros(2, 1, 8), torch.ones(8), torch.ones(8), pos, cos, sin)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.tree_attention(torch.zeros(1, 2, 4, 64).half(), torch.zeros(1, 1, 16, 64).half(), torch.zeros(1, 1, 16, 64).half(),
                         torch.zeros(1, 1).int(), torch.zeros(1).int(), None, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.penalize_logits(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        K.qk_norm_rotary_append_kv(torch.zeros(1, 1, 24), pos[:1], cos, sin, torch.zeros(1, 1).int(), pos[:1],
                                   torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 16, 8), torch.zeros(1, 1, 16, 8), 1, 1)


@pytest.mark.parametrize("most", [1, 7, 49, 74, 148])
def test_tree_attention_shares_cover_once_and_join_what_was_cut(most):
    """csrc/tree_attention.cu's partition: positions are COST per (sequence, KV head) plus one per tile; every tile
    belongs to one share, a share's pieces of a cut (sequence, head) sit in slot 0 (the piece's head holds the share's
    first position) or 1, and the joining kernel's arithmetic finds exactly these slots, in order."""
    COST = 2
    for nkv, tiles in [(1, [1]), (8, [9]), (2, [3, 0, 5, 1]), (8, [17] * 8), (1, [0, 0, 4]), (4, list(range(13))), (8, [257, 1, 30]),
                       (3, [1] * 40), (1, [400])]:
        cum = [0]
        for t in tiles:
            cum.append(cum[-1] + ((t + COST) * nkv if t else 0))
        total = cum[-1]
        shares = min(most, total)
        written, seen = {}, set()
        for c in range(shares):
            beg, end = c * total // shares, (c + 1) * total // shares
            assert beg < end
            g = beg
            while g < end:
                b = max(i for i in range(len(tiles)) if cum[i] <= g)
                cost = (cum[b + 1] - cum[b]) // nkv
                rem = g - cum[b]
                kvh, nt = rem // cost, cost - COST
                at = g - (rem - kvh * cost)
                t0, t1 = max(0, g - at - COST), min(nt, end - at - COST)
                first, g = g == beg, min(end, at + cost)
                if t0 >= t1:
                    continue
                for t in range(t0, t1):
                    assert (b, kvh, t) not in seen
                    seen.add((b, kvh, t))
                if t1 - t0 < nt:
                    key = (c, 0 if first else 1)
                    assert key not in written
                    written[key] = (b, kvh, t0)
        assert len(seen) == nkv * sum(tiles)
        joined = set()

        def share_of(g):
            return ((g + 1) * shares - 1) // total

        for b, nt in enumerate(tiles):
            for kvh in range(nkv if nt else 0):
                at = cum[b] + kvh * (nt + COST)
                s0, s1 = share_of(at + COST), share_of(at + COST + nt - 1)
                last = -1
                for s in range(s0, s1 + 1) if s0 != s1 else ():
                    key = (s, 0 if s > s0 or s * total // shares >= at else 1)
                    assert written[key][:2] == (b, kvh) and written[key][2] > last
                    last = written[key][2]
                    joined.add(key)
        assert joined == set(written)
