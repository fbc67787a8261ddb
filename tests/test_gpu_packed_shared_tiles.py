"""`packed.packed_attention` where both row tiles of a CTA are cut by a mask in the same tile of keys: what is not finite in its V is found once,
by one of them, and has to reach the rows of both that see it, and no other, in every run."""
import pytest
import torch

from packed_util import ints, make

pytestmark = pytest.mark.gpu


def _want(clean, n_q, n_k, H, Hk, at, heads, causal):
    """Rows and heads that see key `at` of the one sequence."""
    hit = torch.zeros(n_q, H, dtype=torch.bool)
    first = max(0, at - (n_k - n_q)) if causal else 0
    for kh in heads:
        hit[first:, kh * (H // Hk):(kh + 1) * (H // Hk)] = True
    return hit


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n_q,n_k,H,Hk,causal", [
    (256, 340, 2, 2, True),          # a pair of tiles of one head whose diagonals pass the same keys
    (50, 50, 10, 2, True),           # 25 tokens x 5 heads to a tile: both in the first 128 keys
    (32, 128 + 20, 40, 5, True),     # 16 tokens x 8 heads
    (200, 200, 1, 1, False),         # the ragged end of the keys, both tiles
    (20, 77, 24, 2, False)])
def test_both_row_tiles_find_it(n_q, n_k, H, Hk, causal, D, value):
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, _, cu_q, cu_k = make([n_q], [n_k], H, Hk, D, torch.bfloat16, seed=n_q)
    clean = packed.packed_attention(q, k, v, ints(cu_q), ints(cu_k), causal=causal).cpu()
    for at in (n_k - 1, n_k - n_q // 2, max(n_k - n_q, 1)):
        x = v.clone()
        x[at, 0, D - 1] = value                              # (the last chunk of the row: the longest way from its flag to its look)
        hit = _want(clean, n_q, n_k, H, Hk, at, [0], causal)
        first = None
        for _ in range(100):
            got = packed.packed_attention(q, k, x, ints(cu_q), ints(cu_k), causal=causal)
            if first is None:
                first = got.cpu()
                assert torch.equal(~torch.isfinite(first[..., D - 1].float()), hit)
                assert torch.equal(first[~hit], clean[~hit]) and torch.isfinite(first[..., :D - 1].float()).all()
            bits = got.view(torch.int16).cpu()
            assert torch.equal(bits, first.view(torch.int16))
