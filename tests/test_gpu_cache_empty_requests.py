"""`prefix_attention` of a batch in which nearly every request is without tokens of its own."""
import pytest
import torch

from test_packed_cpu import _prefix

BF = torch.bfloat16


@pytest.mark.gpu
def test_eight_million_requests_without_tokens():
    """Between two that have some: a CTA that has a part of both passes the others while its other warps wait."""
    from self_trainable_or_free_attn_b200 import cache
    B = 2 ** 23
    g = torch.Generator().manual_seed(0)
    kc, vc = (torch.randn(3, 16, 1, 64, generator=g).to(BF).cuda() for _ in range(2))
    q = torch.ones(B, 1, 1, 64, dtype=BF, device="cuda")
    table, lengths = torch.full((B, 1), 2, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    pages = torch.zeros(0, dtype=torch.int32, device="cuda")
    at = [5, B - 2]
    lengths[at] = torch.tensor([16, 9], dtype=torch.int32, device="cuda")
    o, lse = cache.prefix_attention(q, kc, vc, pages, 0, table, lengths, return_lse=True)
    cache.check_status()
    for b in at:
        one, z = cache.prefix_attention(q[b:b + 1], kc, vc, pages, 0, table[b:b + 1], lengths[b:b + 1], return_lse=True)
        assert torch.equal(o[b:b + 1], one) and torch.equal(lse[b:b + 1], z) and one.any()
    o[at], lse[at] = 0, -torch.inf
    assert not o.any() and torch.isneginf(lse).all()
    more = torch.zeros(1, dtype=torch.int32, device="cuda").expand(B + 1)
    with pytest.raises(RuntimeError, match="requests"):
        cache.prefix_attention(q[:1].expand(B + 1, 1, 1, 64), kc, vc, pages, 0, more[:, None], more)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: without a GPU no call can reach a kernel with them")
def test_more_are_refused():
    from self_trainable_or_free_attn_b200 import _native
    lib = _native.load()
    assert lib.es_prefix_attn(*_prefix(B=2 ** 23).values()) < -1, "stopped by nothing but the missing GPU"
    assert lib.es_prefix_attn(*_prefix(B=2 ** 23 + 1).values()) == -1 and "requests" in _native.last_error()
