"""Calls in which one CTA of a kernel for packed sequences or for a shared prefix is busy for longer than the kernels' limit of half a second on a
wait: the warps that wait for its end, or for a tile with work, have to see that it gets on. Everything but a few rows is zero, so that the
answer is that of a small call."""
import math

import pytest
import torch

from packed_util import close, ints, reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_a_key_tile_that_700_000_tiles_of_rows_walk():
    """dK and dV of 128 keys from 11 million queries of 8 heads. The rows overlap in memory; only the first and the last have an output gradient."""
    from self_trainable_or_free_attn_b200 import _native as N, packed
    D, H, n, others = 64, 8, 700_000 * 16, 100
    g = torch.Generator().manual_seed(0)
    base = {x: torch.zeros(n + H, D, dtype=BF, device="cuda") for x in ("q", "do")}
    ends = list(range(40)) + list(range(n - 40, n))
    for t in base.values():
        t[ends] = torch.randn(80, D, generator=g).to(BF).cuda()
    q, do = (base[x].as_strided((n, H, D), (D, D, 1)) for x in ("q", "do"))
    few = list(range(40)) + list(range(n - 48, n))
    keys = torch.zeros(2, 128 * 1001, 1, D, dtype=BF, device="cuda")
    keys[:, :128] = torch.randn(2, 128, 1, D, generator=g).to(BF).cuda()
    k, v = (x.clone().requires_grad_(True) for x in keys)
    # the other sequences have keys and no queries: with so many key tiles none is shared out
    cu_q = ints([0] + [n] * (others + 1))
    cu_k = ints([0, 128] + [128 + 1280 * (i + 1) for i in range(others)])
    sizes = (others + 1, n, k.shape[0], H, 1, D)
    lib = N.load()
    assert lib.es_packed_bwd_workspace_bytes(*sizes) < n * H * 4 + 256, "the walk is shared out"
    o, lse = packed.packed_attention(q, k, v, cu_q, cu_k, causal=False, return_lse=True)
    dk, dv = torch.autograd.grad(o, (k, v), do)
    packed.check_status()
    want = reference(q[few], k[:128], v[:128], [0, len(few)], [0, 128], False, D ** -0.5, do[few])
    for name, got in (("o", o[few]), ("lse", lse[:, few]), ("dk", dk[:128]), ("dv", dv[:128])):
        close(name, got, want[name])
    assert not dk[128:].any() and not dv[128:].any()


def test_one_query_that_walks_80_million_keys():
    """The other row tile of its CTA has nothing to do, and waits for the end of the walk."""
    from self_trainable_or_free_attn_b200 import _native as N, packed
    D, n, others = 64, 80_000_000, 1500
    g = torch.Generator().manual_seed(1)
    k = torch.zeros(n, 1, D, dtype=BF, device="cuda")
    at = torch.cat([torch.arange(20), torch.arange(n // 2, n // 2 + 20), torch.arange(n - 20, n)]).cuda()
    q = torch.randn(1, 1, D, generator=g).to(BF).cuda()
    # logits between 57 and 67: the zero keys weigh 8e7 e^-57 < 2^-55 of the row
    away = torch.randn(60, D, generator=g).double()
    unit = (q[0, 0].double() / q[0, 0].double().norm()).cpu()
    want_logit = torch.linspace(58, 66, 60).double()
    x = away - (away @ unit)[:, None] * unit + (want_logit * D ** 0.5 / q.double().norm().cpu())[:, None] * unit
    k[at] = x.to(BF).cuda()[:, None]
    cu_q, cu_k = ints([0] + [1] * (others + 1)), ints([0] + [n] * (others + 1))
    assert N.load().es_packed_fwd_workspace_bytes(others + 1, 1, n, 1, 1, D) == 0, "the walk is shared out"
    o, lse = packed.packed_attention(q, k, k, cu_q, cu_k, causal=False, return_lse=True)
    packed.check_status()
    want = reference(q, k[at], k[at], [0, 1], [0, 60], False, D ** -0.5)
    for name, got in (("o", o), ("lse", lse)):
        close(name, got, want[name])


def test_a_prefix_of_40_million_tokens():
    """Two tiles to an SM, of 312,500 key tiles each. The prefix is one page again and again: its LSE is the page's plus log of how often.

    A row's sum is added up from 312,500 numbers of 32 bits: off by less than 312,500 * 2^-24 < 2^-5 relative, which is what its log is off."""
    from self_trainable_or_free_attn_b200 import cache
    B, H, D, page, times = 300, 148, 64, 256, 156_250
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn(1, page, H, D, generator=g).to(BF).cuda() for _ in range(2))
    q = torch.randn(B, 1, H, D, generator=g).to(BF).cuda()
    table, own = ints([[]] * B).reshape(B, 0), ints([0] * B)
    pages = torch.zeros(times, dtype=torch.int32, device="cuda")
    once, z = cache.prefix_attention(q, kc, vc, pages[:1], page, table, own, return_lse=True)
    o, lse = cache.prefix_attention(q, kc, vc, pages, page * times, table, own, return_lse=True)
    cache.check_status()
    assert torch.isfinite(o.float()).all()
    assert (lse - z - math.log(times)).abs().max() <= 2.0 ** -5 + 2.0 ** -13
    assert not torch.isnan(once).any()


def test_four_million_sequences_without_tokens():
    """Behind the one that has some: the CTAs look through 64 million tiles of the grid that have no work."""
    from self_trainable_or_free_attn_b200 import packed
    B, H, D, n = 4_000_000, 16, 64, 10
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(n, H, D, generator=g).to(BF).cuda() for _ in range(4))
    cu = torch.full((B + 1,), n, dtype=torch.int32, device="cuda")
    cu[0] = 0
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o, lse = packed.packed_attention(*x, cu, return_lse=True)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, x, do)), o=o, lse=lse)
    packed.check_status()
    want = reference(q, k, v, [0, n], [0, n], True, D ** -0.5, do)
    for name in want:
        close(name, got[name], want[name])
