"""The paged cache: `extend_tables` against loops in Python, `store_kv` against indexing, `prefix_attention` against its definition in 64
bits (tests/packed_util.py has the bounds), and a prompt followed by tokens through all of them together with `packed_attention`."""
import random

import pytest
import torch

from packed_util import SLACK, close, grid, ints, reference, starts, unit

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------------------------- pages and slots
def _plan(lengths, new, table, free, page, total):
    """(slots, positions, cu, lengths after, taken, table after) by the definition."""
    slots, pos, cu, after, used, missing = [], [], [0], [], 0, 0
    table, width = [list(r) for r in table], len(table[0]) if table else 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        n, m = max(n, 0), max(m, 0)
        have, want = -(-n // page), -(-(n + m) // page)
        stored = n
        for j in range(have, want):
            if j < width:
                table[b][j] = free[used] if used < len(free) else -1
                used += 1
            if j >= width or table[b][j] < 0:
                missing += 1
        for i in range(m):
            j = (n + i) // page
            p = table[b][j] if j < width else -1
            slots.append(p * page + (n + i) % page if p >= 0 else -1)
            pos.append(n + i)
            if p >= 0 and stored == n + i:
                stored += 1
        cu.append(cu[-1] + m)
        after.append(stored)
    slots, pos = slots[:total], pos[:total]
    return slots + [-1] * (total - len(slots)), pos + [-1] * (total - len(pos)), cu, after, [min(used, len(free)), missing], table


def _case(B, width, page, n_free, most, seed, dense=True):
    r = random.Random(seed)
    lengths = [min(r.choice([0, 1, page - 1, page, page + 1, r.randint(0, most)]), width * page) for _ in range(B)]
    new = [r.choice([0, 1, 1, page, r.randint(0, most)]) for _ in range(B)]
    ids = list(range(B * width + n_free))
    r.shuffle(ids)
    table = [[ids.pop() if j < -(-n // page) else -7 for j in range(width)] for n in lengths]
    return lengths, new, table, [ids.pop() for _ in range(n_free)]


@pytest.mark.parametrize("B,width,page,n_free,most", [(1, 4, 16, 3, 40), (7, 6, 16, 60, 60), (64, 9, 64, 600, 300), (300, 5, 16, 800, 40),
                                                      (1023, 3, 4, 3100, 6), (1025, 4, 8, 4200, 20), (2500, 3, 3, 9000, 5), (9, 3, 16, 5, 60),
                                                      (40, 2, 16, 0, 50), (33, 0, 16, 10, 5), (5, 40, 1, 300, 30), (17, 4, 100, 100, 300)])
@pytest.mark.parametrize("extra", [0, 1000, -5])
def test_extend_tables(B, width, page, n_free, most, extra):
    from self_trainable_or_free_attn_b200 import cache
    lengths, new, table, free = _case(B, width, page, n_free, most, B + page)
    total = max(0, sum(new) + extra)
    want = _plan(lengths, new, table, free, page, total)
    t = ints(table).reshape(B, width)
    n0 = ints(lengths)
    for _ in range(2):                                       # again: the same result on the table it has written
        plan = cache.extend_tables(n0, ints(new), t, ints(free), page, total=total)
        assert plan.slots.tolist() == want[0] and plan.positions.tolist() == want[1]
        assert plan.cu_new.tolist() == want[2] and plan.lengths.tolist() == want[3] and plan.taken.tolist() == want[4]
        assert t.tolist() == want[5] and n0.tolist() == lengths


def test_extend_tables_of_nothing_and_of_negative_lengths():
    from self_trainable_or_free_attn_b200 import cache
    e = ints([])
    plan = cache.extend_tables(e, e, ints([]).reshape(0, 4), ints([1, 2]), 16, total=3)
    assert plan.slots.tolist() == [-1] * 3 and plan.cu_new.tolist() == [0] and plan.taken.tolist() == [0, 0]
    t = ints([[5, -1], [6, -1]])
    plan = cache.extend_tables(ints([-3, 2]), ints([2, -4]), t, ints([9]), 16, total=2)
    assert plan.slots.tolist() == [144, 145] and plan.lengths.tolist() == [2, 2] and t.tolist() == [[9, -1], [6, -1]]


def test_slots_past_32_bits_are_none():
    from self_trainable_or_free_attn_b200 import cache
    t = ints([[2 ** 30]])
    plan = cache.extend_tables(ints([1]), ints([1]), t, ints([]), 16, total=1)
    assert plan.slots.tolist() == [-1]
    plan = cache.extend_tables(ints([2 ** 31 - 5]), ints([2 ** 31 - 5]), ints([[3]]), ints([4]), 16, total=4)
    assert plan.slots.tolist() == [-1] * 4 and plan.lengths.tolist() == [2 ** 31 - 5] and plan.taken.tolist()[0] == 0


# ---------------------------------------------------------------------------------------------- storing
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("layout", ["plain", "joint", "head_major"])
@pytest.mark.parametrize("T,Hk,D,page", [(1, 1, 64, 16), (77, 3, 128, 16), (300, 8, 128, 100), (33, 5, 64, 1)])
def test_store_kv(T, Hk, D, page, layout, dtype):
    from self_trainable_or_free_attn_b200 import cache
    P = -(-T // page) + 3
    g = torch.Generator().manual_seed(T)
    if layout == "joint":
        kc, vc = torch.randn(P, 2, page, Hk, D, generator=g).to(dtype).cuda().unbind(1)
    elif layout == "head_major":
        kc, vc = (torch.randn(P, Hk, page, D, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    else:
        kc, vc = (torch.randn(P, page, Hk, D, generator=g).to(dtype).cuda() for _ in range(2))
    fused = torch.randn(T, 2, Hk, D, generator=g).to(dtype).cuda()
    slots = torch.randperm(P * page, generator=g)[:T].to(torch.int32).cuda()
    slots[::7] = torch.tensor([-1, P * page, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).cuda()[torch.arange(len(slots[::7])) % 4]
    want_k, want_v = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = fused[t, 0], fused[t, 1]
    cache.store_kv(fused[:, 0], fused[:, 1], kc, vc, slots)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    cache.store_kv(fused[:0, 0], fused[:0, 1], kc, vc, slots[:0])


def test_store_kv_and_autograd():
    """Nothing that takes part in a graph is stored without its gradient, and a graph that saved the cache does not use what has replaced it."""
    from self_trainable_or_free_attn_b200 import cache
    kc, vc = (torch.ones(2, 16, 2, 64, dtype=BF, device="cuda") for _ in range(2))
    k, v, slots = kc[0, :3].clone(), vc[0, :3].clone(), ints([1, 20, 7])
    for leaf in (k, v, kc, vc):
        leaf.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            cache.store_kv(k, v, kc, vc, slots)
        with torch.no_grad():
            cache.store_kv(k, v, kc, vc, slots)
        leaf.requires_grad_(False)
    w = torch.ones(2, 16, 2, 64, dtype=BF, device="cuda", requires_grad=True)
    for c in (kc, vc):
        y = (w * c).sum()
        cache.store_kv(k, v, kc, vc, slots)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        ki, vi = kc.clone(), vc.clone()
        cache.store_kv(2 * k, 2 * v, ki, vi, slots)
        cache.store_kv(2 * k, 2 * v, kc, vc, slots)
        assert torch.equal(ki, kc) and torch.equal(vi, vc) and float(kc.detach()[1, 4, 0, 0]) == 2


# ---------------------------------------------------------------------------------------------- attention
def _prefix_case(B, N, H, Hk, D, page, prefix, own, dtype, seed=0, layout="plain"):
    g = torch.Generator().manual_seed(seed)
    width = max([-(-n // page) for n in own] + [0]) + 1
    n_prefix = -(-prefix // page)
    P = n_prefix + sum(-(-n // page) for n in own) + 2
    if layout == "joint":
        kc, vc = torch.randn(P, 2, page, Hk, D, generator=g).to(dtype).cuda().unbind(1)
    elif layout == "head_major":
        kc, vc = (torch.randn(P, Hk, page, D, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    else:
        kc, vc = (torch.randn(P, page, Hk, D, generator=g).to(dtype).cuda() for _ in range(2))
    ids = torch.randperm(P, generator=g).tolist()
    pages = [ids.pop() for _ in range(n_prefix)]
    table = [[ids.pop() if j < -(-n // page) else -1 for j in range(width)] for n in own]
    q = (torch.randn(B, N, H, D, generator=g) * 1.5).to(dtype).cuda()
    return q, kc, vc, pages, table


def _prefix_reference(q, kc, vc, pages, prefix, table, own, scale, ok=None):
    """The definition through tests/packed_util.py's: each request as a sequence of its keys, in front of them as many as its queries lack."""
    B, N, H, D = q.shape
    page, Hk = kc.shape[1], kc.shape[2]
    u, g = unit(q.dtype), grid(q.dtype)
    kc, vc = kc.double().cpu(), vc.double().cpu()
    o, to, lse = torch.zeros(B, N, H, D).double(), torch.zeros(B, N, H, D).double(), torch.full((B, H, N), -torch.inf).double()
    for b in range(B):
        for i in range(N):
            at = [(pages[j // page], j % page) for j in range(prefix)] + [(table[b][j // page], j % page) for j in range(max(0, own[b] - N + i + 1))]
            at = [(p, t) for p, t in at if 0 <= p < kc.shape[0]]
            if not at:
                continue
            p, t = zip(*at)
            K, V = kc[list(p), list(t)], vc[list(p), list(t)]
            for h in range(H):
                kh = h // (H // Hk)
                S = scale * K[:, kh] @ q[b, i, h].double().cpu()
                z = torch.logsumexp(S, 0)
                w = torch.exp(S - z)
                o[b, i, h], lse[b, h, i] = w @ V[:, kh], z
                # parts that are joined are rounded once more to 32 bits, inside the slack
                to[b, i, h] = (u + SLACK) * (w @ V[:, kh].abs()) + u * (w @ V[:, kh]).abs() + g * V[:, kh].abs().sum(0) + g
    return (o, to), (lse, torch.full_like(lse, 64 * 2.0 ** -20))


def _prefix_check(B, N, H, Hk, D, page, prefix, own, dtype, seed=0, layout="plain"):
    from self_trainable_or_free_attn_b200 import cache
    q, kc, vc, pages, table = _prefix_case(B, N, H, Hk, D, page, prefix, own, dtype, seed, layout)
    o, lse = cache.prefix_attention(q, kc, vc, ints(pages), prefix, ints(table), ints(own), return_lse=True)
    want_o, want_lse = _prefix_reference(q, kc, vc, pages, prefix, table, own, D ** -0.5)
    close("o", o, want_o)
    close("lse", lse, want_lse)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (BF, 64), (FP, 128)])
def test_prefix_pages(page, dtype, D):
    _prefix_check(5, 1, 4, 2, D, page, 300, [1, 17, 64, 129, 300], dtype, seed=page)


@pytest.mark.parametrize("H,Hk", [(1, 1), (5, 1), (7, 1), (12, 4), (16, 2), (40, 1), (136, 1), (3, 3)])
@pytest.mark.parametrize("N", [1, 2, 5])
def test_prefix_head_groups(H, Hk, N):
    _prefix_check(3, N, H, Hk, 64, 16, 150, [N, 40, 131], BF, seed=H)


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 127, 128, 129, 1000])
@pytest.mark.parametrize("own", [[0, 0], [1, 0], [128, 129], [1, 700]])
def test_prefix_lengths(prefix, own):
    """No prefix, no own tokens (a row without any key is 0, LSE -inf), one, tiles that just end."""
    _prefix_check(2, 1, 2, 1, 128, 16, prefix, own, BF, seed=prefix)


@pytest.mark.parametrize("B", [1, 2, 33, 130, 300])
def test_prefix_batches(B):
    r = random.Random(B)
    _prefix_check(B, 1, 2, 1, 64, 16, 200, [r.randint(1, 60) for _ in range(B)], BF, seed=B)


@pytest.mark.parametrize("layout", ["joint", "head_major"])
def test_prefix_layouts(layout):
    _prefix_check(3, 2, 6, 2, 128, 32, 100, [5, 40, 70], BF, layout=layout)


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_what_is_not_finite_among_the_newest_tokens(which):
    """Three queries each: the second's key or value is NaN; the first must not see it."""
    from self_trainable_or_free_attn_b200 import cache
    own = [40, 66, 3]
    q, kc, vc, pages, table = _prefix_case(3, 3, 4, 2, 64, 16, 50, own, BF)
    args = (ints(pages), 50, ints(table), ints(own))
    clean = cache.prefix_attention(q, kc, vc, *args)
    bad = torch.zeros(3, 3, 4, dtype=torch.bool)             # [request, query, head]
    for b in range(3):
        if which == "q":
            q[b, 1, 2] = float("nan")
            bad[b, 1, 2] = True
        else:
            j = own[b] - 2
            (kc if which == "k" else vc)[table[b][j // 16], j % 16, 1] = float("nan")
            bad[b, 1:, 2:] = True
    got = cache.prefix_attention(q, kc, vc, *args)
    assert torch.equal(~torch.isfinite(got.float()).all(-1).cpu(), bad)
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])


def test_fewer_own_tokens_than_queries():
    """Rows of a padded batch: lengths below the number of queries leave the first queries the prefix alone."""
    _prefix_check(4, 4, 4, 2, 64, 16, 40, [0, 1, 3, 4], BF)
    _prefix_check(4, 4, 4, 2, 64, 16, 0, [0, 1, 3, 4], BF)


@pytest.mark.parametrize("B", [3, 70])
def test_bad_pages_and_what_lies_behind(B):
    """Pages of -1 or beyond the cache are not attended to; lengths beyond the table's row count as the row; NaN in pages of others, and behind the last token
    in a request's own last page, reaches nothing."""
    from self_trainable_or_free_attn_b200 import cache
    own = ([40, 70, 33] * B)[:B]
    q, kc, vc, pages, table = _prefix_case(B, 1, 4, 2, 64, 16, 100, own, BF)
    used = {(p, j) for i, p in enumerate(pages) for j in range(16) if 16 * i + j < 100}
    used |= {(table[b][j // 16], j % 16) for b in range(B) for j in range(own[b])}
    for p in range(kc.shape[0]):
        for j in range(16):
            if (p, j) not in used:
                kc[p, j], vc[p, j] = float("nan"), float("inf")
    pages[2], table[0][1], table[1][0], table[1][3] = -1, kc.shape[0], 2 ** 31 - 1, -2 ** 31
    o, lse = cache.prefix_attention(q, kc, vc, ints(pages), 100, ints(table), ints(own), return_lse=True)
    want_o, want_lse = _prefix_reference(q, kc, vc, pages, 100, table, own, 0.125)
    close("o", o, want_o)
    close("lse", lse, want_lse)
    # every page bad, no prefix
    o, lse = cache.prefix_attention(q, kc, vc, ints([]), 0, ints([[-1] * 6] * B), ints(own), return_lse=True)
    assert (o == 0).all() and torch.isinf(lse).all()
    o, lse = cache.prefix_attention(q, kc, vc, ints([-1] * 9), 140, ints([[-1] * 6] * B), ints(own), return_lse=True)
    assert (o == 0).all() and torch.isinf(lse).all()
    # lengths beyond the row
    full = cache.prefix_attention(q, kc, vc, ints(pages), 100, ints(table)[:, :2].contiguous(), ints([32] * B))
    assert torch.equal(cache.prefix_attention(q, kc, vc, ints(pages), 100, ints(table)[:, :2].contiguous(), ints(([99, 2 ** 31 - 1, 32] * B)[:B])), full)


@pytest.mark.parametrize("B", [4, 70])
@pytest.mark.parametrize("which", ["q", "k_prefix", "v_prefix", "v_last", "k_own", "v_own"])
def test_what_is_not_finite_stays_with_its_request(which, B):
    from self_trainable_or_free_attn_b200 import cache
    own = ([40, 70, 33, 150] * B)[:B]
    q, kc, vc, pages, table = _prefix_case(B, 1, 4, 2, 128, 16, 200, own, BF)
    args = (ints(pages), 200, ints(table), ints(own))
    clean = cache.prefix_attention(q, kc, vc, *args)
    bad = torch.zeros(B, 4, dtype=torch.bool)                # [request, head]
    if which == "q":
        q[1, 0, 2] = float("nan")
        bad[1, 2] = True
    else:
        page, at = (table[1][2], 9) if which.endswith("own") else (pages[5], 3) if which.endswith("prefix") else (pages[12], 6)
        (kc if which[0] == "k" else vc)[page, at, 1] = float("inf")
        bad[:, 2:] = True
        if which.endswith("own"):
            bad[torch.arange(B) != 1] = False
    got = cache.prefix_attention(q, kc, vc, *args)
    assert torch.equal(~torch.isfinite(got[:, 0].float()).all(-1).cpu(), bad)
    assert torch.equal(got[:, 0].cpu()[~bad], clean[:, 0].cpu()[~bad])


def test_long_axis_few_rows():
    """One request against a long prefix and a long answer: the keys are shared out over the GPU and joined."""
    _prefix_check(1, 1, 4, 1, 128, 64, 20000, [9000], BF)


def test_same_bits_twice_on_another_stream_and_captured():
    from self_trainable_or_free_attn_b200 import cache
    own = [40, 700, 33]
    q, kc, vc, pages, table = _prefix_case(3, 2, 8, 2, 128, 16, 500, own, BF)
    at = [ints(pages), 500, ints(table), ints(own)]
    want = cache.prefix_attention(q, kc, vc, *at, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(want, cache.prefix_attention(q, kc, vc, *at, return_lse=True)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = torch.empty_like(q).copy_(q)
        got = cache.prefix_attention(late, kc, vc, *at, return_lse=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(cache.prefix_attention(q, kc, vc, *at, return_lse=True))
    for lengths in (own, [3, 12, 0], [48, 690, 40]):
        at[3].copy_(ints(lengths))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = cache.prefix_attention(q, kc, vc, *at[:3], ints(lengths), return_lse=True)
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


def test_cache_past_32_bits():
    """Caches of more than 2^31 elements, the pages in use at their end: stored, and attended to by both kernels of the prefix."""
    from self_trainable_or_free_attn_b200 import cache
    P, S, Hk, D = 2 ** 31 // (64 * 4 * 128) + 60, 64, 4, 128
    kc, vc = (torch.zeros(P, S, Hk, D, dtype=BF, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(1)
    n = 300
    k, v = (torch.randn(n, Hk, D, generator=g).to(BF).cuda() for _ in range(2))
    pages = [P - 1, P - 9, P - 3, P - 30, P - 5]
    slots = ints([pages[j // S] * S + j % S for j in range(n)])
    cache.store_kv(k, v, kc, vc, slots)
    assert torch.equal(kc[pages[1], 7], k[S + 7]) and torch.equal(vc[pages[4], 2], v[4 * S + 2])
    small = [torch.zeros(5, S, Hk, D, dtype=BF, device="cuda") for _ in range(2)]
    cache.store_kv(k, v, *small, ints(range(n)))
    for B in (2, 40):
        q = torch.randn(B, 1, 8, D, generator=g).to(BF).cuda()
        own = ints([40 + b for b in range(B)])
        far = cache.prefix_attention(q, kc, vc, ints(pages[:4]), 250, ints([[pages[4], pages[0]]] * B), own)
        near = cache.prefix_attention(q, *small, ints([0, 1, 2, 3]), 250, ints([[4, 0]] * B), own)
        assert torch.equal(far, near) and far.any()


def test_outputs_are_nan_until_the_status_word_is_read():
    """As tests/test_gpu_packed.py: with the prefix in own_kernel and on the tcgen05 kernel."""
    from self_trainable_or_free_attn_b200 import _native as N, cache
    cache.check_status()
    for B in (2, 70):
        own = [40] * B
        q, kc, vc, pages, table = _prefix_case(B, 1, 4, 2, 64, 16, 300, own, BF)
        run = lambda: cache.prefix_attention(q, kc, vc, ints(pages), 300, ints(table), ints(own), return_lse=True)
        good = run()
        N.check(N.load().es_selftest_wait_timeout(2000, N.stream_ptr()), "selftest")
        assert all(torch.isnan(t).all() for t in run())
        with pytest.raises(N.NativeError, match="status 777"):
            cache.check_status()
        assert all(torch.equal(a, b) for a, b in zip(good, run()))
    cache.check_status()


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("N", [1, 3])
def test_prompts_then_tokens(N):
    """A shared prefix and ragged prompts enter the cache, their attention is the packed operator's; then three steps of N tokens each. Every
    output against the definition over the whole sequence of its request."""
    from self_trainable_or_free_attn_b200 import cache, packed
    B, H, Hk, D, page, prefix = 4, 6, 2, 64, 16, 37
    prompts = [1, 50, 16, 31]
    g = torch.Generator().manual_seed(4)
    mk = lambda n, h: torch.randn(n, h, D, generator=g).to(BF).cuda()
    steps = 3
    whole = [prefix + n + steps * N for n in prompts]
    q, k, v = mk(sum(whole), H), mk(sum(whole), Hk), mk(sum(whole), Hk)
    first = starts(whole)
    for b in range(1, B):                                    # the prefix is one for all
        for t in (q, k, v):
            t[first[b]:first[b] + prefix] = t[:prefix]
    want = reference(q, k, v, first, first, True, D ** -0.5)
    kc, vc = (torch.full((64, page, Hk, D), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    free = torch.randperm(64, generator=g).to(torch.int32).cuda()
    zero = ints([0])
    # the prefix is a request of its own
    t0 = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    plan = cache.extend_tables(zero, ints([prefix]), t0, free, page, total=prefix)
    cache.store_kv(k[:prefix], v[:prefix], kc, vc, plan.slots)
    prefix_pages, free = t0[0, :3].contiguous(), free[3:]
    assert plan.taken.tolist() == [3, 0]
    # the prompts: their queries against prefix and prompt
    table, lengths = torch.full((B, 8), -1, dtype=torch.int32, device="cuda"), ints([0] * B)
    at = torch.cat([torch.arange(first[b] + prefix, first[b] + prefix + prompts[b]) for b in range(B)]).cuda()
    plan = cache.extend_tables(lengths, ints(prompts), table, free, page, total=len(at))
    cache.store_kv(k[at], v[at], kc, vc, plan.slots)
    seen = torch.cat([torch.arange(first[b], first[b] + prefix + prompts[b]) for b in range(B)]).cuda()
    cu_k = plan.cu_new + prefix * torch.arange(B + 1, device="cuda", dtype=torch.int32)
    o = packed.packed_attention(q[at], k[seen], v[seen], plan.cu_new, cu_k)
    close("prompts", o, tuple(x[at.cpu()] for x in want["o"]))
    used = int(plan.taken[0])
    lengths, free = plan.lengths, free[used:]
    for s in range(steps):
        plan = cache.extend_tables(lengths, ints([N] * B), table, free, page, total=B * N)
        at = torch.cat([torch.arange(first[b] + prefix + prompts[b] + s * N, first[b] + prefix + prompts[b] + (s + 1) * N) for b in range(B)]).cuda()
        assert plan.positions.tolist() == [prompts[b] + s * N + i for b in range(B) for i in range(N)]
        cache.store_kv(k[at], v[at], kc, vc, plan.slots)
        o = cache.prefix_attention(q[at].view(B, N, H, D), kc, vc, prefix_pages, prefix, table, plan.lengths)
        close("step", o.view(B * N, H, D), tuple(x[at.cpu()] for x in want["o"]))
        lengths, free = plan.lengths, free[int(plan.taken[0]):]


def test_refusals():
    from self_trainable_or_free_attn_b200 import cache
    q, kc, vc, pages, table = _prefix_case(2, 1, 4, 2, 64, 16, 40, [3, 20], BF)
    p, t, n = ints(pages), ints(table), ints([3, 20])
    f = cache.prefix_attention
    for args, error in (((q.cpu(), kc, vc, p, 40, t, n), RuntimeError), ((q, kc.half(), vc, p, 40, t, n), RuntimeError), ((q[0], kc, vc, p, 40, t, n), RuntimeError),
                        ((q, kc, vc[:-1], p, 40, t, n), RuntimeError), ((q, kc, vc, p, 49, t, n), ValueError), ((q, kc, vc, p, -1, t, n), ValueError),
                        ((q, kc[:, :12], vc[:, :12], p, 0, t, n), RuntimeError), ((q[:, :, :3], kc, vc, p, 40, t, n), RuntimeError),
                        ((q, kc, vc, p.cpu(), 40, t, n), RuntimeError), ((q, kc, vc, p, 40, t[:1], n), RuntimeError), ((q, kc, vc, p, 40, t, n[:1]), RuntimeError),
                        ((q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, p, 40, t, n), RuntimeError)):
        with pytest.raises(error):
            f(*args)
    with pytest.raises(RuntimeError, match="no backward"):
        f(q.requires_grad_(True), kc, vc, p, 40, t, n)
    with pytest.raises(RuntimeError):
        cache.extend_tables(n, n[:1], t, p, 16, total=2)
    with pytest.raises(RuntimeError):
        cache.extend_tables(n, n, t.long(), p, 16, total=2)
    with pytest.raises(ValueError):
        cache.extend_tables(n, n, t, p, 0, total=2)
    with pytest.raises(ValueError):
        cache.extend_tables(n, n, t, p, 16, total=-1)
    x = kc[0, :2]
    with pytest.raises(RuntimeError):
        cache.store_kv(x, x[:1], kc, vc, n)
    with pytest.raises(RuntimeError):
        cache.store_kv(x, x, kc, vc, n[:1])
    with pytest.raises(RuntimeError):
        cache.store_kv(x.half(), x.half(), kc, vc, n)
