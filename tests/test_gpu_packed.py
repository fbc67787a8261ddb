"""`packed.packed_attention` against its definition in 64 bits (tests/packed_util.py has the bounds): outputs, LSE and gradients, at the
lengths, head groups, strides and masks where a kernel in tiles goes wrong."""
import pytest
import torch

from packed_util import close, ints, make, reference, starts

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _run(q, k, v, do, cu_q, cu_k, causal, scale=None):
    from self_trainable_or_free_attn_b200 import packed
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o, lse = packed.packed_attention(*leaves, ints(cu_q), None if cu_k is None else ints(cu_k), causal=causal, scale=scale, return_lse=True)
    got = dict(o=o, lse=lse)
    got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))
    return got


def _check(lengths_q, lengths_k, H, Hk, D, dtype, causal, scale=None, **more):
    q, k, v, do, cu_q, cu_k = make(lengths_q, lengths_k, H, Hk, D, dtype, **more)
    got = _run(q, k, v, do, cu_q, cu_k, causal, scale)
    want = reference(q, k, v, cu_q, cu_k, causal, scale or D ** -0.5, do)
    for n in want:
        close(n, got[n], want[n])
    return got, want


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (FP, 128), (FP, 64)])
def test_lengths(dtype, D, causal):
    n = [1, 2, 63, 64, 65, 0, 127, 128, 129, 200, 255, 256, 257, 0, 300]
    _check(n, n, 2, 2, D, dtype, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (FP, 128), (FP, 64)])
@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 2), (5, 1)])
def test_short_sequences_are_as_exact_as_their_type(H, Hk, dtype, D, causal):
    """With up to 32 keys the roundings of P and dS do not average out, and are made up for: what is left is each output's own rounding.

    P and dS keep 16 bits of mantissa at least (2^-17 relative), sums 22: in the norm 2^-7 of an output's own rounding (2^-9 and less) in
    bf16, and in fp16 (whose halves keep 22 bits down to 2^-24) 2^-9 of 2^-12, each as many times as dP stands above dP - delta: 8 here. Added
    in squares that is below 1 %; 5 are allowed."""
    n = [1, 2, 3, 5, 8, 13, 21, 32, 6, 1, 4]
    got, want = _check(n, n, H, Hk, D, dtype, causal, seed=3)
    for name in ("o", "dq", "dk", "dv"):
        exact = want[name][0]
        own = float((exact.to(dtype).double() - exact).norm())
        assert float((got[name].detach().cpu().double() - exact).norm()) <= 1.05 * own, name


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 1), (6, 2), (5, 1), (7, 1), (12, 4), (16, 2), (40, 1), (71, 1), (129, 1), (136, 1)])
def test_head_groups(H, Hk, causal):
    n = [130, 1, 67, 18]
    _check(n, n, H, Hk, 128 if H < 100 else 64, BF, causal, seed=H)


@pytest.mark.parametrize("n", [513, 1000])
@pytest.mark.parametrize("causal", [True, False])
def test_long(n, causal):
    _check([n, 700], [n, 700], 3, 1, 128, BF, causal, seed=n)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_more_keys_than_queries_and_fewer(D, causal):
    """A prompt's next chunk (keys in front), and more queries than keys: causal, the first rows then see none."""
    got, want = _check([1, 5, 130, 40, 260, 3, 0, 7], [400, 300, 131, 20, 100, 0, 9, 1500], 4, 2, D, BF, causal, seed=5)
    if causal:
        empty = torch.isinf(want["lse"][0])
        assert empty.any() and (got["o"].cpu()[empty[0]] == 0).all() and (got["dq"].cpu()[empty[0]] == 0).all()


@pytest.mark.parametrize("behind", [1, 130, 300])
def test_tokens_of_no_sequence(behind):
    """Tokens before the first and behind the last sequence hold NaN: zeros and -inf there, and nothing of it elsewhere."""
    q, k, v, do, cu_q, cu_k = make([70, 140, 1], [70, 140, 1], 4, 2, 128, BF, first=37, behind=behind)
    want = reference(q, k, v, cu_q, cu_k, True, 128 ** -0.5, do)
    for t in (q, k, v, do):
        t[:37] = float("nan")
        t[cu_q[-1]:] = float("inf")
    got = _run(q, k, v, do, cu_q, cu_k, True)
    for n in want:
        close(n, got[n], want[n])
        if n != "lse":
            assert (got[n][:37] == 0).all() and (got[n][cu_q[-1]:] == 0).all()
    assert torch.isinf(got["lse"][:, :37]).all() and torch.isinf(got["lse"][:, cu_q[-1]:]).all()


def test_no_sequences_and_no_tokens():
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, do, _, _ = make([5], [5], 2, 1, 64, BF)
    got = _run(q, k, v, do, [3], None, True)
    assert all((got[n] == 0).all() for n in ("o", "dq", "dk", "dv")) and torch.isinf(got["lse"]).all()
    o, lse = packed.packed_attention(q[:0], k[:0], v[:0], ints([0, 0]), return_lse=True)
    assert o.shape == (0, 2, 64) and lse.shape == (2, 0)
    # queries without any key tensor row
    o, lse = packed.packed_attention(q, k[:0], v[:0], ints([0, 5]), ints([0, 0]), return_lse=True)
    assert (o == 0).all() and torch.isinf(lse).all()
    got = _run(q[:0], k, v, do[:0], [0, 0], [0, 5], True)
    assert (got["dk"] == 0).all() and (got["dv"] == 0).all()


def _bad(t):
    return ~torch.isfinite(t.float().cpu())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("causal", [True, False])
def test_what_is_not_finite_stays_where_it_is_seen(which, value, D, causal):
    """One token of the middle sequence is NaN or infinite: rows that may not see it (other sequences; with the causal mask, the tokens
    before it or the keys behind it) come out as without it, the others not finite."""
    n, H, Hk = [150, 300, 130], 4, 2
    q, k, v, do, cu, _ = make(n, n, H, Hk, D, BF, seed=3)
    clean = _run(q, k, v, do, cu, None, causal)
    at, kh = cu[1] + 140, 1
    x = dict(q=q, k=k, v=v, do=do)
    x[which][at, kh if which in "kv" else 2 * kh] = value
    got = _run(q, k, v, do, cu, None, causal)
    rows = torch.zeros(cu[-1], dtype=torch.bool)             # query rows / key rows that it reaches
    keys = rows.clone()
    if which in ("q", "do"):
        rows[at] = True
        keys[cu[1]:at + 1 if causal else cu[2]] = True
    else:
        rows[at if causal else cu[1]:cu[2]] = True
        keys[cu[1]:cu[2]] = True
    heads = [2 * kh] if which in ("q", "do") else [2 * kh, 2 * kh + 1]
    for h in range(H):
        hit = rows if h in heads else rows & False
        if which != "do":
            assert torch.equal(_bad(got["o"][:, h]).any(1), hit)
        assert torch.equal(_bad(got["dq"][:, h]).any(1), hit)
        assert torch.equal(got["dq"][:, h].cpu()[~hit], clean["dq"][:, h].cpu()[~hit])
        if which != "do":
            assert torch.equal(got["o"][:, h].cpu()[~hit], clean["o"][:, h].cpu()[~hit])
        if which in ("q", "k"):
            assert torch.equal(~torch.isfinite(got["lse"][h].cpu()), hit)
    for h in range(Hk):
        hit = keys if h == kh else keys & False
        assert torch.equal(_bad(got["dk"][:, h]).any(1), hit)
        if which != "v":
            assert torch.equal(_bad(got["dv"][:, h]).any(1), hit)
        for n_ in ("dk", "dv"):
            assert torch.equal(got[n_][:, h].cpu()[~hit], clean[n_][:, h].cpu()[~hit])


@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("causal", [True, False])
def test_what_is_not_finite_where_the_keys_are_shared_out(which, causal):
    """The same with so few tiles that several CTAs share a tile's keys, and several the rows that walk a key tile: parts that are added up."""
    for n_q, n_k, at_q, at_k in (([40, 30], [5000, 3000], 20, 4970), ([1500], [1500], 700, 700)):
        q, k, v, do, cu_q, cu_k = make(n_q, n_k, 8, 1, 128, BF, seed=4)
        clean = _run(q, k, v, do, cu_q, cu_k, causal)
        x = dict(q=q, k=k, v=v, do=do)
        x[which][at_q if which in ("q", "do") else at_k, 0, 3] = float("nan")
        got = _run(q, k, v, do, cu_q, cu_k, causal)
        off = n_k[0] - n_q[0]
        rows, keys = torch.zeros(cu_q[-1], dtype=torch.bool), torch.zeros(cu_k[-1], dtype=torch.bool)
        if which in ("q", "do"):
            rows[at_q] = True
            keys[:at_q + off + 1 if causal else n_k[0]] = True
        else:
            rows[max(0, at_k - off) if causal else 0:n_q[0]] = True
            keys[:n_k[0]] = True
        heads = range(1) if which in ("q", "do") else range(8)
        for h in range(8):
            hit = rows if h in heads else rows & False
            for name in ("o", "dq")[which == "do":]:
                assert torch.equal(_bad(got[name][:, h]).any(1), hit), name
                assert torch.equal(got[name][:, h].cpu()[~hit], clean[name][:, h].cpu()[~hit])
        for name in ("dk", "dv")[:1 if which == "v" else 2]:
            assert torch.equal(_bad(got[name][:, 0]).any(1), keys), name
            assert torch.equal(got[name][:, 0].cpu()[~keys], clean[name][:, 0].cpu()[~keys])


@pytest.mark.parametrize("B", [29, 30, 31, 70, 1100])
@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences(B, causal):
    """Up to 30 sequences are taken longest first, more in their order; empty ones among them."""
    g = torch.Generator().manual_seed(B)
    n = torch.randint(0, 40, (B,), generator=g).tolist()
    n[3], n[B // 2], n[-1] = 300, 0, 0
    _check(n, n, 4, 2, 64, BF, causal, seed=B, first=5, behind=9)


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last sequences against the definition."""
    T, H, D = 2 ** 31 // (64 * 64) + 300, 64, 64
    g = torch.Generator().manual_seed(0)
    tail = [torch.randn(190, H, D, generator=g).to(BF).cuda() for _ in range(4)]
    big = [torch.zeros(T, H, D, dtype=BF, device="cuda") for _ in range(4)]
    for t, x in zip(big, tail):
        t[-190:] = x
    from self_trainable_or_free_attn_b200 import packed
    do = big.pop()
    leaves = [t.requires_grad_(True) for t in big]
    o, lse = packed.packed_attention(*leaves, ints([T - 190, T - 100, T]), return_lse=True)
    grads = torch.autograd.grad(o, leaves, do)
    want = reference(*tail[:3], [0, 90, 190], [0, 90, 190], True, 0.125, tail[3])
    close("o", o[-190:], want["o"])
    close("lse", lse[:, -190:], want["lse"])
    for name, got in zip(("dq", "dk", "dv"), grads):
        close(name, got[-190:], want[name])
        assert not got[:-190].any()
    assert not o[:-190].any()


def test_outputs_are_nan_until_the_status_word_is_read():
    """A kernel that starts while the status word is set (a wait of an earlier one gave up; here the library's self test, a barrier nobody
    arrives on, for 2 ms) leaves NaN in all it owns; check_status raises and clears the word."""
    from self_trainable_or_free_attn_b200 import _native as N, packed
    packed.check_status()
    for n_q, n_k, Hk in (([300, 0, 77], [300, 0, 77], 4), ([20], [3000], 1), ([1500], [1500], 1)):
        q, k, v, do, cu_q, cu_k = make(n_q, n_k, 4, Hk, 128, BF, behind=3)
        good = _run(q, k, v, do, cu_q, cu_k, True)
        N.check(N.load().es_selftest_wait_timeout(2000, N.stream_ptr()), "selftest")
        bad = _run(q, k, v, do, cu_q, cu_k, True)
        assert all(torch.isnan(bad[n]).all() for n in bad)
        with pytest.raises(N.NativeError, match="status 777"):
            packed.check_status()
        again = _run(q, k, v, do, cu_q, cu_k, True)
        assert all(torch.equal(good[n], again[n]) for n in good)
    packed.check_status()


@pytest.mark.parametrize("D", [64, 128])
def test_strides(D):
    """Thirds of a fused projection, head-major tensors, broadcast heads, rows off 16 bytes, and an output gradient of one value."""
    from self_trainable_or_free_attn_b200 import packed
    n = [100, 33]
    cu = starts(n)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(133, 3, 4, D, generator=g).to(BF).cuda()
    major = torch.randn(3, 4, 133, D, generator=g).to(BF).cuda().transpose(1, 2)
    odd = torch.randn(133 * 3 * 4 * D + 1, generator=g).to(BF).cuda()[1:].view(3, 133, 4, D)
    tail = torch.randn(3, 133, 4, D + 4, generator=g).to(BF).cuda()[..., :D]
    wide = torch.randn(3, 133, 1, D, generator=g).to(BF).cuda().expand(-1, -1, 4, -1)
    across = torch.randn(3, 133, D, 4, generator=g).to(BF).cuda().transpose(2, 3)
    for q, k, v in (fused.unbind(1), major.unbind(0), odd.unbind(0), tail.unbind(0), wide.unbind(0), across.unbind(0)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o, lse = packed.packed_attention(*leaves, ints(cu), return_lse=True)
        do = torch.ones((), device="cuda", dtype=BF).expand_as(o)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o, lse=lse)
        want = reference(q, k, v, cu, cu, True, D ** -0.5, do)
        for name in want:
            close(name, got[name], want[name])


def test_one_head_views_with_odd_strides():
    """A dimension of one entry may have any stride: nothing uses it."""
    q, k, v, do, cu, _ = make([50], [50], 1, 1, 64, BF)
    x = [t.as_strided((50, 1, 64), (64, 3, 1)) for t in (q, k, v)]
    got = _run(*x, do, cu, None, True)
    want = reference(q, k, v, cu, cu, True, 0.125, do)
    for n in want:
        close(n, got[n], want[n])


@pytest.mark.parametrize("scale", [0.5, 0.01])
def test_scale(scale):
    _check([90, 200], [90, 200], 2, 1, 64, BF, True, scale=scale)


def test_large_logits():
    """Logits of some hundred, growing along the keys: every tile raises the running maximum. The 64-bit result of such rows is
    one key's value, or two keys' whose logits differ in the last place of a 32-bit sum: only rows with a clear maximum are compared."""
    q, k, v, do, cu, _ = make([400], [400], 1, 1, 128, BF)
    k *= torch.linspace(0.2, 12.0, 400, device="cuda")[:, None, None].to(BF)
    q *= 4
    got = _run(q, k, v, do, cu, None, False)
    S = (q[:, 0].double() @ k[:, 0].double().T).cpu() * 128 ** -0.5
    top = S.topk(2, -1)
    clear = top.values[:, 0] - top.values[:, 1] > 20.0          # the second key weighs less than 2^-28
    assert clear.sum() > 100 and torch.isfinite(got["o"].float()).all()
    assert torch.equal(got["o"][:, 0].cpu()[clear], v[:, 0].cpu()[top.indices[clear, 0]])
    # a logit's 32-bit sum is off by less than 128 * 2^-24 of the terms' absolute sum, here under 2^12: 2^-5 at most
    assert (got["lse"][0].double().cpu() - torch.logsumexp(S, -1)).abs().max() <= 2.0 ** -5


def test_gradients_against_differences():
    """The directional derivative of sum(O dO) along random directions, by central differences in 64 bits: of fourth order, step 1e-3,
    exact to 1e-9 of the scale here; the kernels' gradients may be off by their bounds summed along the direction."""
    q, k, v, do, cu, _ = make([60, 90], [60, 90], 4, 2, 64, BF)
    got = _run(q, k, v, do, cu, None, True)
    want = reference(q, k, v, cu, cu, True, 0.125, do)
    x = {n: t.double().cpu() for n, t in (("q", q), ("k", k), ("v", v))}

    def loss(y):
        return (reference(y["q"], y["k"], y["v"], cu, cu, True, 0.125)["o"][0] * do.double().cpu()).sum()

    g = torch.Generator().manual_seed(2)
    for n in "qkv":
        d = torch.randn(x[n].shape, generator=g).double()
        at = lambda h: loss({**x, n: x[n] + h * d})
        h = 1e-3
        slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        assert abs((want["d" + n][0] * d).sum() - slope) <= 1e-7 * (1 + abs(slope))
        bound = (want["d" + n][1] * d.abs()).sum()
        assert abs((got["d" + n].double().cpu() * d).sum() - slope) <= bound + 1e-7 * (1 + abs(slope))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,H,Hk", [(128, 24, 4), (64, 5, 1), (64, 2, 2)])
def test_rows_that_see_one_key(D, H, Hk, causal):
    """Their P is 1 whatever the logit: dQ, and what they add to dK, is 0 exactly, and not what rounding leaves of a difference."""
    q, k, v, do, cu, _ = make([1] * 40, [1] * 40, H, Hk, D, BF)
    got = _run(q, k, v, do, cu, None, causal)
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all()
    q, k, v, do, cu_q, cu_k = make([5, 1, 3, 200], [1, 1, 3, 150], H, Hk, D, BF)
    got = _run(q, k, v, do, cu_q, cu_k, causal)
    first = [4, 5, 6, 9 + 50] if causal else [0, 1, 2, 3, 4, 5]
    assert (got["dq"][first] == 0).all() and (got["dk"][:2] == 0).all() and (got["dq"][-1] != 0).any()
    want = reference(q, k, v, cu_q, cu_k, causal, D ** -0.5, do)
    for n in want:
        close(n, got[n], want[n])


def test_same_bits_twice_and_partial_gradients():
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, do, cu, _ = make([300, 77, 140], [300, 77, 140], 6, 2, 128, BF)
    one, two = _run(q, k, v, do, cu, None, True), _run(q, k, v, do, cu, None, True)
    assert all(torch.equal(one[n], two[n]) for n in one)
    for n, t in (("dq", q), ("dk", k), ("dv", v)):
        leaf = t.detach().requires_grad_(True)
        args = [leaf if x is t else x for x in (q, k, v)]
        g, = torch.autograd.grad(packed.packed_attention(*args, ints(cu)), leaf, do)
        assert torch.equal(g, one[n])
    # a second backward through the same graph, and a refused derivative of the derivative
    leaf = q.detach().requires_grad_(True)
    o = packed.packed_attention(leaf, k, v, ints(cu))
    a, = torch.autograd.grad(o, leaf, do, retain_graph=True)
    b, = torch.autograd.grad(o, leaf, do, create_graph=True)
    assert torch.equal(a, one["dq"]) and torch.equal(b, one["dq"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(b.float().sum(), leaf)


def test_int64_starts_and_wrong_starts_stay_in_bounds():
    """int64 starts are taken; starts outside the tensor are clamped."""
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, do, cu, _ = make([30, 40], [30, 40], 2, 2, 64, BF)
    want = packed.packed_attention(q, k, v, ints(cu))
    assert torch.equal(packed.packed_attention(q, k, v, ints(cu).long()), want)
    assert torch.equal(packed.packed_attention(q, k, v, ints([-9, 30, 1000])), want)


def test_on_another_stream():
    q, k, v, do, cu, _ = make([300, 200], [300, 200], 4, 2, 128, BF)
    want = _run(q, k, v, do, cu, None, True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = [torch.empty_like(t).copy_(t) for t in (q, k, v)]
        got = _run(*late, do, cu, None, True)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_captured_forward_and_backward_follow_the_starts():
    """A captured step replayed with other lengths in the same starts tensor and other values; a second graph beside it."""
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, do, cu, _ = make([100, 156], [100, 156], 4, 2, 64, BF)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    at = ints(cu)

    def step():
        o, lse = packed.packed_attention(*leaves, at, return_lse=True)
        return (o.detach(), lse, *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for cu2 in ([0, 100, 256], [0, 1, 256], [0, 250, 256]):
        at.copy_(ints(cu2))
        with torch.no_grad():
            leaves[0].copy_(torch.randn(q.shape, device="cuda").to(BF))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = _run(*leaves, do, cu2, None, True)
        for out in outs:
            assert all(torch.equal(a, want[n]) for a, n in zip(out, ("o", "lse", "dq", "dk", "dv")))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_another_device():
    q, k, v, do, cu, _ = make([100, 56], [100, 56], 4, 2, 64, BF)
    want = _run(q, k, v, do, cu, None, True)
    from self_trainable_or_free_attn_b200 import packed
    x = [t.to("cuda:1").requires_grad_(True) for t in (q, k, v)]
    o = packed.packed_attention(*x, ints(cu).to("cuda:1"))
    assert torch.equal(o.cpu(), want["o"].cpu())
    assert torch.equal(torch.autograd.grad(o, x, do.to("cuda:1"))[1].cpu(), want["dk"].cpu())


def test_refusals():
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, do, cu, _ = make([30], [30], 4, 2, 64, BF)
    c = ints(cu)
    f = packed.packed_attention
    for args, error in (((q.cpu(), k, v, c), RuntimeError), ((q, k.half(), v, c), RuntimeError), ((q.float(), k.float(), v.float(), c), RuntimeError),
                        ((q[None], k, v, c), RuntimeError), ((q, k, v[:, :1], c), RuntimeError), ((q[:, :3], k, v, c), RuntimeError),
                        ((q[..., :32], k[..., :32], v[..., :32], c), RuntimeError), ((q, k[:20], v[:20], c), RuntimeError), ((q, k, v, c.cpu()), RuntimeError),
                        ((q, k, v, c.float()), RuntimeError), ((q, k, v, c, ints([0, 1, 2])), RuntimeError), ((q, k, v, c[:0]), RuntimeError)):
        with pytest.raises(error):
            f(*args)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            f(q, k, v, c, scale=scale)
