"""Whole numbers in int64 that 32 bits do not hold: they keep their side of every bound (a slot or page that is not of the cache, a start behind
the last token) and are not wrapped to a number that means something else."""
import pytest
import torch

BF = torch.bfloat16
FAR = [2 ** 32, 2 ** 32 + 5, 2 ** 31, 2 ** 40 + 1, 2 ** 63 - 1]
BELOW = [-2 ** 32, -2 ** 32 + 3, -2 ** 31 - 1, -2 ** 63]


def test_narrowing_keeps_the_order():
    from self_trainable_or_free_attn_b200.packed import check_ints
    x = torch.tensor(BELOW + [-2 ** 31, -1, 0, 7, 2 ** 31 - 1] + FAR)
    got, = check_ints(x, x=x)
    assert got.dtype == torch.int32 and got.tolist() == [max(-2 ** 31, min(n, 2 ** 31 - 1)) for n in x.tolist()]
    assert check_ints(got, x=got)[0] is got
    with pytest.raises(RuntimeError):
        check_ints(x, x=x.to(torch.int16))


@pytest.mark.gpu
def test_slots_and_pages_and_lengths():
    from self_trainable_or_free_attn_b200 import cache
    long = lambda x: torch.tensor(x, dtype=torch.int64, device="cuda")
    g = torch.Generator().manual_seed(0)
    kc, vc = (torch.randn(6, 16, 2, 64, generator=g).to(BF).cuda() for _ in range(2))
    was = kc.clone(), vc.clone()
    k = torch.zeros(len(FAR + BELOW), 2, 64, dtype=BF, device="cuda")
    cache.store_kv(k, k, kc, vc, long(FAR + BELOW))
    assert torch.equal(kc, was[0]) and torch.equal(vc, was[1])
    q = torch.randn(1, 1, 4, 64, generator=g).to(BF).cuda()
    want = cache.prefix_attention(q, kc, vc, long([1, -1, 2]), 48, long([[3, -1]]), long([32]))
    for far in FAR + BELOW:
        assert torch.equal(cache.prefix_attention(q, kc, vc, long([1, far, 2]), 48, long([[3, far]]), long([32])), want)
    whole, none = (cache.prefix_attention(q, kc, vc, long([1]), 16, long([[3, 4]]), long([n])) for n in (32, 0))
    assert not torch.equal(whole, none)
    for far, expect in [(n, whole) for n in FAR] + [(n, none) for n in BELOW]:
        assert torch.equal(cache.prefix_attention(q, kc, vc, long([1]), 16, long([[3, 4]]), long([far])), expect)


@pytest.mark.gpu
def test_starts():
    from self_trainable_or_free_attn_b200 import packed
    long = lambda x: torch.tensor(x, dtype=torch.int64, device="cuda")
    q, k, v = (torch.randn(70, 2, 64, generator=torch.Generator().manual_seed(i)).to(BF).cuda() for i in range(3))
    want = packed.packed_attention(q, k, v, long([0, 30, 70]))
    for far in FAR:
        for below in BELOW:
            assert torch.equal(packed.packed_attention(q, k, v, long([below, 30, far])), want)


@pytest.mark.gpu
def test_sizes_that_the_library_takes_in_32_bits():
    """A page of 2^32 + 16 tokens is not one of 16, nor is a prefix of 2^32 + 8 tokens one of 8."""
    from self_trainable_or_free_attn_b200 import cache
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for page in (2 ** 31, 2 ** 32 + 16):
        with pytest.raises(ValueError):
            cache.extend_tables(i([0]), i([3]), i([[-1]]), i([4]), page, total=3)
    plan = cache.extend_tables(i([0]), i([3]), i([[-1]]), i([0]), 2 ** 31 - 1, total=3)
    assert plan.slots.tolist() == [0, 1, 2]
    q, kc = torch.zeros(1, 1, 1, 64, dtype=BF, device="cuda"), torch.zeros(1, 256, 1, 64, dtype=BF, device="cuda")
    pages = torch.zeros(2 ** 24 + 1, dtype=torch.int32, device="cuda")
    for n in (2 ** 31 - 256, 2 ** 31, 2 ** 32 + 8):
        with pytest.raises(ValueError):
            cache.prefix_attention(q, kc, kc, pages, n, i([[0]]), i([0]))
