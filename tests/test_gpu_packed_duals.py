"""Forward-mode derivatives: the operators for packed sequences and for a paged cache have none, and say so instead of dropping a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

BF = torch.bfloat16


def _tensors(device):
    mk = lambda *shape: torch.ones(*shape, dtype=BF, device=device)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return dict(q=mk(4, 2, 64), k=mk(4, 2, 64), v=mk(4, 2, 64), k_cache=mk(3, 16, 2, 64), v_cache=mk(3, 16, 2, 64)), i


def _calls(device):
    from self_trainable_or_free_attn_b200 import cache, packed
    _, i = _tensors(device)
    return ((("q", "k", "v"), lambda t: packed.packed_attention(t["q"], t["k"], t["v"], i([0, 4]))),
            (("k", "v", "k_cache", "v_cache"), lambda t: cache.store_kv(t["k"], t["v"], t["k_cache"], t["v_cache"], i([0, 1, 2, 40]))),
            (("q", "k_cache", "v_cache"), lambda t: cache.prefix_attention(t["q"][:, None], t["k_cache"], t["v_cache"], i([0]), 9, i([[1]] * 4), i([1] * 4))))


def _check(device):
    for names, call in _calls(device):
        for name in names:
            t, _ = _tensors(device)
            with forward_ad.dual_level():
                t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
                with pytest.raises(NotImplementedError, match="tangent"):
                    call(t)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                    call(t)


def test_a_tangent_is_refused_before_anything_else():
    _check("cpu")


@pytest.mark.gpu
def test_a_tangent_is_refused():
    from self_trainable_or_free_attn_b200 import packed
    _check("cuda")
    t, i = _tensors("cuda")
    for grad in (False, True):                               # with a gradient wanted as well; then without tangents inside a level, as outside
        with forward_ad.dual_level():
            q = forward_ad.make_dual(t["q"].clone().requires_grad_(grad), torch.ones_like(t["q"]))
            with pytest.raises(NotImplementedError):
                packed.packed_attention(q, t["k"], t["v"], i([0, 4]))
            inside = packed.packed_attention(t["q"], t["k"], t["v"], i([0, 4]))
        assert torch.equal(inside, packed.packed_attention(t["q"], t["k"], t["v"], i([0, 4])))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: packed.packed_attention(q, t["k"], t["v"], i([0, 4])), (t["q"],), (t["q"],))
