"""The softmax scale: what 32 bits hold as a normal number with room for log2(e) is taken, the rest is refused, in Python and by the C ABI."""
import pytest
import torch

from packed_util import close, ints, make, reference
from test_packed_cpu import _bwd, _fwd, _prefix

BF = torch.bfloat16
REFUSED = [0.0, -1.0, float("nan"), float("inf"), 1e-50, 1e-45, 1e-39, 2.0 ** 127, 3e38, 1e39, 1e300]


def test_scales():
    from self_trainable_or_free_attn_b200.packed import softmax_scale
    for scale in (2.0 ** -126, 0.3, 1, 2.0 ** 126):
        assert softmax_scale(scale, 64) == scale
    assert softmax_scale(None, 64) == 0.125
    for scale in REFUSED:
        with pytest.raises(ValueError):
            softmax_scale(scale, 64)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: without a GPU no call can reach a kernel with them")
@pytest.mark.parametrize("name,make_args", [("es_packed_attn_fwd", _fwd), ("es_packed_attn_bwd", _bwd), ("es_prefix_attn", _prefix)])
def test_the_c_abi_refuses_them_too(name, make_args):
    from self_trainable_or_free_attn_b200 import _native
    fn = getattr(_native.load(), name)
    for scale in (2.0 ** -126, 2.0 ** 126):
        assert fn(*make_args(scale=scale).values()) < -1, "stopped by nothing but the missing GPU"
    for scale in REFUSED:
        assert fn(*make_args(scale=scale).values()) == -1 and name in _native.last_error() and "scale" in _native.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -60])
def test_the_smallest(scale):
    """Every visible key weighs the same; the gradients of q and k are below what the type holds, and no NaN."""
    from self_trainable_or_free_attn_b200 import packed
    q, k, v, do, cu, _ = make([150, 20], [150, 20], 2, 1, 64, BF)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o, lse = packed.packed_attention(*x, ints(cu), scale=scale, return_lse=True)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, x, do)), o=o, lse=lse)
    want = reference(q, k, v, cu, cu, True, scale, do)
    for n in ("o", "lse", "dv"):
        close(n, got[n], want[n])
    for n in ("dq", "dk"):
        assert torch.isfinite(got[n].float()).all() and got[n].float().abs().max() <= scale * 2 ** 16
