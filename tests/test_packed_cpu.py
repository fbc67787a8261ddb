"""The entry points for packed sequences and the paged cache without a GPU: what they refuse is refused before any launch, by the
Python layer and by the C ABI, and the layout checks say what they should."""
import ctypes

import pytest
import torch

BIG = 0x10000


def _fwd(**over):
    a = dict(q=BIG, k=2 * BIG, v=3 * BIG, o=4 * BIG, rest=8 * BIG, lse=5 * BIG, cu_q=6 * BIG, cu_k=7 * BIG, B=2, Tq=10, Tk=12, H=4, Hk=2, D=64,
             qt=256, qh=64, kt=128, kh=64, vt=128, vh=64, scale=0.1, causal=1, dtype=0, ws=9 * BIG, st=None)
    a.update(over)
    return a


def _bwd(**over):
    a = dict(q=BIG, k=2 * BIG, v=3 * BIG, o=4 * BIG, rest=None, do=5 * BIG, lse=6 * BIG, dq=7 * BIG, dk=8 * BIG, dv=9 * BIG, cu_q=10 * BIG, cu_k=11 * BIG, B=2,
             Tq=10, Tk=12, H=4, Hk=2, D=64, qt=256, qh=64, kt=128, kh=64, vt=128, vh=64, dt=256, dh=64, scale=0.1, causal=1, dtype=0, ws=12 * BIG, st=None)
    a.update(over)
    return a


def _prefix(**over):
    a = dict(q=BIG, k=2 * BIG, v=3 * BIG, o=4 * BIG, lse=5 * BIG, pages=6 * BIG, np=3, plen=40, table=7 * BIG, width=4, lengths=8 * BIG, B=2, N=1,
             H=4, Hk=2, D=64, P=20, page=16, kp=2048, kt=128, kh=64, vp=2048, vt=128, vh=64, scale=0.1, dtype=0, ws=9 * BIG, st=None)
    a.update(over)
    return a


def _extend(**over):
    a = dict(lengths=BIG, new=2 * BIG, table=3 * BIG, free=4 * BIG, nf=5, B=2, width=4, page=16, total=7, slots=5 * BIG, pos=6 * BIG, cu=7 * BIG,
             out=8 * BIG, taken=9 * BIG, st=None)
    a.update(over)
    return a


def _store(**over):
    a = dict(k=BIG, v=2 * BIG, kc=3 * BIG, vc=4 * BIG, slots=5 * BIG, T=7, Hk=2, D=64, P=20, page=16, kt=128, kh=64, vt=128, vh=64, kcp=2048, kct=128,
             kch=64, vcp=2048, vct=128, vch=64, st=None)
    a.update(over)
    return a


SIZES = [dict(B=-1), dict(Tq=-1), dict(Tk=-1), dict(Tq=0x7FFFFF00), dict(H=0), dict(H=3), dict(Hk=0), dict(D=96), dict(dtype=2)]
REFUSED = (
    [("es_packed_attn_fwd", _fwd, x) for x in SIZES + [dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(lse=None), dict(cu_q=None), dict(cu_k=None),
                                                       dict(q=BIG + 8), dict(k=BIG + 8), dict(v=BIG + 2), dict(o=BIG + 16), dict(rest=BIG + 8), dict(ws=BIG + 16), dict(qt=257), dict(kh=60), dict(vt=4)]]
    + [("es_packed_attn_bwd", _bwd, x) for x in SIZES + [dict(q=None), dict(k=None), dict(o=None), dict(do=None), dict(lse=None), dict(dk=None), dict(dv=None), dict(cu_q=None),
                                                         dict(cu_k=None), dict(ws=None), dict(do=BIG + 8), dict(rest=BIG + 8), dict(dq=BIG + 16), dict(dk=BIG + 16), dict(ws=BIG + 16),
                                                         dict(dt=4), dict(qh=65)]]
    + [("es_prefix_attn", _prefix, x) for x in [dict(B=-1), dict(N=-1), dict(H=3), dict(D=32), dict(dtype=9), dict(page=48), dict(page=512), dict(plen=49), dict(plen=-1),
                                                dict(width=-1), dict(P=-1), dict(np=-1), dict(P=2 ** 30), dict(width=2 ** 28), dict(q=None), dict(k=None), dict(o=None),
                                                dict(lse=None), dict(pages=None), dict(table=None), dict(lengths=None), dict(q=BIG + 8), dict(v=BIG + 8), dict(o=BIG + 4),
                                                dict(kp=2047), dict(vh=4)]]
    + [("es_extend_tables", _extend, x) for x in [dict(nf=-1), dict(B=-1), dict(width=-1), dict(page=0), dict(total=-1), dict(lengths=None), dict(new=None), dict(table=None),
                                                  dict(free=None), dict(slots=None), dict(pos=None), dict(cu=None), dict(out=None), dict(taken=None)]]
    + [("es_store_kv", _store, x) for x in [dict(T=-1), dict(Hk=0), dict(D=80), dict(P=-1), dict(page=0), dict(P=2 ** 30), dict(k=None), dict(vc=None), dict(slots=None),
                                            dict(k=BIG + 8), dict(kc=BIG + 8), dict(kt=4), dict(vcp=2050)]])
GOOD = {"es_packed_attn_fwd": _fwd, "es_packed_attn_bwd": _bwd, "es_prefix_attn": _prefix, "es_extend_tables": _extend, "es_store_kv": _store}


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: without a GPU no call can reach a kernel with them")
@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused_before_any_launch(i):
    from self_trainable_or_free_attn_b200 import _native
    name, make, over = REFUSED[i]
    fn, before = getattr(_native.load(), name), _native.launch_count()
    assert fn(*GOOD[name]().values()) < -1, "the good call is stopped by nothing but the missing GPU"
    assert fn(*make(**over).values()) == -1, (name, over)
    assert name in _native.last_error() and _native.launch_count() == before


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up")
def test_empty_calls_return_at_once():
    from self_trainable_or_free_attn_b200 import _native
    lib = _native.load()
    assert lib.es_packed_attn_fwd(*_fwd(Tq=0).values()) == 0
    assert lib.es_packed_attn_bwd(*_bwd(Tq=0, Tk=0).values()) == 0
    assert lib.es_packed_attn_bwd(*_bwd(dq=None, dk=None, dv=None).values()) == 0
    assert lib.es_packed_attn_bwd(*_bwd(Tk=0, dq=None).values()) == 0
    assert lib.es_prefix_attn(*_prefix(B=0).values()) == 0
    assert lib.es_store_kv(*_store(T=0).values()) == 0


def test_no_cpu_path():
    from self_trainable_or_free_attn_b200 import cache, packed
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        packed.packed_attention(q, q, q, cu)
    kc = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.prefix_attention(q[:, None], kc, kc, cu, 0, cu[None], cu)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.store_kv(q, q, kc, kc, cu)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.extend_tables(cu, cu, torch.zeros(2, 3, dtype=torch.int32), cu, 16, total=1)


def test_layouts():
    from self_trainable_or_free_attn_b200.packed import rows, strides, usable
    x = torch.zeros(10, 3, 4, 64, dtype=torch.bfloat16)
    for t, ok in ((x[:, 0], True), (x[:, 0].transpose(0, 1), True), (x[..., :32].flatten(0, 1), True), (x[:, 0, :, ::2], False), (torch.zeros(10, 64, 4, dtype=torch.bfloat16).transpose(1, 2), False),
                  (x[:, 0, :1].expand(-1, 4, -1), False), (torch.zeros(641, dtype=torch.bfloat16)[1:].view(10, 1, 64), False),
                  (torch.zeros(10, 4, 68, dtype=torch.bfloat16)[..., :64], False), (torch.zeros(10, 1, 64, dtype=torch.bfloat16).as_strided((10, 1, 64), (64, 3, 1)), True)):
        assert usable(t) == ok, (t.shape, t.stride())
        r = rows(t)
        assert usable(r) and torch.equal(r, t) and (r is t) == ok
    assert strides(torch.zeros(10, 1, 64).as_strided((10, 1, 64), (64, 3, 1))) == (64, 64)
    assert strides(x[:, 1]) == (768, 64)
    assert strides(torch.zeros(1, 1, 64).as_strided((1, 1, 64), (1, 1, 1))) == (64, 64)


def test_reference_gradients_against_autograd():
    """The 64-bit definition that the GPU tests compare with, against torch's own derivative of its forward."""
    from packed_util import make, reference, starts
    q, k, v, do, cu_q, cu_k = make([5, 0, 9], [7, 3, 4], 4, 2, 64, torch.bfloat16, first=2, behind=3, device="cpu")
    want = reference(q, k, v, cu_q, cu_k, True, 0.125, do)
    x = [t.double().requires_grad_(True) for t in (q, k, v)]
    total = 0.0
    for b in range(3):
        for i in range(cu_q[b], cu_q[b + 1]):
            n = cu_k[b] + (i - cu_q[b]) + (cu_k[b + 1] - cu_k[b]) - (cu_q[b + 1] - cu_q[b]) + 1
            if n <= cu_k[b]:
                continue
            for h in range(4):
                p = torch.softmax(0.125 * x[1][cu_k[b]:n, h // 2] @ x[0][i, h], 0)
                o = p @ x[2][cu_k[b]:n, h // 2]
                assert torch.allclose(o, want["o"][0][i, h], rtol=1e-12, atol=1e-12)
                total = total + (o * do[i, h].double()).sum()
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(total, x)):
        assert torch.allclose(g, want[name][0], rtol=1e-10, atol=1e-10)
