"""What rounding O left, which the forward keeps in training for the row sums of the backward: as the forward writes it where a row's keys are one
CTA's, where they are shared out and joined, and in the gradients.

Values with a mean (V about 3, K about 2) make O's own rounding the largest error there is. What may be left of it, in the root of the mean of the squares
over rows and columns, u = eps / 2 of the type and independent roundings of P (each at most u relative; in fp16 also half of 2^-24):

  O + rest   u sqrt(sum_j P^2 V^2) + grid sqrt(sum V^2), the rest's own rounding u^2 |O|, and 32-bit sums: a step of 16 products adds at most 2^-23 of the
             sum so far, n / 16 steps and 64 for what is joined; logits 2^-17
  dQ         scale (u sqrt(sum dS^2 K^2) + |sum_j P K| e), e = u sqrt(sum P^2 dP^2) + the 32-bit part of O + rest times sum |dO|; its own rounding u |dQ|
"""
import pytest
import torch

from packed_util import grid, ints, make, unit

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rms(x):
    return float(x.double().square().mean().sqrt())


def _case(n_q, n_k, H, Hk, D, dtype):
    q, k, v, do, cu_q, cu_k = make(n_q, n_k, H, Hk, D, dtype, seed=7)
    return q, (k.float() + 2).to(dtype), (v.float() + 3).to(dtype), do, cu_q, cu_k


def _exact(q, k, v, do, cu_q, cu_k, causal, scale):
    """Per sequence and head in 64 bits: rows, head, P, Q, K, V, dO."""
    q, k, v, do = (t.double().cpu() for t in (q, k, v, do))
    for b in range(len(cu_q) - 1):
        r, c = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        nq, nk = r.stop - r.start, c.stop - c.start
        seen = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool)
        for h in range(q.shape[1]):
            kh = h // (q.shape[1] // k.shape[1])
            S = (scale * q[r, h] @ k[c, kh].T).masked_fill(~seen, -torch.inf)
            yield r, h, torch.softmax(S, -1), q[r, h], k[c, kh], v[c, kh], do[r, h]


SHARED = ([20], [3000], True)                                # a few queries on many keys: the keys are shared out
TILES = ([700, 900, 20, 650, 333], [900] * 5, False)


def _tells(n_q, n_k, causal):
    """Whether O without the rest has to be off by more than the bound: not where a causal row sees one key, or few, as sqrt(sum P^2 V^2) is |O| there and the
    bound is what O's rounding is."""
    return not causal or all(k - q >= 64 for q, k in zip(n_q, n_k))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n_q,n_k,shared", [SHARED, TILES])
def test_output_and_rest(n_q, n_k, shared, causal, D, dtype):
    from self_trainable_or_free_attn_b200 import _native as N, packed
    H, Hk = (4, 2) if shared else (32, 32)
    q, k, v, do, cu_q, cu_k = _case(n_q, n_k, H, Hk, D, dtype)
    sizes = (len(n_q), q.shape[0], k.shape[0], H, Hk, D)
    assert (N.load().es_packed_fwd_workspace_bytes(*sizes) > 0) == shared
    o, rest, _ = packed._fwd(q, k, v, ints(cu_q), ints(cu_k), D ** -0.5, int(causal), True)
    o, rest, u, g = o.double().cpu(), rest.double().cpu(), unit(dtype), grid(dtype)
    off, alone, first, second, size = [], [], [], [], []
    for r, h, P, _, _, V, _ in _exact(q, k, v, do, cu_q, cu_k, causal, D ** -0.5):
        if h % 4 and not shared:
            continue
        O = P @ V
        off.append(o[r, h] + rest[r, h] - O)
        alone.append(o[r, h] - O)
        first.append(P.square() @ V.square())
        second.append(V.square().sum(0, keepdim=True).expand_as(O))
        size.append(P @ V.abs())
    off, alone, first, second, size = (torch.cat(x) for x in (off, alone, first, second, size))
    bound = u * float(first.mean().sqrt()) + g * float(second.mean().sqrt()) + (u * u + (max(n_k) / 16 + 64) * 2.0 ** -23 + 2.0 ** -17) * rms(size)
    print(f"rms of what is left {rms(off):.2e}, bound {bound:.2e}, O alone {rms(alone):.2e}")
    assert rms(off) <= bound
    assert rms(alone) > 2 * bound or not _tells(n_q, n_k, causal), "the case does not tell"


def _dq(q, k, v, o, rest, do, lse, cu_q, cu_k, scale, causal):
    """The backward's C entry point, dQ alone, with the rest or without."""
    from self_trainable_or_free_attn_b200 import _native as N, packed
    (T, H, D), (Tk, Hk, _) = q.shape, k.shape
    sizes = (cu_q.shape[0] - 1, T, Tk, H, Hk, D)
    dq, ws = torch.empty_like(q), packed._workspace("es_packed_bwd_workspace_bytes", q, sizes)
    packed._call("es_packed_attn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), N.ptr(rest), do.data_ptr(), lse.data_ptr(), dq.data_ptr(), None, None,
                 cu_q.data_ptr(), cu_k.data_ptr(), *sizes, *packed.strides(q), *packed.strides(k), *packed.strides(v), *packed.strides(do), scale, causal,
                 packed._DTYPES[q.dtype], N.ptr(ws), N.stream_ptr())
    return dq


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n_q,n_k,shared", [SHARED, TILES])
def test_gradient_of_the_queries(n_q, n_k, shared, causal, D):
    from self_trainable_or_free_attn_b200 import packed
    H, Hk = (4, 2) if shared else (32, 32)
    q, k, v, do, cu_q, cu_k = _case(n_q, n_k, H, Hk, D, BF)
    at, scale, u = (ints(cu_q), ints(cu_k)), D ** -0.5, unit(BF)
    leaf = q.clone().requires_grad_(True)
    dq, = torch.autograd.grad(packed.packed_attention(leaf, k, v, *at, causal=causal), leaf, do)
    o, rest, lse = packed._fwd(q, k, v, *at, scale, int(causal), True)
    assert torch.equal(_dq(q, k, v, o, rest, do, lse, *at, scale, int(causal)), dq)
    without = _dq(q, k, v, o, None, do, lse, *at, scale, int(causal)).double().cpu()
    dq = dq.double().cpu()
    off, alone, bound = [], [], []
    for r, h, P, Q, K, V, dO in _exact(q, k, v, do, cu_q, cu_k, causal, scale):
        if h % 4 and not shared:
            continue
        dP, O = dO @ V.T, P @ V
        dS = P * (dP - (dO * O).sum(-1, keepdim=True))
        want = scale * dS @ K
        off.append(dq[r, h] - want)
        alone.append(without[r, h] - want)
        narrow = (max(n_k) / 16 + 64) * 2.0 ** -23 + 2.0 ** -17
        e = u * (P.square() * dP.square()).sum(-1, keepdim=True).sqrt() + (narrow + u * u) * ((P @ V.abs()) * dO.abs()).sum(-1, keepdim=True)
        bound.append((scale * (u * (dS.square() @ K.square()).sqrt() + (P @ K).abs() * e + narrow * (dS.abs() @ K.abs())) + u * want.abs()))
    off, alone, bound = rms(torch.cat(off)), rms(torch.cat(alone)), rms(torch.cat(bound))
    print(f"rms of dQ's error {off:.2e}, bound {bound:.2e}, without the rest {alone:.2e}")
    assert off <= bound
    assert alone > 1.5 * bound or not _tells(n_q, n_k, causal), "the case does not tell"
