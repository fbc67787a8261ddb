"""Attention over packed sequences in 64 bits, by the definition, with a bound on what the kernels' roundings may change.

The kernels round P and dS to the element type before they multiply with them, and every output once: u = eps / 2 relative each. In
fp16, values under 2^-14 are rounded to a grid of 2^-24 instead, half of which is `grid`. What is computed in 32 bits (scores of up to 128 products, exponentials,
sums) is off by less than 2^-12 of the terms' absolute sum: logits below 64, products' sums to 128 * 2^-24 of their absolute sum.

  O    u (|O| + sum_j P |V|),  + grid sum_j |V|
  dV   u (|dV| + sum_i P |dO|), + grid sum_i |dO|
  dS   u (|dS| + P e_i) + grid, e_i = |delta_i - delta_i exact| / u <= sum_c |dO| (|O| + sum_j P |V|): delta is made of the rounded O
  dQ, dK  u |.| + scale * (the error of dS) times |K|, |Q|
"""
import torch

SLACK = 2.0 ** -12


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def grid(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def reference(q, k, v, cu_q, cu_k, causal, scale, dout=None):
    """{name: (value, bound)} of o, lse (and dq, dk, dv), on the CPU in float64; cu as lists."""
    u, g = unit(q.dtype), grid(q.dtype)
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    do = None if dout is None else dout.detach().double().cpu()
    (T, H, D), (Tk, Hk, _) = q.shape, k.shape
    out = {"o": torch.zeros(T, H, D).double(), "lse": torch.full((H, T), -torch.inf).double()}
    tol = {"o": torch.zeros(T, H, D).double(), "lse": torch.full((H, T), 64 * 2.0 ** -20).double()}
    if do is not None:
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            out[n], tol[n] = torch.zeros_like(t), torch.zeros_like(t)
    for b in range(len(cu_q) - 1):
        r, c = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        nq, nk = r.stop - r.start, c.stop - c.start
        if nq <= 0 or nk <= 0:
            continue
        seen = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            seen = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq)
        for h in range(H):
            kh = h // (H // Hk)
            Q, K, V = q[r, h], k[c, kh], v[c, kh]
            S = (scale * Q @ K.T).masked_fill(~seen, -torch.inf)
            z = torch.logsumexp(S, -1)
            P = torch.where(seen, torch.exp(S - z[:, None]), 0.0).nan_to_num(0.0)
            Pv = P @ V.abs()
            out["o"][r, h], out["lse"][h, r] = P @ V, z
            eo = u * ((P @ V).abs() + Pv) + SLACK * Pv + g * (seen.double() @ V.abs())
            tol["o"][r, h] = eo
            if do is None:
                continue
            dO = do[r, h]
            dP, delta = dO @ V.T, (dO * out["o"][r, h]).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            e = (dO.abs() * eo).sum(-1, keepdim=True)
            eS = u * dS.abs() + P * (e + SLACK * (dO.abs() @ V.abs().T + delta.abs())) + g * seen
            out["dq"][r, h] = scale * dS @ K
            tol["dq"][r, h] = scale * eS @ K.abs() + u * out["dq"][r, h].abs() + SLACK * scale * dS.abs() @ K.abs()
            out["dk"][c, kh] += scale * dS.T @ Q
            tol["dk"][c, kh] += scale * eS.T @ Q.abs() + SLACK * scale * dS.abs().T @ Q.abs()
            out["dv"][c, kh] += P.T @ dO
            tol["dv"][c, kh] += (u + SLACK) * (P.T @ dO.abs()) + g * (seen.double().T @ dO.abs())
    if do is not None:
        for n in ("dk", "dv"):
            tol[n] += u * out[n].abs()
    # outputs below the type's normal range are rounded to its grid
    return {n: (out[n], tol[n] + (g if n != "lse" else 0.0)) for n in out}


def close(name, got, want):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    same = torch.isinf(value) & (got == value)
    off = torch.where(same, 0.0, (got - value).abs() - bound)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0.0 and not torch.isnan(off).any(), (name, "off its bound by", worst, "at", (off == off.max()).nonzero()[:3].tolist())


def starts(lengths, first=0):
    cu = [first]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def make(lengths_q, lengths_k, H, Hk, D, dtype, seed=0, first=0, behind=0, device="cuda"):
    """q, k, v, dout, cu_q, cu_k (lists): `first` tokens before the first sequence and `behind` behind the last."""
    g = torch.Generator().manual_seed(seed)
    cu_q, cu_k = starts(lengths_q, first), starts(lengths_k, first)
    mk = lambda n, h, s: (torch.randn(n, h, D, generator=g) * s).to(dtype).to(device)
    return (mk(cu_q[-1] + behind, H, 1.5), mk(cu_k[-1] + behind, Hk, 1.0), mk(cu_k[-1] + behind, Hk, 1.0), mk(cu_q[-1] + behind, H, 1.0), cu_q, cu_k)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")
