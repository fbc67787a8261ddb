"""Attention over packed sequences: the tokens of a batch lie behind one another, without padding between them.

`packed_attention` is exact softmax attention of every sequence to its own keys, with gradients: causal or full, with as many
query heads to a key head as the model has, from sequences of one token to long ones. It stands beside the block-sparse operators of
`vsa`, which take sequences of one length: the same kernels' conventions (bf16 or fp16, head dim 64 or 128, one owner per gradient row:
reproducible bit for bit). Scores, softmax statistics, LSE and sums are fp32; the weights P and, in the backward, dS are rounded to the inputs' type
before they are multiplied with V, dO, Q and K, which leaves an output off by 1.1 to 1.5 times its own rounding. Where rows see up to 32 keys the training
path multiplies what these roundings left as well, and the outputs are off by their own rounding alone.

Memory: a call that records a graph keeps, beside q, k, v, the output and its LSE, what rounding the output left, a second tensor of the output's size.

  q        [tokens, heads, D]; k, v [tokens, kv_heads, D], heads a multiple of kv_heads; any token and head strides (the thirds
           of a fused projection, say); what the kernels' loads cannot take (a last dimension with a stride, rows off 16 bytes) is copied
  cu_q     int32 [batch + 1] on the device, not decreasing: sequence b has the tokens cu_q[b] .. cu_q[b + 1] - 1
  cu_k     the same for the keys where they are more than the queries (a prompt's next chunk behind what is there)

Tokens of no sequence (behind the last, say) get output 0, LSE -inf and gradient 0, and what they hold reaches no other row; the same
is true of keys that the causal mask hides.

Forward and backward can be captured into a CUDA graph, by autograd's rule for captures: warm up on a side stream and drop every
graph that was recorded eagerly from the same leaves before the capture begins (an eager graph that lives on ties its leaves'
accumulation to another stream, and a capture that reaches into that stream ends with an error).
"""
import functools
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N
from ._native import check_status  # noqa: F401

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
DIMS = (64, 128)


def usable(t):
    """Whether the kernels' 16-byte loads can take t [..., D] as it lies: its rows in one piece, no two rows the same memory."""
    if t.data_ptr() % 16:
        return False
    if t.is_contiguous() and t.shape[-1] % 8 == 0:
        return True
    return t.stride(-1) == 1 and all(n == 1 or (s % 8 == 0 and t.shape[-1] <= s < 2 ** 39) for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def rows(t):
    """t itself where the kernels can read it, else a copy."""
    return t if usable(t) else t.clone(memory_format=torch.contiguous_format)


def strides(t):
    """Element strides of all but the last dimension; those of dimensions of one entry, which nothing uses, as if contiguous."""
    if t.is_contiguous():
        shape = t.shape
        if len(shape) == 3:
            return shape[1] * shape[2], shape[2]
        return shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3]
    whole, out = t.shape[-1], []
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        out.append(s if n > 1 else whole)
        whole = max(whole, out[-1] * n)
    return tuple(reversed(out))


def lay(t, whole):
    """t, or a copy where the kernels cannot read it as it lies, and its strides; `whole`: those of a contiguous one."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, whole
    if usable(t):
        return t, strides(t)
    return t.clone(memory_format=torch.contiguous_format), whole


def empty(t):
    """Memory for a contiguous tensor like t."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def softmax_scale(scale, D):
    if scale is None:
        return 1.0 / math.sqrt(D)
    scale = float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:               # a normal number of 32 bits, as is its product with log2(e)
        raise ValueError(f"scale must be above 0 and from 2**-126 to 2**126, got {scale}")
    return scale


def check_heads(q_heads, kv_heads, D):
    if D not in DIMS:
        raise RuntimeError(f"the head dim must be one of {DIMS}, got {D}")
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise RuntimeError(f"the query heads ({q_heads}) must be a multiple of the key heads ({kv_heads})")


def check_tokens(ref, **tensors):
    """Every tensor on the CUDA device of `ref` and in its dtype, bf16 or fp16, and none with a tangent: the kernels compute no forward-mode
    derivatives, and would take a dual tensor for its value."""
    if forward_ad._current_level >= 0:                       # (inside torch.autograd.forward_ad.dual_level)
        for name, t in tensors.items():
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} carries a tangent: this operator has no forward-mode derivative")
    dev, dtype = ref.get_device(), ref.dtype
    for name, t in tensors.items():
        if t.is_cuda and t.dtype is dtype and dtype in _DTYPES and t.get_device() == dev:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor: this operator has no CPU path")
        if t.get_device() != dev:
            raise RuntimeError(f"{name} must be on {ref.device}, got {t.device}")
        raise RuntimeError("all of them must share the dtype bfloat16 or float16: " + ", ".join(tensors))


def check_ints(ref, **tensors):
    """Device tensors of whole numbers as int32, contiguous. int64 is narrowed to the nearest 32 bits hold: outside a bound stays outside."""
    out, dev = [], ref.get_device()
    for name, t in tensors.items():
        if t.get_device() != dev:
            raise RuntimeError(f"{name} must be on {ref.device}, got {t.device}")
        if t.dtype is not torch.int32 or not t.is_contiguous():
            if t.dtype not in (torch.int32, torch.int64):
                raise RuntimeError(f"{name} must be int32, got {t.dtype}")
            if t.dtype is torch.int64:
                t = t.clamp(-2 ** 31, 2 ** 31 - 1)
            t = t.to(torch.int32).contiguous()
        out.append(t)
    return out


def _call(name, *args):
    rc = getattr(N._lib or N.load(), name)(*args)
    if rc:
        N.check(rc, name)


@functools.lru_cache(maxsize=4096)
def _bytes(name, device, sizes):
    """Bytes of scratch, which follow from the sizes (and from the device's number of SMs)."""
    return int(getattr(N.load(), name)(*sizes))


def _workspace(name, q, sizes):
    n = _bytes(name, q.get_device(), sizes)
    return torch.empty(n, device=q.device, dtype=torch.uint8) if n else None


def _fwd(q, k, v, cu_q, cu_k, scale, causal, with_rest):
    T, H, D = q.shape
    Tk, Hk, _ = k.shape
    q, rq = lay(q, (H * D, D))
    k, rk = lay(k, (Hk * D, D))
    v, rv = lay(v, (Hk * D, D))
    o = empty(q)
    rest = empty(q) if with_rest else None
    lse = torch.empty(H, T, device=q.device, dtype=torch.float32)
    sizes = (cu_q.shape[0] - 1, T, Tk, H, Hk, D)
    ws = _workspace("es_packed_fwd_workspace_bytes", q, sizes)
    _call("es_packed_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), N.ptr(rest), lse.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), *sizes,
          *rq, *rk, *rv, scale, causal, _DTYPES[q.dtype], N.ptr(ws), N.stream_ptr())
    return o, rest, lse


class _Function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, causal):
        o, rest, lse = _fwd(q, k, v, cu_q, cu_k, scale, causal, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, cu_q, cu_k)
        ctx.scale, ctx.causal = scale, causal
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    @N.device_guard
    def backward(ctx, dout, dlse):
        if dout is None:
            return (None,) * 7
        q, k, v, o, rest, lse, cu_q, cu_k = ctx.saved_tensors
        (T, H, D), (Tk, Hk, _) = q.shape, k.shape
        dout, rdo = lay(dout, (H * D, D))
        sizes = (cu_q.shape[0] - 1, T, Tk, H, Hk, D)
        need = ctx.needs_input_grad
        dq = empty(q) if need[0] else None
        dk, dv = (empty(k), empty(v)) if need[1] or need[2] else (None, None)
        ws = _workspace("es_packed_bwd_workspace_bytes", q, sizes)
        _call("es_packed_attn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), rest.data_ptr(), dout.data_ptr(), lse.data_ptr(), N.ptr(dq), N.ptr(dk),
              N.ptr(dv), cu_q.data_ptr(), cu_k.data_ptr(), *sizes, *strides(q), *strides(k), *strides(v), *rdo, ctx.scale, ctx.causal, _DTYPES[q.dtype],
              N.ptr(ws), N.stream_ptr())
        return dq, dk, dv, None, None, None, None


@N.device_guard
def packed_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, return_lse=False):
    """Softmax attention of every sequence of a packed batch to its own keys: [tokens, heads, D], and with return_lse also the
    natural-log LSE [heads, tokens] in fp32 (no gradient flows through it).

    `causal`: query i of nq sees the keys j <= i + nk - nq of its sequence's nk (the last query sees all); a row that sees none is 0 with
    LSE -inf. `scale`: factor of q k^T, 1 / sqrt(D) by default. cu_q, cu_k are read on the GPU only: nothing synchronises, and a
    captured call follows them when they change."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise RuntimeError(f"q, k, v must be [tokens, heads, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    check_tokens(q, q=q, k=k, v=v)
    T, H, D = q.shape
    Tk, Hk, Dk = k.shape
    if k.shape != v.shape or Dk != D:
        raise RuntimeError("k and v must have one shape, and the head dim of q")
    check_heads(H, Hk, D)
    if cu_k is None:
        if Tk != T:
            raise RuntimeError(f"without cu_k there are as many keys as queries, got {Tk} and {T}")
        cu_q, = check_ints(q, cu_q=cu_q)
        cu_k = cu_q
    else:
        cu_q, cu_k = check_ints(q, cu_q=cu_q, cu_k=cu_k)
    if cu_q.dim() != 1 or cu_q.shape[0] < 1 or cu_k.shape != cu_q.shape:
        raise RuntimeError("cu_q and cu_k must be [batch + 1]")
    if max(T, Tk) >= 2 ** 31 - 256:
        raise RuntimeError("at most 2**31 - 257 tokens")
    scale, causal = softmax_scale(scale, D), 1 if causal else 0
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, lse = _Function.apply(rows(q), rows(k), rows(v), cu_q, cu_k, scale, causal)
    else:
        o, _, lse = _fwd(q, k, v, cu_q, cu_k, scale, causal, False)
    return (o, lse) if return_lse else o
