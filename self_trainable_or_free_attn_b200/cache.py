"""A paged cache of keys and values: pages and slots of new tokens, their keys and values written there, and the attention of a
batch's next tokens to a prefix that all its requests share and to what each has added.

  k_cache, v_cache  [pages, page_size, kv_heads, D], bf16 or fp16, any page, token and head strides; the caller's own
  table             int32 [batch, width]: the pages of each request's own tokens; entries behind the last are not read
  lengths           int32 [batch]: tokens of its own that each request holds

A step of a decoding loop, all of it on the GPU and nothing synchronising, so that it can be captured into a graph:

    plan = extend_tables(lengths, new, table, free_pages, page_size, total=batch)        # once per step
    store_kv(k, v, k_cache, v_cache, plan.slots)                                         # per layer
    out = prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, table, plan.lengths)

A prompt enters the same way; its own attention is `packed.packed_attention` with `plan.cu_new`, which reads no pages: behind a shared prefix each prompt
brings the prefix's keys and values in front of its own (`cu_k`, as the prompt's next chunk does).
"""
from dataclasses import dataclass

import torch

from . import _native as N
from ._native import check_status  # noqa: F401
from .packed import _DTYPES, _call, _workspace, check_heads, check_ints, check_tokens, empty, lay, softmax_scale, strides, usable

PAGE_SIZES = (16, 32, 64, 128, 256)


@dataclass
class CachePlan:
    """Where the new tokens of a batch of requests go. All int32, on the device."""
    slots: torch.Tensor        # [total] page * page_size + offset of each new token; -1: it has none
    positions: torch.Tensor    # [total] position in its request, from 0 (behind a shared prefix, add its length); -1 behind the last
    cu_new: torch.Tensor       # [batch + 1] the new tokens of request b are cu_new[b] .. cu_new[b + 1] - 1
    lengths: torch.Tensor      # [batch] tokens that each request holds now
    taken: torch.Tensor        # [2] pages taken from the free list; pages that were needed but not there


@N.device_guard
def extend_tables(lengths, new_tokens, table, free_pages, page_size, *, total):
    """Pages and slots of `new_tokens[b]` more tokens for each request, which holds `lengths[b]`: a CachePlan.

    The pages that are missing come from `free_pages` (int32, distinct) in order, request by request, and are written into `table`. `total` is
    the number of new tokens, or a bound on it that the host knows: slots and positions have that length. `lengths` and `free_pages` stay as
    they are; the caller drops the first `taken[0]` pages. Where the free list or a row of the table is too short, the tokens without a
    page have slot -1, the plan's `lengths` leave them out, and `taken[1]` says how many pages were missing."""
    if not table.is_cuda:
        raise RuntimeError("table must be a CUDA tensor: this operator has no CPU path")
    if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous():
        raise RuntimeError("table must be int32 [batch, width], contiguous: it is written in place")
    lengths, new_tokens, free_pages = check_ints(table, lengths=lengths, new_tokens=new_tokens, free_pages=free_pages)
    B, width = table.shape
    if lengths.shape != (B,) or new_tokens.shape != (B,) or free_pages.dim() != 1:
        raise RuntimeError("lengths and new_tokens must be [batch] like the rows of table, free_pages [pages]")
    page_size, total = int(page_size), int(total)
    if not 1 <= page_size < 2 ** 31:
        raise ValueError(f"page_size must be at least 1 and below 2**31, got {page_size}")
    if not 0 <= total < 2 ** 31:
        raise ValueError(f"total must be 0 or more, got {total}")
    plan = CachePlan(*torch.empty(2 * total + 2 * B + 3, device=table.device, dtype=torch.int32).split_with_sizes((total, total, B + 1, B, 2)))
    _call("es_extend_tables", N.ptr(lengths), N.ptr(new_tokens), N.ptr(table), N.ptr(free_pages), free_pages.numel(), B, width, page_size,
          total, N.ptr(plan.slots), N.ptr(plan.positions), N.ptr(plan.cu_new), N.ptr(plan.lengths), N.ptr(plan.taken), N.stream_ptr())
    return plan


def _check_cache(k_cache, v_cache):
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise RuntimeError(f"k_cache and v_cache must be [pages, page_size, kv_heads, D], got {tuple(shape)}, {tuple(v_cache.shape)}")
    if not (usable(k_cache) and usable(v_cache)):
        raise RuntimeError("the rows of a cache must be contiguous and start on 16 bytes")
    if shape[0] * shape[1] >= 2 ** 31:
        raise RuntimeError("a cache holds fewer than 2**31 tokens")
    return shape


@N.device_guard
def store_kv(k, v, k_cache, v_cache, slots):
    """Writes k, v [tokens, kv_heads, D] into the cache: token t at slots[t] (page * page_size + offset). Tokens whose slot is
    -1, or lies outside the cache, are skipped. The slots of a call are distinct: of two tokens with one slot either may be stored. No
    gradients; autograd knows that the cache has changed, and a graph that had saved it says so in its backward."""
    check_tokens(k, k=k, v=v, k_cache=k_cache, v_cache=v_cache)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError("store_kv has no backward: call it under torch.no_grad()")
    P, S, Hk, D = _check_cache(k_cache, v_cache)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (Hk, D):
        raise RuntimeError("k and v must be [tokens, kv_heads, D] with the heads of the cache")
    check_heads(Hk, Hk, D)
    slots, = check_ints(k, slots=slots)
    if slots.shape != (k.shape[0],):
        raise RuntimeError("slots must be [tokens]")
    k, rk = lay(k, (Hk * D, D))
    v, rv = lay(v, (Hk * D, D))
    _call("es_store_kv", k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), k.shape[0], Hk, D, P, S, *rk, *rv,
          *strides(k_cache), *strides(v_cache), N.stream_ptr())
    torch.autograd.graph.increment_version([t for t in (k_cache, v_cache) if not t.is_inference()])


@N.device_guard
def prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, table, lengths, *, scale=None, return_lse=False):
    """Attention of the newest tokens of a batch of requests, q [batch, tokens, heads, D], to a prefix that all of them share and to
    their own tokens: [batch, tokens, heads, D], and with return_lse the natural-log LSE [batch, heads, tokens] in fp32. At most 2**23 requests. Softmax
    statistics and sums are fp32, the weights are rounded to the inputs' type before they are multiplied with the values.

    The prefix is the first `prefix_len` tokens (an int; 0 for none) of the pages `prefix_pages` (int32); its keys and values are read once for
    the whole batch. The queries' own keys are the last of a request's `lengths[b]` tokens (what `extend_tables` returns), and query i
    sees the own tokens up to its own, 0 .. lengths[b] - tokens + i. A request of length 0 sees the prefix alone, a row without any key is 0
    with LSE -inf. Keys in a page that is not of the cache (-1, say) are not attended to. What lies behind a request's last token in its last page
    is not read into the result. No gradients."""
    check_tokens(q, q=q, k_cache=k_cache, v_cache=v_cache)
    if q.requires_grad or k_cache.requires_grad or v_cache.requires_grad:
        if torch.is_grad_enabled():
            raise RuntimeError("prefix_attention has no backward: call it under torch.no_grad()")
    P, S, Hk, D = _check_cache(k_cache, v_cache)
    if q.dim() != 4 or q.shape[3] != D:
        raise RuntimeError("q must be [batch, tokens, heads, D] with the head dim of the cache")
    if S not in PAGE_SIZES:
        raise RuntimeError(f"the page size must be one of {PAGE_SIZES}, got {S}")
    B, T, H, _ = q.shape
    check_heads(H, Hk, D)
    prefix_pages, table, lengths = check_ints(q, prefix_pages=prefix_pages, table=table, lengths=lengths)
    if prefix_pages.dim() != 1 or table.dim() != 2 or table.shape[0] != B or lengths.shape != (B,):
        raise RuntimeError("prefix_pages must be [pages], table [batch, width], lengths [batch]")
    prefix_len = int(prefix_len)
    if not 0 <= prefix_len <= prefix_pages.numel() * S:
        raise ValueError(f"prefix_len = {prefix_len}: the {prefix_pages.numel()} prefix pages hold 0 to {prefix_pages.numel() * S} tokens")
    if prefix_len >= 2 ** 31 - 256:
        raise ValueError(f"at most 2**31 - 257 prefix tokens, got {prefix_len}")
    if table.shape[1] * S > 2 ** 31 - 256 or B * T * H >= 2 ** 31 or B > 2 ** 23:
        raise RuntimeError("at most 2**31 - 256 tokens to a row of table, fewer than 2**31 query rows and at most 2**23 requests")
    q = q.contiguous() if q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format)
    o = empty(q)
    lse = torch.empty(B, H, T, device=q.device, dtype=torch.float32)
    ws = _workspace("es_prefix_workspace_bytes", q, (B, T, H, Hk, D, prefix_len, table.shape[1], S))
    _call("es_prefix_attn", N.ptr(q), N.ptr(k_cache), N.ptr(v_cache), N.ptr(o), N.ptr(lse), N.ptr(prefix_pages), prefix_pages.numel(), prefix_len,
          N.ptr(table), table.shape[1], N.ptr(lengths), B, T, H, Hk, D, P, S, *strides(k_cache), *strides(v_cache), softmax_scale(scale, D),
          _DTYPES[q.dtype], N.ptr(ws), N.stream_ptr())
    return (o, lse) if return_lse else o
