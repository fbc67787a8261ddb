"""The work of the operators for packed sequences and for a paged cache of keys and values, as cases that can be timed and compared.

  prompt   `packed.packed_attention` without gradients: prompts of different lengths behind one another, grouped heads
  train    the same operator forward and backward
  prefix   `cache.prefix_attention`: the next tokens of a batch of requests that share a long prefix
  append   `cache.extend_tables` and `cache.store_kv`: pages and slots of the new tokens, and their keys and values written there

`run` computes them in their plain form, in float32 from elementary operations, or through the entry points where `own` is true.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_FLOPS = 3.2e12            # no drawn case computes more than the largest listed one
MOST_BYTES = 0.8e9             # nor moves more
ROWS = 2048                    # query rows of a chunk of the plain forms: bounds the memory of their score matrices


# ------------------------------------------------------------------------------------------------------------ the cases
def _packed(name, kind, batch, total, heads, kv_heads, dim=128, dtype="bf16", causal=True, past=0, mix=1):
    """`batch` sequences of `total` query tokens in all; `past`: keys in front of each sequence's own (a prompt's next chunk)."""
    return dict(name=name, kind=kind, batch=batch, total=total, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal,
                past=past, mix=mix)


def _prefix(name, batch, new, heads, kv_heads, prefix, most, page, dim=128, dtype="bf16", mix=1):
    """`batch` requests with `new` tokens each, a shared prefix, and 1 to `most` further tokens of their own in pages of `page`."""
    return dict(name=name, kind="prefix", batch=batch, new=new, heads=heads, kv_heads=kv_heads, prefix=prefix, most=most, page=page,
                dim=dim, dtype=dtype, mix=mix)


def _append(name, batch, total, kv_heads, most, page, dim=128, dtype="bf16", mix=1):
    """`total` new tokens for `batch` requests that hold 0 to `most` tokens."""
    return dict(name=name, kind="append", batch=batch, total=total, kv_heads=kv_heads, most=most, page=page, dim=dim, dtype=dtype, mix=mix)


def listed():
    return [
        # one short prompt (the conditioning text of one request): launches and latency
        _packed("prompt_77_tokens", "prompt", 1, 77, 12, 12),
        # a batch of ragged prompts of a 40-head model with grouped heads, five query heads to a key head
        _packed("prompt_packed_16k", "prompt", 24, 16383, 40, 8, mix=2),
        # one prompt of 32,760 tokens, fp16
        _packed("prompt_long_32k", "prompt", 1, 32760, 12, 2, dtype="fp16"),
        # the next 200 tokens of two prompts whose first 16,000 are there already: few rows against a long axis
        _packed("prompt_chunk_16k", "prompt", 2, 400, 28, 4, past=16000),
        # a packed training batch at the length and heads of the sparse training shape
        _packed("train_packed_32k", "train", 8, 32768, 12, 12, mix=3),
        # a small training step with grouped heads, ragged
        _packed("train_grouped_4k", "train", 5, 4157, 16, 4, mix=4),
        # several short videos packed into one batch, everything attends to everything, head dim 64, fp16
        _packed("train_full_fp16_d64", "train", 6, 9360, 4, 4, dim=64, dtype="fp16", causal=False, mix=5),
        # the smallest decoding step: one request, a short prefix
        _prefix("prefix_one_request", 1, 1, 12, 2, 513, 40, 16),
        # 64 samples of one prompt of 8,000 tokens, some hundred tokens into their answers
        _prefix("prefix_64_samples", 64, 1, 32, 4, 8000, 1024, 16, mix=2),
        # the largest: 256 requests with five query heads to a key head, long answers, two tokens at a time
        _prefix("prefix_256_requests", 256, 2, 40, 8, 32760, 4096, 64, mix=3),
        # a decoding step's bookkeeping: one token for each of 256 requests
        _append("append_256_tokens", 256, 256, 8, 4096, 16, mix=2),
        # a batch of prompts enters the cache
        _append("append_prompts_16k", 48, 16384, 8, 700, 64, mix=3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["prompt", "prompt", "train", "train", "prefix", "prefix", "append"])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 8])
        dim, dtype, mix = rng.choice([64, 128, 128]), rng.choice(["bf16", "bf16", "fp16"]), rng.randint(1, 10 ** 6)
        if kind in ("prompt", "train"):
            batch = _log_int(rng, 1, 64)
            total = max(batch, _log_int(rng, 16, 32768))
            past = _log_int(rng, 64, 16000) if kind == "prompt" and rng.random() < 0.3 else 0
            c = _packed("", kind, batch, total, heads, kv_heads, dim, dtype, rng.random() < 0.7, past, mix)
        elif kind == "prefix":
            c = _prefix("", _log_int(rng, 1, 256), rng.choice([1, 1, 1, 2, 4]), heads, kv_heads, _log_int(rng, 64, 32768),
                        _log_int(rng, 8, 4096), rng.choice([16, 32, 64, 128]), dim, dtype, mix)
        else:
            batch = _log_int(rng, 1, 256)
            total = batch if rng.random() < 0.4 else max(batch, _log_int(rng, 64, 16384))
            c = _append("", batch, total, kv_heads, _log_int(rng, 8, 4096), rng.choice([16, 32, 64, 128]), dim, dtype, mix)
        del c["name"]
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return c


# ------------------------------------------------------------------------------------------------------------ sizes
def _lengths(c):
    """Tokens of each sequence: uneven shares of the whole, one token at least."""
    rng = random.Random(c["mix"])
    share = [math.exp(rng.gauss(0.0, 0.8)) for _ in range(c["batch"])]
    free, whole = c["total"] - c["batch"], sum(share)
    got = [1 + int(free * s / whole) for s in share]
    got[0] += c["total"] - sum(got)
    return got


def _held(c):
    """Tokens that each request holds of its own; a decoding step's new ones are the last of them."""
    rng = random.Random(c["mix"])
    low = c["new"] if c["kind"] == "prefix" else 0
    return [max(low, _log_int(rng, 1, max(2, c["most"])) - (0 if low else 1)) for _ in range(c["batch"])]


def work(case):
    c = case
    D = c["dim"]
    if c["kind"] in ("prompt", "train"):
        n = _lengths(c)
        pairs = sum(x * c["past"] + (x * (x + 1) // 2 if c["causal"] else x * x) for x in n)
        q = c["total"] * c["heads"] * D * 2.0
        kv = 2.0 * (c["total"] + c["past"] * c["batch"]) * c["kv_heads"] * D * 2.0
        lse = c["total"] * c["heads"] * 4.0
        flops = 4.0 * D * c["heads"] * pairs
        if c["kind"] == "train":                       # q, k, v, do in; o, lse, dq, dk, dv out; 2 products forward, 5 backward
            return dict(bytes=4 * q + 2 * kv + lse, flops=3.5 * flops)
        return dict(bytes=2 * q + kv + lse, flops=flops)
    if c["kind"] == "prefix":
        held, N = _held(c), c["new"]
        pairs = sum(N * (c["prefix"] + h) - N * (N - 1) // 2 for h in held)
        io = 2.0 * c["batch"] * N * c["heads"] * D * 2
        kv = 2.0 * (c["prefix"] + sum(held)) * c["kv_heads"] * D * 2
        return dict(bytes=io + kv + c["batch"] * N * c["heads"] * 4.0, flops=4.0 * D * c["heads"] * pairs)
    pages = sum(-(-h // c["page"]) for h in _held(c))
    return dict(bytes=4.0 * c["total"] * c["kv_heads"] * D * 2 + 4.0 * (2 * c["total"] + 4 * c["batch"] + pages), flops=0.0)


# ------------------------------------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, D = DTYPES[c["dtype"]], c["dim"]

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dt)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def starts(n):
        return [sum(n[:i]) for i in range(len(n) + 1)]

    s = dict(c=c)
    if c["kind"] in ("prompt", "train"):
        n = _lengths(c)
        s["n_q"], s["n_k"] = n, [x + c["past"] for x in n]
        s["cu_q"], s["cu_k"] = ints(starts(s["n_q"])), ints(starts(s["n_k"]))
        s["q"] = rnd(sum(s["n_q"]), c["heads"], D, scale=1.5)
        s["k"], s["v"] = rnd(sum(s["n_k"]), c["kv_heads"], D), rnd(sum(s["n_k"]), c["kv_heads"], D)
        if c["kind"] == "train":
            s["do"] = rnd(sum(s["n_q"]), c["heads"], D)
            for x in ("q", "k", "v"):
                s[x].requires_grad_(True)
        return s
    held, page = _held(c), c["page"]
    new = [c["new"]] * c["batch"] if c["kind"] == "prefix" else _lengths(c)
    after = [h + (0 if c["kind"] == "prefix" else n) for h, n in zip(held, new)]
    width = max(-(-a // page) for a in after) + 1
    n_prefix = -(-c["prefix"] // page) if c["kind"] == "prefix" else 0
    n_pages = n_prefix + sum(-(-a // page) for a in after) + 5
    ids = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)      # requests come and go: pages lie in no order
    table = torch.full((c["batch"], width), -1, dtype=torch.int32)
    used, host = n_prefix, ids.cpu()
    for b, h in enumerate(held):                                                # pages that the request holds already
        have = -(-h // page)
        table[b, :have] = host[used:used + have]
        used += have
    s.update(new=ints(new), lengths=ints(held), table=table.to(DEV), held=held, n_new=new)
    if c["kind"] == "prefix":
        s["k_cache"], s["v_cache"] = rnd(n_pages, page, c["kv_heads"], D), rnd(n_pages, page, c["kv_heads"], D)
        s["q"] = rnd(c["batch"], c["new"], c["heads"], D, scale=1.5)
        s["prefix_pages"] = ids[:n_prefix].contiguous()
    else:
        s["k_cache"], s["v_cache"] = (torch.zeros(n_pages, page, c["kv_heads"], D, device=DEV, dtype=dt) for _ in range(2))
        s["k"], s["v"] = rnd(c["total"], c["kv_heads"], D), rnd(c["total"], c["kv_heads"], D)
        s["free"] = ids[used:].contiguous()
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"prompt": _run_packed, "train": _run_packed, "prefix": _run_prefix, "append": _run_append}[state["c"]["kind"]](state)


def _run_packed(s):
    c = s["c"]
    train = c["kind"] == "train"
    if own:
        from self_trainable_or_free_attn_b200 import packed
        o, lse = packed.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"] if c["past"] else None, causal=c["causal"],
                                         return_lse=True)
        if train:
            return (o.detach(), lse, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))
        return o, lse
    H, D = c["heads"], c["dim"]
    with torch.no_grad():
        o = torch.empty_like(s["q"])
        lse = torch.empty(H, o.shape[0], device=DEV)
        grads = [torch.empty_like(s[x]) for x in ("q", "k", "v")] if train else []
        q0 = k0 = 0
        for nq, nk in zip(s["n_q"], s["n_k"]):
            for h in range(c["kv_heads"]):
                heads = slice(h * (H // c["kv_heads"]), (h + 1) * (H // c["kv_heads"]))
                k, v = s["k"][k0:k0 + nk, h].float(), s["v"][k0:k0 + nk, h].float()
                dk, dv = torch.zeros_like(k), torch.zeros_like(v)
                step = max(1, ROWS // (H // c["kv_heads"]))
                for r in range(0, nq, step):
                    rows, seen = slice(q0 + r, q0 + min(r + step, nq)), nk - nq + min(r + step, nq) if c["causal"] else nk
                    q = s["q"][rows, heads].float().transpose(0, 1)
                    x = q @ k[:seen].T / math.sqrt(D)
                    if c["causal"]:
                        at = torch.arange(r, min(r + step, nq), device=DEV) + (nk - nq)
                        x.masked_fill_(torch.arange(seen, device=DEV)[None] > at[:, None], -math.inf)
                    top = x.amax(-1, keepdim=True)
                    x.sub_(top).exp_()
                    whole = x.sum(-1, keepdim=True)
                    p = x.div_(whole)
                    out = p @ v[:seen]
                    o[rows, heads] = out.transpose(0, 1).to(o.dtype)
                    lse[heads, rows] = (top + whole.log())[..., 0]
                    if train:
                        do = s["do"][rows, heads].float().transpose(0, 1)
                        dv[:seen] += torch.einsum("hij,hid->jd", p, do)
                        ds = (do @ v[:seen].T).sub_((do * out).sum(-1, keepdim=True)).mul_(p).div_(math.sqrt(D))
                        grads[0][rows, heads] = (ds @ k[:seen]).transpose(0, 1).to(o.dtype)
                        dk[:seen] += torch.einsum("hij,hid->jd", ds, q)
                if train:
                    grads[1][k0:k0 + nk, h], grads[2][k0:k0 + nk, h] = dk.to(o.dtype), dv.to(o.dtype)
            q0, k0 = q0 + nq, k0 + nk
    return (o, lse, *grads)


def _run_prefix(s):
    c = s["c"]
    if own:
        from self_trainable_or_free_attn_b200 import cache
        return cache.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"], c["prefix"], s["table"], s["lengths"],
                                      return_lse=True)
    B, N, H, D = s["q"].shape
    Hk, G, P = c["kv_heads"], c["heads"] // c["kv_heads"], c["prefix"]
    q = s["q"].float().reshape(B, N, Hk, G, D)

    def keys(x, pages, rows):                            # [..., rows, Hk, D] of the pages in this order
        return x[pages.clamp(min=0).long()].flatten(-4, -3)[..., :rows, :, :]

    # the requests' own tokens, padded to the longest, a few requests at a time
    most, o, lse = max(s["held"]), [], []
    k, v = (keys(s[x], s["prefix_pages"], P).float() for x in ("k_cache", "v_cache"))
    step = max(1, min(B, int(2e9 / (max(P, most) * H * max(N * 4, 2 * D // G)))))
    for b in range(0, B, step):
        rows = slice(b, min(b + step, B))
        shared = torch.einsum("bnhgd,phd->bhgnp", q[rows], k) / math.sqrt(D)
        mine_k, mine_v = (keys(s[x], s["table"][rows], most).float() for x in ("k_cache", "v_cache"))
        mine = torch.einsum("bnhgd,bphd->bhgnp", q[rows], mine_k) / math.sqrt(D)
        last = s["lengths"][rows, None] - N + torch.arange(N, device=DEV)
        hide = torch.arange(most, device=DEV) > last[..., None]
        mine.masked_fill_(hide[:, None, None], -math.inf)
        mine_v.masked_fill_(hide[:, -1, :, None, None], 0.0)         # what lies behind a request's last token is not its own
        top = torch.maximum(shared.amax(-1), mine.amax(-1))[..., None]
        shared.sub_(top).exp_()
        mine.sub_(top).exp_()
        whole = (shared.sum(-1) + mine.sum(-1))[..., None]
        out = (torch.einsum("bhgnp,phd->bhgnd", shared, v) + torch.einsum("bhgnp,bphd->bhgnd", mine, mine_v)) / whole
        o.append(out.permute(0, 3, 1, 2, 4).reshape(-1, N, H, D).to(s["q"].dtype))
        lse.append((top + whole.log())[..., 0].reshape(-1, H, N))
    return torch.cat(o), torch.cat(lse)


def _run_append(s):
    c = s["c"]
    if own:
        from self_trainable_or_free_attn_b200 import cache
        plan = cache.extend_tables(s["lengths"], s["new"], s["table"], s["free"], c["page"], total=c["total"])
        cache.store_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], plan.slots)
        return plan.slots, plan.positions, plan.cu_new, plan.lengths, plan.taken, s["table"], s["k_cache"], s["v_cache"]
    page, B = c["page"], c["batch"]
    held, new = s["lengths"].long(), s["new"].long()
    have, want = (held + page - 1) // page, (held + new + page - 1) // page
    need = want - have
    first = need.cumsum(0) - need
    # pages: column j of request b is new where have <= j < want, and takes the next of the free ones
    col = torch.arange(s["table"].shape[1], device=DEV)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    pick = (first[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    s["table"].copy_(torch.where(fresh, s["free"][pick], s["table"]))
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    cu[1:] = new.cumsum(0)
    tok = torch.arange(c["total"], device=DEV)
    req = (tok[:, None] >= cu[None, 1:]).sum(1)
    pos = held[req] + tok - cu[req]
    slots = s["table"][req, pos // page].long() * page + pos % page
    for x, y in (("k", "k_cache"), ("v", "v_cache")):
        s[y].view(-1, c["kv_heads"], c["dim"])[slots] = s[x]
    return (slots.int(), pos.int(), cu, (held + new).int(), torch.stack((need.sum(), need.sum() * 0)).int(), s["table"], s["k_cache"],
            s["v_cache"])


# ------------------------------------------------------------------------------------------------------------ the definition
def exact(case, seed):
    c = case
    if c["kind"] == "append":
        return None                                      # whole numbers and copies
    s = prepare(case, seed)
    return _exact_prefix(s) if c["kind"] == "prefix" else _exact_packed(s)


def _softmax_attention(q, k, v, scale, offset):
    """One head in 64 bits: row i sees the keys up to i + offset (every key where offset is None). (O, LSE)."""
    x = scale * torch.matmul(q, k.transpose(-1, -2))
    if offset is not None:
        x = x + torch.full_like(x, -math.inf).triu(offset + 1)
    lse = torch.logsumexp(x, -1)
    return torch.matmul(torch.exp(x - lse[..., None]), v), lse


def _exact_packed(s):
    c = s["c"]
    H, Hk, scale = c["heads"], c["kv_heads"], c["dim"] ** -0.5
    train = c["kind"] == "train"
    x = {n: s[n].detach().double() for n in ("q", "k", "v", "do") if n in s}
    outs = [torch.zeros_like(x["q"]), torch.zeros(H, x["q"].shape[0], device=DEV, dtype=torch.float64)]
    grads = [torch.zeros_like(x[n]) for n in "qkv"] if train else []
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(c["batch"]):
        for h in range(H):
            rows, cols, kh = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1]), h * Hk // H
            n, m = rows.stop - rows.start, cols.stop - cols.start
            k, v = x["k"][cols, kh].requires_grad_(train), x["v"][cols, kh].requires_grad_(train)
            for r in range(0, n, 4096):                  # in chunks of rows, for their memory
                part = slice(rows.start + r, min(rows.start + r + 4096, rows.stop))
                q = x["q"][part, h].requires_grad_(train)
                with torch.set_grad_enabled(train):
                    o, lse = _softmax_attention(q, k, v, scale, m - n + r if c["causal"] else None)
                outs[0][part, h], outs[1][h, part] = o.detach(), lse.detach()
                if train:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), x["do"][part, h])
                    grads[0][part, h] = dq
                    grads[1][cols, kh] += dk
                    grads[2][cols, kh] += dv
    return (*outs, *grads)


def _exact_prefix(s):
    c = s["c"]
    page, scale = c["page"], c["dim"] ** -0.5
    B, N, H, D = s["q"].shape
    G = H // c["kv_heads"]
    flat = {n: s[n].reshape(-1, c["kv_heads"], D) for n in ("k_cache", "v_cache")}

    def rows(pages, n):
        i = torch.arange(n, device=DEV)
        at = pages[i // page].long() * page + i % page
        return [flat[n_][at].double().transpose(0, 1).repeat_interleave(G, 0) for n_ in ("k_cache", "v_cache")]

    shared = rows(s["prefix_pages"], c["prefix"])
    out, lse = torch.empty(B, N, H, D, device=DEV, dtype=torch.float64), torch.empty(B, H, N, device=DEV, dtype=torch.float64)
    for b, held in enumerate(s["held"]):
        k, v = (torch.cat(p, 1) for p in zip(shared, rows(s["table"][b], held)))
        o, z = _softmax_attention(s["q"][b].double().transpose(0, 1), k, v, scale, c["prefix"] + held - N)
        out[b], lse[b] = o.transpose(0, 1), z
    return out, lse
