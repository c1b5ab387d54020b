"""Workloads of four operators that answering over a paged cache needs, and their plain forms.

  write4     rotary positions on the new queries and keys of a step; keys and values into a cache that
             holds them in 4 bits (llama.paged.rope_paged_write_int4)
  attn4      causal grouped-query attention of each request's new tokens (one token, a few, a chunk of a
             prompt) over that cache (llama.paged.paged_attention_int4)
  fork       requests that go on from other requests' tokens, or end: shared pages, block tables, free
             pages, and copies of the pages that are not full (llama.paged.paged_fork)
  logprobs   log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits
             (llama.logprobs.token_logprobs)

A 4-bit row is cut into groups of 32 dims.  A group has a scale s and an offset m of the row's 16-bit type
and codes c in 0 .. 15; it stands for the values c s + m, rounded to that type.  m is the group's smallest
value, s the difference to its largest over 15, rounded towards zero, and c the nearest code (ties to even,
15 at most).  Eight codes make a 32-bit word: those of even dims in its low half, of odd dims in its high one.

Every case is a dict of plain values.  Lengths follow from the case alone (`lens_seed`), values and
page orders from the seed given to prepare().  With own = False run() computes in elementary torch
operations; with own = True it makes the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-efficient-inference_b200")
GROUP = 32


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from llama import logprobs, paged

    return paged, logprobs


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step at batch 16 (Llama-3.2-1B heads): one new token each
        dict(name="write4_decode", op="write4", type="float16", heads=32, kv_heads=8, head_dim=64, tokens=16,
             page_size=16, max_pos=8192, lens_seed=1),
        # the same for a packed prompt step, an odd number of tokens, 128-wide heads
        dict(name="write4_prompt", op="write4", type="bfloat16", heads=32, kv_heads=8, head_dim=128, tokens=16381,
             page_size=64, max_pos=32768, lens_seed=2),
        # a decode step at batch 1 over the benchmark's context (512 prompt tokens and a few more)
        dict(name="attn4_single", op="attn4", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=1,
             new=1, chunks=0, chunk=0, ctx_lo=575, ctx_hi=575, page_size=16, lens_seed=3),
        # a decode step at batch 64, contexts from a few hundred tokens to 16 thousand
        dict(name="attn4_batch", op="attn4", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=64,
             new=1, chunks=0, chunk=0, ctx_lo=300, ctx_hi=16000, page_size=16, lens_seed=4),
        # few requests with long contexts, two tokens each (one drafted), 128-wide heads, a group of seven
        dict(name="attn4_long", op="attn4", type="bfloat16", heads=28, kv_heads=4, head_dim=128, seqs=4,
             new=2, chunks=0, chunk=0, ctx_lo=30001, ctx_hi=120000, page_size=64, lens_seed=5),
        # chunks of four prompts over what the cache holds already
        dict(name="attn4_chunk", op="attn4", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=4,
             new=1, chunks=4, chunk=1021, ctx_lo=500, ctx_hi=8000, page_size=16, lens_seed=6),
        # a mixed step: one chunk of a prompt among decoding requests, 128-wide heads
        dict(name="attn4_mixed", op="attn4", type="bfloat16", heads=32, kv_heads=8, head_dim=128, seqs=32,
             new=1, chunks=1, chunk=512, ctx_lo=200, ctx_hi=6000, page_size=32, lens_seed=7),
        # eight prompts, each answered eight times: the copies share the prompts' full pages (16 layers)
        dict(name="fork_samples", op="fork", kind="samples", groups=8, copies=8, ctx_lo=300, ctx_hi=3000, layers=16,
             kv_heads=8, head_dim=64, page_size=16, lens_seed=8),
        # one step of a search over four continuations of 64 prompts: each goes on from one of the four, some end
        dict(name="fork_search", op="fork", kind="search", groups=64, copies=4, ctx_lo=200, ctx_hi=2000, layers=8,
             kv_heads=8, head_dim=64, page_size=32, lens_seed=9),
        # one answer's token at a time, twenty alternatives (Llama-3.2-1B vocabulary, the model's fp32 logits)
        dict(name="logprobs_single", op="logprobs", type="float32", rows=1, vocab=128256, top=20, lens_seed=10),
        # a decode step of 64 answers
        dict(name="logprobs_batch", op="logprobs", type="float32", rows=64, vocab=128256, top=5, lens_seed=11),
        # the tokens of a prompt scored, the projection's own 16-bit logits
        dict(name="logprobs_prompt", op="logprobs", type="float16", rows=2047, vocab=128256, top=8, lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["write4", "attn4", "attn4", "attn4", "fork", "logprobs", "logprobs"])
    heads = dict(type=rng.choice(["float16", "bfloat16"]), head_dim=rng.choice([32, 64, 64, 96, 128, 128]))
    heads["kv_heads"] = rng.choice([1, 2, 4, 8])
    heads["heads"] = heads["kv_heads"] * rng.choice([1, 2, 3, 4, 6, 7, 8])
    if heads["heads"] > 32:
        heads["heads"] = heads["kv_heads"] * 4
    page_size = rng.choice([8, 16, 32, 64, 128])
    lens_seed = rng.randrange(1 << 30)
    if op == "write4":
        return dict(op=op, **heads, tokens=_log_int(rng, 1, 16000), page_size=page_size,
                    max_pos=_log_int(rng, 512, 32768), lens_seed=lens_seed)
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 150000)
        return dict(op=op, type=rng.choice(["float32", "float16", "bfloat16"]),
                    rows=_log_int(rng, 1, min(4000, 200000000 // vocab)), vocab=vocab,
                    top=rng.choice([0, 1, 2, 5, 10, 20, 32]), lens_seed=lens_seed)
    if op == "fork":
        copies = rng.choice([2, 3, 4, 8])
        case = dict(op=op, kind=rng.choice(["samples", "search"]), groups=_log_int(rng, 1, 256 // copies), copies=copies,
                    ctx_lo=rng.choice([1, 100]), layers=rng.choice([1, 2, 4, 8]), kv_heads=heads["kv_heads"],
                    head_dim=rng.choice([64, 128]), page_size=rng.choice([8, 16, 32]), lens_seed=lens_seed)
        most = 250000000 // (case["groups"] * case["layers"] * case["kv_heads"] * case["head_dim"])  # of a gigabyte
        return dict(case, ctx_hi=_log_int(rng, 101, max(120, min(2000, most))))
    kind = rng.choice(["decode", "decode", "chunk", "mixed"])
    if kind == "decode":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, min(100000, 250000 // seqs))
        return dict(op="attn4", **heads, seqs=seqs, new=rng.choice([1, 1, 1, 2, 4]), chunks=0, chunk=0,
                    ctx_lo=max(1, hi // rng.choice([1, 4, 64])), ctx_hi=hi, page_size=page_size, lens_seed=lens_seed)
    seqs = _log_int(rng, 1, 8) if kind == "chunk" else _log_int(rng, 2, 32)
    chunks = seqs if kind == "chunk" else max(1, seqs // 8)
    return dict(op="attn4", **heads, seqs=seqs, new=1, chunks=chunks, chunk=_log_int(rng, 2, 4000 // chunks),
                ctx_lo=1, ctx_hi=_log_int(rng, 1, 8000), page_size=page_size, lens_seed=lens_seed)


# ---------------------------------------------------------------------------------------------
# lengths (from the case alone)
# ---------------------------------------------------------------------------------------------
def _pages(n, page_size):
    return -(-n // page_size)


def _attn_lens(case):
    """(tokens the cache holds before the step, new tokens) per request."""
    rng = random.Random(case["lens_seed"])
    ctx = [_log_int(rng, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    new = [case["new"]] * case["seqs"]
    for b in rng.sample(range(case["seqs"]), case["chunks"]):
        new[b] = case["chunk"]
    return ctx, new


def _fork_plan(case):
    """(tokens of a group's prompt, tokens that each request holds, whom each goes on from: -1 ends it)."""
    rng = random.Random(case["lens_seed"])
    n = case["copies"]
    prompt, lens, parents = [], [], []
    for g in range(case["groups"]):
        shared = _log_int(rng, case["ctx_lo"], case["ctx_hi"])
        prompt.append(shared)
        first = g * n
        if case["kind"] == "samples":  # the prompt is there once, the others come to it
            lens += [shared] + [0] * (n - 1)
            parents += [first] * n
        else:  # all have gone on from the prompt by the same number of tokens
            lens += [shared + 1 + rng.randrange(40)] * n
            ends = rng.random() < 0.2  # the group's last one
            parents += [first + rng.randrange(n - ends) for _ in range(n - ends)] + [-1] * ends
    return prompt, lens, parents


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _shifts(device):
    """Bit of the word where the code of dim 0 .. 7 begins."""
    return torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=device)


def _pack(codes):
    """int32 codes [..., d] as uint8 [..., d / 2]."""
    words = (codes.unflatten(-1, (-1, 8)) << _shifts(codes.device)).sum(-1, dtype=torch.int32)
    return words.view(torch.uint8)


def _unpack(packed):
    """uint8 [..., d / 2] as int32 codes [..., d]."""
    words = packed.contiguous().view(torch.int32)
    return ((words.unsqueeze(-1) >> _shifts(packed.device)) & 15).flatten(-2)


def _values(packed, params):
    """What codes and (scale, offset) pairs [..., d / 32, 2] stand for, in their 16-bit type."""
    c = _unpack(packed).unflatten(-1, (-1, GROUP)).float()
    p = params.float()
    return (c * p[..., 0:1] + p[..., 1:2]).flatten(-2).to(params.dtype)


def _quantize(x):
    """Rows [..., d] of 16-bit values as (packed codes, params): the definition, in 64 bits."""
    g = x.double().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = (high - low) / 15
    s = step.to(x.dtype)  # the nearest, then down where it lies above: towards zero
    over = s.double() > step
    s = torch.where(over, (s.view(torch.int16) - 1).view(x.dtype), s)
    sd = s.double()
    c = torch.where(sd > 0, ((g - low) / sd).round(), torch.zeros_like(g)).clamp(0, 15)
    params = torch.cat([s, low.to(x.dtype)], dim=-1)
    return _pack(c.to(torch.int32).flatten(-2)), params


def _cache4(num_pages, case, dtype, gen, keys=False):
    """A 4-bit cache filled with quantized normal values: (codes, params), pages and heads contiguous."""
    H, P, D = case["kv_heads"], case["page_size"], case["head_dim"]
    codes = torch.empty(num_pages, H, P, D // 2, dtype=torch.uint8, device="cuda")
    params = torch.empty(num_pages, H, P, D // GROUP, 2, dtype=dtype, device="cuda")
    offset = torch.randn(H, 1, D, generator=gen, device="cuda") * (0.5 if keys else 0.0)
    for at in range(0, num_pages, 512):  # in pieces: the wide values are never held whole
        x = torch.randn(codes[at:at + 512].shape[:3] + (D,), generator=gen, device="cuda") + offset
        c, p = _quantize(x.to(dtype))
        codes[at:at + 512].copy_(c)
        params[at:at + 512].copy_(p)
    return codes.transpose(1, 2), params.transpose(1, 2)


def _prepare_fork(case, gen):
    prompt, lens, parents = _fork_plan(case)
    n, ps, B = case["copies"], case["page_size"], len(lens)
    shared = [prompt[b // n] // ps for b in range(B)]  # full pages of the prompt, held by all of a group that hold any
    first = [0] * len(prompt)
    page, at = [], 0
    for b in range(B):
        g = b // n
        if b % n == 0:
            first[g], at = at, at + shared[b]
        page.append(at)
        at += max(0, _pages(lens[b], ps) - shared[b])
    pool, width = at + B + 29, max(_pages(c, ps) for c in lens) + 2
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    j = torch.arange(width, device="cuda")[None, :]
    as_column = lambda v: torch.tensor(v, device="cuda")[:, None]  # noqa: E731
    number = torch.where(j < as_column(shared), as_column([first[b // n] for b in range(B)]) + j,
                         as_column(page) + j - as_column(shared))
    held = j < as_column([_pages(c, ps) for c in lens])
    tables = torch.where(held, order[number.clamp(0, pool - 1)], 0).to(torch.int32)
    free = torch.zeros(pool, dtype=torch.int32, device="cuda")
    free[:pool - at] = order[at:]
    shape = (2, case["layers"], pool, case["kv_heads"], ps, case["head_dim"])
    bits = torch.empty(shape, dtype=torch.int16, device="cuda").random_(0, 15000, generator=gen)
    both = bits.view(torch.float16)  # values from 0 to 1
    pools = [t.transpose(1, 2) for half in both for t in half]
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(kv_lens=torch.tensor(lens, **i32), parents=torch.tensor(parents, **i32), block_tables=tables,
                free_pages=free, n_free=torch.tensor([pool - at], **i32), both=both, pools=pools)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"op": case["op"], "case": case, "page_size": case.get("page_size", 0)}
    if case["op"] == "fork":
        st.update(_prepare_fork(case, gen))
        return st
    dtype = getattr(torch, case["type"])
    if case["op"] == "logprobs":
        T, V = case["rows"], case["vocab"]
        logits = torch.empty(T, V, dtype=dtype, device="cuda")
        for at in range(0, T, 256):  # rows of their own sharpness
            part = logits[at:at + 256]
            width = 1.0 + 2.0 * torch.rand(part.shape[0], 1, generator=gen, device="cuda")
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * width)
        # a token among the likelier ones
        some = torch.randint(0, V, (T, 64), generator=gen, device="cuda")
        pick = logits.gather(1, some).float().argmax(1, keepdim=True)
        st.update(logits=logits, tokens=some.gather(1, pick).view(-1))
        return st
    H, Hkv, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    if case["op"] == "write4":
        T = case["tokens"]
        num_pages = _pages(T, ps) + 5
        # a fused projection's output: the rows of q, k and v are parts of one wide row
        qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=gen, device="cuda").to(dtype)
        inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        angles = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * inv
        st.update(q=qkv[:, :H * D].view(T, H, D), k=qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D),
                  v=qkv[:, (H + Hkv) * D:].view(T, Hkv, D), cos=angles.cos().float(), sin=angles.sin().float(),
                  positions=torch.randint(0, case["max_pos"], (T,), generator=gen, device="cuda", dtype=torch.int32),
                  slots=torch.randperm(num_pages * ps, generator=gen, device="cuda")[:T].contiguous(),
                  cache_k=_cache4(num_pages, case, dtype, gen, keys=True), cache_v=_cache4(num_pages, case, dtype, gen))
        return st
    ctx, new = _attn_lens(case)
    kv = [c + n for c, n in zip(ctx, new)]
    total = sum(_pages(n, ps) for n in kv)
    num_pages = total + 11
    order = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    tables = torch.zeros(len(kv), _pages(max(kv), ps) + 3, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(kv):
        blocks = _pages(n, ps)
        tables[b, :blocks] = order[at:at + blocks]
        at += blocks
    st.update(ctx=ctx, new=new, q=torch.randn(sum(new), H, D, generator=gen, device="cuda").to(dtype),
              cache_k=_cache4(num_pages, case, dtype, gen, keys=True), cache_v=_cache4(num_pages, case, dtype, gen),
              block_tables=tables, kv_lens=torch.tensor(kv, dtype=torch.int32, device="cuda"),
              cu_seqlens=torch.tensor(_cumulative(new), dtype=torch.int32, device="cuda"), max_new=max(new))
    return st


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _turn(x, cos, sin):
    even, odd = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.stack([even * c - odd * s, even * s + odd * c], dim=-1).flatten(-2)


def _plain_write4(st):
    q, k, v, ps = st["q"], st["k"], st["v"], st["page_size"]
    pos = st["positions"].long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    q_rot = _turn(q.float(), cos, sin).to(q.dtype)
    # in 64 bits: the codes must not depend on how a value beside a border was rounded on its way
    k_rot = _turn(k.double(), cos.double(), sin.double()).to(k.dtype)
    page, row = st["slots"] // ps, st["slots"] % ps
    held = []
    for x, (codes, params) in ((k_rot, st["cache_k"]), (v, st["cache_v"])):
        c, p = _quantize(x)
        codes[page, row] = c
        params[page, row] = p
        held.append(_values(c, p))
    return (q_rot, *held, *st["cache_k"], *st["cache_v"])


def _plain_attn4(st):
    q, ps = st["q"], st["page_size"]
    out = torch.empty_like(q)
    H, D = q.shape[1:]
    at = 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["new"])):
        L = c + n
        pages = st["block_tables"][b, :_pages(L, ps)].long()
        k, v = (_values(codes[pages].flatten(0, 1)[:L], params[pages].flatten(0, 1)[:L]).float().transpose(0, 1)
                for codes, params in (st["cache_k"], st["cache_v"]))  # [kv_heads, L, D]
        Hkv = k.shape[0]
        qs = q[at:at + n].float().view(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3)  # [kv_heads, rep, n, D]
        hidden = torch.arange(L, device=q.device)[None, :] > torch.arange(n, device=q.device)[:, None] + c
        s = torch.matmul(qs, k.transpose(1, 2)[:, None]) * (1.0 / math.sqrt(D))
        s = s.masked_fill(hidden, float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(e, v[:, None]) / e.sum(-1, keepdim=True)
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, H, D).to(out.dtype)
        at += n
    return out


def _plain_fork(st):
    lens, tables, free, ps = st["kv_lens"].long(), st["block_tables"], st["free_pages"], st["page_size"]
    n_free, parents = st["n_free"].long(), st["parents"].long()
    B, width = tables.shape
    mine, j = torch.arange(B, device=tables.device), torch.arange(width, device=tables.device)
    comes = (parents >= 0) & (parents != mine)
    need = (comes & (lens[parents.clamp(min=0)] % ps != 0)).long()  # a page of its own for the part of a page
    upto = need.cumsum(0)
    granted = (need == 0) | (upto <= n_free)
    source = torch.where(granted, parents, mine)
    new_lens = torch.where(source < 0, 0, lens[source.clamp(min=0)])
    held, want = (lens + ps - 1) // ps, (new_lens + ps - 1) // ps
    moved = (granted & comes)[:, None]
    old = tables.clone()
    last = j == want[:, None] - 1
    part = moved & (need > 0)[:, None] & last
    fresh = free[(n_free - upto).clamp(0, free.numel() - 1)]
    now = torch.where(moved & (j < want[:, None]), old[source.clamp(min=0)], old)
    from_page = torch.where(part, now, 0).sum(1)
    now = torch.where(part, fresh[:, None], now)
    # a page goes back where none holds it any more, at its first holder's place in the order of requests and blocks
    kept = torch.zeros(free.numel(), dtype=torch.bool, device=tables.device)
    kept[now[j < want[:, None]].long()] = True
    was = (j < held[:, None]).flatten().nonzero().view(-1)
    page = old.flatten()[was].long()
    owner = torch.full((free.numel(),), B * width, dtype=torch.long, device=tables.device)
    owner.scatter_reduce_(0, page, was, "amin")
    back = page[~kept[page] & (owner[page] == was)]
    height = n_free - torch.where(granted, need, 0).sum()
    free[height + torch.arange(back.numel(), device=tables.device)] = back.int()
    tables.copy_(now)
    some = part.any(1).nonzero().view(-1)
    for pool in st["pools"]:
        pool[fresh[some].long()] = pool[from_page[some].long()]
    st["kv_lens"].copy_(new_lens)
    st["n_free"].copy_(height + back.numel())
    return st["kv_lens"], st["n_free"], granted, tables, free, st["both"]


def _plain_logprobs(st):
    x, tokens, k = st["logits"].float(), st["tokens"], st["case"]["top"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, dtype=torch.float64)
    log_total = total.log()
    chosen = d.gather(1, tokens[:, None]).view(-1).double() - log_total
    entropy = log_total - e.mul_(d).sum(-1, dtype=torch.float64) / total
    if k == 0:
        return chosen.float(), entropy.float()
    # unique keys: the value's order in the high half, the lower index first in the low one
    bits = (st["logits"].float() + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    keys = (bits << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))
    top = torch.topk(keys, k, dim=-1).values
    ids = 0x7FFFFFFF - (top & 0xFFFFFFFF)
    best = d.gather(1, ids).double() - log_total[:, None]
    return chosen.float(), entropy.float(), ids, best.float()


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if not own:
        return {"write4": _plain_write4, "attn4": _plain_attn4, "fork": _plain_fork,
                "logprobs": _plain_logprobs}[op](st)
    paged, logprobs = _framework()
    if op == "write4":
        q, k, v = paged.rope_paged_write_int4(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"],
                                              st["slots"], st["cache_k"], st["cache_v"])
        return (q, k, v, *st["cache_k"], *st["cache_v"])
    if op == "attn4":
        return paged.paged_attention_int4(st["q"], st["cache_k"], st["cache_v"], st["block_tables"], st["kv_lens"],
                                          st["cu_seqlens"], st["max_new"])
    if op == "fork":
        fork = paged.paged_fork(st["kv_lens"], st["block_tables"], st["free_pages"], st["n_free"], st["parents"],
                                st["page_size"], st["pools"], kv_lens_out=st["kv_lens"], n_free_out=st["n_free"])
        return fork.kv_lens, fork.n_free, fork.granted, st["block_tables"], st["free_pages"], st["both"]
    r = logprobs.token_logprobs(st["logits"], st["tokens"], st["case"]["top"])
    return r if st["case"]["top"] else (r.logprobs, r.entropy)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "logprobs":
        T, V = case["rows"], case["vocab"]
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": T * (V * size + 8 + 8 + case["top"] * 12), "flops": 5 * T * V}
    if case["op"] == "fork":
        prompt, lens, parents = _fork_plan(case)
        ps, B = case["page_size"], len(lens)
        moved = [p for b, p in enumerate(parents) if p >= 0 and p != b]
        parts = sum(1 for p in moved if lens[p] % ps)
        page = 2 * case["kv_heads"] * ps * case["head_dim"]
        # lengths and parents in, lengths and flags out, the tables of those that come or go in, of those that come out,
        # a page in and out per layer, keys and values for each that is not full
        entries = sum(_pages(lens[b], ps) for b, p in enumerate(parents) if p != b) + \
            2 * sum(_pages(lens[p], ps) for p in moved)
        return {"bytes": B * 13 + 8 + 4 * entries + 4 * parts + 2 * 2 * case["layers"] * parts * page, "flops": 2 * entries}
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    held = D // 2 + 4 * (D // GROUP)  # bytes of a 4-bit row
    if case["op"] == "write4":
        T = case["tokens"]
        rows = min(T, case["max_pos"])
        # q in and out, k and v in and, as the cache holds them, out, 4-bit rows out, table rows, positions, slots
        return {"bytes": T * (2 * D * (2 * H + 4 * Hkv) + 2 * Hkv * held) + rows * D * 4 + T * 12,
                "flops": T * D * (3 * (H + Hkv) + 2 * Hkv * 6)}
    ctx, new = _attn_lens(case)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    kv = sum(c + n for c, n in zip(ctx, new))
    blocks = sum(_pages(c + n, case["page_size"]) for c, n in zip(ctx, new))
    return {"bytes": 2 * D * 2 * H * sum(new) + 2 * Hkv * kv * held + 4 * blocks + 8 * len(ctx),
            "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_group(x):
    """(codes, scales, offsets, values) of rows [..., d], a group after another."""
    out = []
    for g in x.double().split(GROUP, dim=-1):
        m, top = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        # towards zero: binary exponent, then the type's digits of the significand cut off
        want = (top - m) / 15
        frac, power = torch.frexp(want)
        digits = {torch.float16: 11, torch.bfloat16: 8}[x.dtype]
        lowest = {torch.float16: -24, torch.bfloat16: -133}[x.dtype]
        unit = torch.ldexp(torch.ones_like(want), (power - digits).clamp(min=lowest))
        s = torch.floor(want / unit) * unit
        t = (g - m) / torch.where(s > 0, s, torch.ones_like(s))
        below = torch.floor(t)
        up = (t - below > 0.5) | ((t - below == 0.5) & (below % 2 == 1))
        c = torch.where(s > 0, (below + up).clamp(max=15), torch.zeros_like(t))
        out.append((c, s, m, (c * s + m).to(x.dtype).double()))
    return [torch.cat(parts, dim=-1) for parts in zip(*out)]


def _exact_write4(st):
    def turned(x):
        z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous())
        turn = torch.complex(st["cos"].double(), st["sin"].double()).index_select(0, st["positions"].long())
        return torch.view_as_real(z * turn.unsqueeze(1)).reshape(x.shape)

    q, k = turned(st["q"]), turned(st["k"]).to(st["k"].dtype)
    after, values = [], []
    for (codes, params), x in ((st["cache_k"], k), (st["cache_v"], st["v"])):
        pages, ps, Hkv = codes.shape[:3]
        c, s, m, held = _exact_group(x)
        flat = params.double().reshape(pages * ps, Hkv, -1, 2)
        rows = torch.stack([s, m], dim=-1)
        after.append((None, flat.index_copy(0, st["slots"], rows).view(params.shape)))
        values.append(held)
    return (q, *values, *after[0], *after[1])


def _exact_attn4(st, case):
    q, ps = st["q"], case["page_size"]
    rep = case["heads"] // case["kv_heads"]
    low = torch.arange(case["head_dim"], device=q.device) % 8
    byte = torch.arange(case["head_dim"], device=q.device) // 8 * 4 + low % 2 * 2 + low // 4
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    at = 0
    for b, n in enumerate(st["new"]):
        token = torch.arange(st["ctx"][b] + n, device=q.device)
        page = st["block_tables"][b].long()[token // ps]
        for h in range(case["kv_heads"]):
            rows = []
            for codes, params in (st["cache_k"], st["cache_v"]):
                c = codes[page, token % ps, h][:, byte].to(torch.int64)
                c = torch.where(low // 2 % 2 == 0, c % 16, c // 16).double()
                p = params[page, token % ps, h].double().repeat_interleave(GROUP, dim=1)
                rows.append((c * p[..., 0] + p[..., 1]).to(q.dtype).double())
            k, v = rows
            L = k.shape[0]
            for i in range(h * rep, (h + 1) * rep):
                for r in range(0, n, 1024):  # query i sees keys 0 .. L - n + i
                    some = q[at + r:at + min(n, r + 1024), i].double()
                    s = some @ k.t() / math.sqrt(q.shape[2])
                    seen = torch.ones(some.shape[0], L, dtype=torch.bool, device=q.device).tril(L - n + r)
                    s = s.where(seen, torch.full_like(s, -math.inf))
                    out[at + r:at + r + some.shape[0], i] = torch.softmax(s, dim=1) @ v
        at += n
    return out


def _exact_fork(st):
    lens, tables, parents = st["kv_lens"].tolist(), st["block_tables"].tolist(), st["parents"].tolist()
    ps, top = st["page_size"], int(st["n_free"].item())
    stack = st["free_pages"].tolist()
    both = st["both"].clone()
    before = [row[:_pages(c, ps)] for row, c in zip(tables, lens)]
    new_lens, granted, after, height = list(lens), [True] * len(lens), [list(p) for p in before], top
    asked = 0
    for b, p in enumerate(parents):
        if p < 0:
            new_lens[b], after[b] = 0, []
        elif p != b:
            part = lens[p] % ps != 0
            asked += part
            if part and asked > top:
                granted[b] = False
                continue
            new_lens[b], after[b] = lens[p], list(before[p])
            if part:
                height -= 1
                after[b][-1] = stack[height]
                both[:, :, stack[height]] = st["both"][:, :, before[p][-1]]
    still = {page for row in after for page in row}
    for row in before:
        for page in row:
            if page not in still:
                still.add(page)
                stack[height] = page
                height += 1
    for row, pages in zip(tables, after):
        row[:len(pages)] = pages
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(new_lens, **i32), torch.tensor([height], **i32), torch.tensor(granted, device="cuda"),
            torch.tensor(tables, **i32), torch.tensor(stack, **i32), both.double())


def _exact_logprobs(st, case):
    logits, tokens, k = st["logits"], st["tokens"], case["top"]
    chosen, entropy, ids, best = [], [], [], []
    for at in range(0, logits.shape[0], 128):
        p = torch.log_softmax(logits[at:at + 128].double(), dim=1)
        chosen.append(p.gather(1, tokens[at:at + 128, None]).view(-1))
        entropy.append(-(p.exp() * p).sum(1))
        if k:
            order = torch.sort(logits[at:at + 128].double(), dim=1, descending=True, stable=True).indices[:, :k]
            ids.append(order)
            best.append(p.gather(1, order))
    out = (torch.cat(chosen), torch.cat(entropy))
    return out + (torch.cat(ids), torch.cat(best)) if k else out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "write4":
        return _exact_write4(st)
    if case["op"] == "attn4":
        return _exact_attn4(st, case)
    return _exact_fork(st) if case["op"] == "fork" else _exact_logprobs(st, case)
