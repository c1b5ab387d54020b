"""Workloads of the paged-cache operators (llama.paged) and their plain forms.

Four operators carry one step of a serving loop over a paged KV cache:

  paged_append       the step's bookkeeping: pages for the new tokens from a free stack, block
                     tables, positions and cache slots, from the requests' lengths
  rope_paged_write   rotary positions on the new queries and keys, keys and values into their slots
  prompt_attention   causal grouped-query attention of whole prompts packed one after another
  paged_attention    causal grouped-query attention of each request's new tokens (one token, a few,
                     or a chunk of a prompt) over everything the cache holds of that request

Every case is a dict of plain values.  Lengths follow from the case alone (`lens_seed`), values and
page orders from the seed given to prepare().  With own = False run() computes in elementary torch
operations in 32 bits and rounds once; with own = True it makes the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-efficient-inference_b200")


def _paged():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from llama import paged

    return paged


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a middling batch: every request appends one token
        dict(name="append_decode", op="append", requests=64, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=4096,
             page_size=16, max_len=4352, lens_seed=1),
        # a step that admits many ragged prompts beside requests that append nothing
        dict(name="append_prompts", op="append", requests=256, new_lo=0, new_hi=509, ctx_lo=0, ctx_hi=2000,
             page_size=32, max_len=8192, lens_seed=2),
        # RoPE and cache write of a decode step at batch 16 (Llama-3.2-1B heads)
        dict(name="rope_decode", op="rope", type="float16", heads=32, kv_heads=8, head_dim=64, tokens=16,
             page_size=16, max_pos=8192, lens_seed=3),
        # the same for a packed prompt step, an odd number of tokens, 128-wide heads
        dict(name="rope_prompt", op="rope", type="bfloat16", heads=32, kv_heads=8, head_dim=128, tokens=16381,
             page_size=64, max_pos=32768, lens_seed=4),
        # three short prompts: latency counts
        dict(name="prompt_short", op="prompt", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=3,
             tokens=211, lens_seed=5),
        # a ragged batch of prompts (Llama-3.2-1B heads)
        dict(name="prompt_ragged", op="prompt", type="bfloat16", heads=32, kv_heads=8, head_dim=64, seqs=16,
             tokens=15001, lens_seed=6),
        # one long prompt, 128-wide heads
        dict(name="prompt_long", op="prompt", type="float16", heads=32, kv_heads=8, head_dim=128, seqs=1,
             tokens=8192, lens_seed=7),
        # a decode step at batch 1 over the benchmark's context (512 prompt tokens and a few more)
        dict(name="decode_single", op="paged", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=1,
             new=1, chunks=0, chunk=0, ctx_lo=575, ctx_hi=575, page_size=16, lens_seed=8),
        # a decode step at batch 64, contexts from a few hundred tokens to 16 thousand
        dict(name="decode_batch", op="paged", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=64,
             new=1, chunks=0, chunk=0, ctx_lo=300, ctx_hi=16000, page_size=16, lens_seed=9),
        # few requests with long contexts, two tokens each (one drafted), 128-wide heads, a group of seven
        dict(name="decode_long", op="paged", type="bfloat16", heads=28, kv_heads=4, head_dim=128, seqs=4,
             new=2, chunks=0, chunk=0, ctx_lo=30001, ctx_hi=120000, page_size=64, lens_seed=10),
        # chunks of four prompts over what the cache holds already
        dict(name="chunk_prefill", op="paged", type="float16", heads=32, kv_heads=8, head_dim=64, seqs=4,
             new=1, chunks=4, chunk=1021, ctx_lo=500, ctx_hi=8000, page_size=16, lens_seed=11),
        # a mixed step: one chunk of a prompt among decoding requests, 128-wide heads
        dict(name="chunk_mixed", op="paged", type="bfloat16", heads=32, kv_heads=8, head_dim=128, seqs=32,
             new=1, chunks=1, chunk=512, ctx_lo=200, ctx_hi=6000, page_size=32, lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "rope", "prompt", "prompt", "paged", "paged", "paged"])
    heads = dict(type=rng.choice(["float16", "bfloat16"]), head_dim=rng.choice([64, 128]))
    heads["kv_heads"] = rng.choice([1, 2, 4, 8])
    heads["heads"] = heads["kv_heads"] * rng.choice([1, 2, 3, 4, 6, 7, 8])
    if heads["heads"] > 32:
        heads["heads"] = heads["kv_heads"] * 4
    page_size = rng.choice([8, 16, 32, 64, 128])
    lens_seed = rng.randrange(1 << 30)
    if op == "append":
        requests = _log_int(rng, 1, 256)
        new_hi = _log_int(rng, 1, 500)
        ctx_hi = _log_int(rng, 16, 4000)
        return dict(op=op, requests=requests, new_lo=rng.choice([0, 1]), new_hi=new_hi, ctx_lo=rng.choice([0, 1]),
                    ctx_hi=ctx_hi, page_size=page_size, max_len=ctx_hi + new_hi + rng.randrange(600),
                    lens_seed=lens_seed)
    if op == "rope":
        return dict(op=op, **heads, tokens=_log_int(rng, 1, 16000), page_size=page_size,
                    max_pos=_log_int(rng, 512, 32768), lens_seed=lens_seed)
    if op == "prompt":
        seqs = _log_int(rng, 1, 32)
        return dict(op=op, **heads, seqs=seqs, tokens=max(seqs, _log_int(rng, 1, 8000)), lens_seed=lens_seed)
    kind = rng.choice(["decode", "decode", "chunk", "mixed"])
    if kind == "decode":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, min(100000, 250000 // seqs))
        return dict(op="paged", **heads, seqs=seqs, new=rng.choice([1, 1, 1, 2, 4]), chunks=0, chunk=0,
                    ctx_lo=max(1, hi // rng.choice([1, 4, 64])), ctx_hi=hi, page_size=page_size, lens_seed=lens_seed)
    seqs = _log_int(rng, 1, 8) if kind == "chunk" else _log_int(rng, 2, 32)
    chunks = seqs if kind == "chunk" else max(1, seqs // 8)
    return dict(op="paged", **heads, seqs=seqs, new=1, chunks=chunks, chunk=_log_int(rng, 2, 4000 // chunks),
                ctx_lo=1, ctx_hi=_log_int(rng, 1, 8000), page_size=page_size, lens_seed=lens_seed)


# ---------------------------------------------------------------------------------------------
# lengths (from the case alone)
# ---------------------------------------------------------------------------------------------
def _append_lens(case):
    rng = random.Random(case["lens_seed"])
    ctx, new = [], []
    for _ in range(case["requests"]):
        ctx.append(rng.randint(case["ctx_lo"], case["ctx_hi"]))
        new.append(rng.randint(case["new_lo"], case["new_hi"]))
    return ctx, new


def _prompt_lens(case):
    """`tokens` cut into `seqs` ragged prompts of at least one token."""
    rng = random.Random(case["lens_seed"])
    weights = [math.exp(rng.gauss(0.0, 0.8)) for _ in range(case["seqs"])]
    spare = case["tokens"] - case["seqs"]
    lens = [1 + int(spare * w / sum(weights)) for w in weights]
    lens[-1] += case["tokens"] - sum(lens)
    return lens


def _paged_lens(case):
    """(tokens the cache holds before the step, new tokens) per request."""
    rng = random.Random(case["lens_seed"])
    ctx = [_log_int(rng, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    new = [case["new"]] * case["seqs"]
    for b in rng.sample(range(case["seqs"]), case["chunks"]):
        new[b] = case["chunk"]
    return ctx, new


def _pages(n, page_size):
    return -(-n // page_size)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _keys(shape, dtype, gen):
    """Keys with a few strong channels, as trained models have them."""
    k = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    offset = torch.randn(shape[-2:], generator=gen, device="cuda") * 0.5
    return (k + offset).to(dtype)


def _cache(num_pages, case, dtype, gen, keys=False):
    """A cache of [num_pages, page_size, kv_heads, head_dim], each page and head contiguous."""
    shape = (num_pages, case["kv_heads"], case["page_size"], case["head_dim"])
    t = torch.empty(shape, dtype=dtype, device="cuda")
    offset = torch.randn(case["kv_heads"], 1, case["head_dim"], generator=gen, device="cuda") * (0.5 if keys else 0.0)
    for at in range(0, num_pages, 1024):  # in pieces: the 32-bit values are never held whole
        part = t[at:at + 1024]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") + offset)
    return t.transpose(1, 2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"op": case["op"], "case": case}
    if case["op"] == "append":
        ctx, new = _append_lens(case)
        ps = case["page_size"]
        need = sum(_pages(c + n, ps) for c, n in zip(ctx, new))
        held = sum(_pages(c, ps) for c in ctx)
        pool = need + 37
        order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
        tables = torch.zeros(len(ctx), _pages(case["max_len"], ps), dtype=torch.int32, device="cuda")
        at = 0
        for b, c in enumerate(ctx):
            n = _pages(c, ps)
            tables[b, :n] = order[at:at + n]
            at += n
        free = torch.zeros(pool, dtype=torch.int32, device="cuda")
        free[:pool - held] = order[held:]
        st.update(kv_lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"),
                  new_lens=torch.tensor(new, dtype=torch.int32, device="cuda"), block_tables=tables,
                  free_pages=free, n_free=torch.tensor([pool - held], dtype=torch.int32, device="cuda"),
                  page_size=ps, num_tokens=sum(new))
        return st
    dtype = getattr(torch, case["type"])
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        T, ps = case["tokens"], case["page_size"]
        num_pages = _pages(T, ps) + 5
        # a fused projection's output: the rows of q, k and v are parts of one wide row
        qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=gen, device="cuda").to(dtype)
        inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        angles = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * inv
        st.update(q=qkv[:, :H * D].view(T, H, D), k=qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D),
                  v=qkv[:, (H + Hkv) * D:].view(T, Hkv, D), cos=angles.cos().float(), sin=angles.sin().float(),
                  positions=torch.randint(0, case["max_pos"], (T,), generator=gen, device="cuda", dtype=torch.int32),
                  slots=torch.randperm(num_pages * ps, generator=gen, device="cuda")[:T].contiguous(),
                  cache_k=_cache(num_pages, case, dtype, gen, keys=True), cache_v=_cache(num_pages, case, dtype, gen))
        return st
    if case["op"] == "prompt":
        lens = _prompt_lens(case)
        T = sum(lens)
        st.update(lens=lens, q=torch.randn(T, H, D, generator=gen, device="cuda").to(dtype),
                  k=_keys((T, Hkv, D), dtype, gen), v=torch.randn(T, Hkv, D, generator=gen, device="cuda").to(dtype),
                  cu_seqlens=torch.tensor(_cumulative(lens), dtype=torch.int32, device="cuda"), max_len=max(lens))
        return st
    ctx, new = _paged_lens(case)
    ps = case["page_size"]
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
              cache_k=_cache(num_pages, case, dtype, gen, keys=True), cache_v=_cache(num_pages, case, dtype, gen),
              block_tables=tables, kv_lens=torch.tensor(kv, dtype=torch.int32, device="cuda"),
              cu_seqlens=torch.tensor(_cumulative(new), dtype=torch.int32, device="cuda"), max_new=max(new))
    return st


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _plain_append(st):
    ctx, new, ps, T = st["kv_lens"].long(), st["new_lens"].long(), st["page_size"], st["num_tokens"]
    tables, free, n_free = st["block_tables"], st["free_pages"], st["n_free"].long()
    B, width = tables.shape
    held, want = (ctx + ps - 1) // ps, (ctx + new + ps - 1) // ps
    need = torch.where(want > width, 0, want - held)
    upto = need.cumsum(0)
    granted = (want <= width) & ((need == 0) | (upto <= n_free))
    # page j of request b, for held <= j < want, is the next one from the top of the free stack
    j = torch.arange(width, device=tables.device)
    fresh = granted[:, None] & (j >= held[:, None]) & (j < want[:, None])
    rank = (upto - need)[:, None] + j - held[:, None]
    page = free[(n_free - 1 - rank).clamp(0, free.numel() - 1)]
    tables.copy_(torch.where(fresh, page, tables))
    cu = torch.zeros(B + 1, dtype=torch.int32, device=tables.device)
    cu[1:] = new.cumsum(0)
    owner = torch.repeat_interleave(torch.arange(B, device=tables.device), new, output_size=T)
    pos = ctx[owner] + torch.arange(T, device=tables.device) - cu.long()[owner]
    slot = tables[owner, (pos // ps).clamp(max=width - 1)].long() * ps + pos % ps
    slots = torch.where(granted[owner], slot, -1)
    taken = torch.where(granted, need, 0).sum()
    return (tables, cu, pos.int(), slots, torch.where(granted, ctx + new, ctx).int(), (n_free - taken).int(), granted)


def _rotate(x, cos, sin):
    x = x.float()
    even, odd = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.stack([even * c - odd * s, even * s + odd * c], dim=-1).flatten(-2)


def _plain_rope(st):
    q, k, v, ps = st["q"], st["k"], st["v"], st["cache_k"].shape[1]
    pos = st["positions"].long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    q_rot, k_rot = _rotate(q, cos, sin).to(q.dtype), _rotate(k, cos, sin).to(k.dtype)
    page, row = st["slots"] // ps, st["slots"] % ps
    st["cache_k"][page, row] = k_rot
    st["cache_v"][page, row] = v
    return q_rot, k_rot, st["cache_k"], st["cache_v"]


def _attend(q, k, v, out):
    """Causal attention of the last q.shape[0] tokens over k / v [L, kv_heads, d], a KV head at a time."""
    n, H, D = q.shape
    L, Hkv = k.shape[:2]
    rep = H // Hkv
    hidden = torch.arange(L, device=q.device)[None, :] > torch.arange(n, device=q.device)[:, None] + (L - n)
    for h in range(Hkv):
        qs = q[:, h * rep:(h + 1) * rep].float().transpose(0, 1)  # [rep, n, D]
        s = torch.matmul(qs, k[:, h].float().t()) * (1.0 / math.sqrt(D))
        s = s.masked_fill(hidden, float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(e, v[:, h].float()) / e.sum(-1, keepdim=True)
        out[:, h * rep:(h + 1) * rep] = o.transpose(0, 1).to(out.dtype)


def _plain_prompt(st):
    q, k, v = st["q"], st["k"], st["v"]
    out = torch.empty_like(q)
    at = 0
    for n in st["lens"]:
        _attend(q[at:at + n], k[at:at + n], v[at:at + n], out[at:at + n])
        at += n
    return out


def _plain_paged(st):
    q, ps = st["q"], st["cache_k"].shape[1]
    out = torch.empty_like(q)
    at = 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["new"])):
        pages = st["block_tables"][b, :_pages(c + n, ps)].long()
        k = st["cache_k"][pages].flatten(0, 1)[:c + n]
        v = st["cache_v"][pages].flatten(0, 1)[:c + n]
        _attend(q[at:at + n], k, v, out[at:at + n])
        at += n
    return out


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if not own:
        return {"append": _plain_append, "rope": _plain_rope, "prompt": _plain_prompt, "paged": _plain_paged}[op](st)
    paged = _paged()
    if op == "append":
        step = paged.paged_append(st["kv_lens"], st["new_lens"], st["block_tables"], st["free_pages"], st["n_free"],
                                  st["page_size"], st["num_tokens"])
        return (st["block_tables"], step.cu_seqlens, step.positions, step.slots, step.kv_lens, step.n_free,
                step.granted)
    if op == "rope":
        q_rot, k_rot = paged.rope_paged_write(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"],
                                              st["slots"], st["cache_k"], st["cache_v"])
        return q_rot, k_rot, st["cache_k"], st["cache_v"]
    if op == "prompt":
        return paged.prompt_attention(st["q"], st["k"], st["v"], st["cu_seqlens"], st["max_len"])
    return paged.paged_attention(st["q"], st["cache_k"], st["cache_v"], st["block_tables"], st["kv_lens"],
                                 st["cu_seqlens"], st["max_new"])


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "append":
        ctx, new = _append_lens(case)
        ps = case["page_size"]
        fresh = sum(_pages(c + n, ps) - _pages(c, ps) for c, n in zip(ctx, new))
        open_pages = sum(1 for c, n in zip(ctx, new) if n and c % ps)
        B, T = len(ctx), sum(new)
        # lengths in and out, offsets, flags; a free page in and a table entry out per new page;
        # a table entry in per open page; position and slot per token
        return {"bytes": B * (4 + 4 + 4 + 4 + 1) + 12 + fresh * 8 + open_pages * 4 + T * 12, "flops": T * 4}
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        T = case["tokens"]
        rows = min(T, case["max_pos"])
        # q and k in and out, the rotated k and v into the cache, table rows, positions and slots
        return {"bytes": 2 * T * D * (2 * H + 2 * Hkv + 3 * Hkv - Hkv) + rows * D * 4 + T * 12,
                "flops": 3 * T * D * (H + Hkv)}
    if case["op"] == "prompt":
        lens = _prompt_lens(case)
        pairs = sum(n * (n + 1) // 2 for n in lens)
        T = sum(lens)
        return {"bytes": 2 * T * D * (2 * H + 2 * Hkv) + 4 * (len(lens) + 1), "flops": 4 * D * H * pairs}
    ctx, new = _paged_lens(case)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    kv = sum(c + n for c, n in zip(ctx, new))
    blocks = sum(_pages(c + n, case["page_size"]) for c, n in zip(ctx, new))
    return {"bytes": 2 * D * (2 * H * sum(new) + 2 * Hkv * kv) + 4 * blocks + 8 * len(ctx),
            "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, one request and one head at a time
# ---------------------------------------------------------------------------------------------
def _exact_append(st):
    ctx, new = st["kv_lens"].tolist(), st["new_lens"].tolist()
    tables, stack = st["block_tables"].tolist(), st["free_pages"].tolist()
    top, ps = int(st["n_free"].item()), st["page_size"]
    stack = stack[:top]
    asked = 0
    cu, positions, slots, lens, granted = [0], [], [], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        held, want = _pages(c, ps), _pages(c + n, ps)
        fits = want <= len(tables[b])
        asked += want - held if fits else 0
        ok = fits and (want == held or asked <= top)
        if ok:
            for j in range(held, want):
                tables[b][j] = stack.pop()
        for p in range(c, c + n):
            positions.append(p)
            slots.append(tables[b][p // ps] * ps + p % ps if ok else -1)
        cu.append(cu[-1] + n)
        lens.append(c + n if ok else c)
        granted.append(ok)
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(tables, **i32), torch.tensor(cu, **i32), torch.tensor(positions, **i32),
            torch.tensor(slots, dtype=torch.int64, device="cuda"), torch.tensor(lens, **i32),
            torch.tensor([len(stack)], **i32), torch.tensor(granted, device="cuda"))


def _exact_rope(st):
    def turned(x):
        z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous())
        turn = torch.complex(st["cos"].double(), st["sin"].double()).index_select(0, st["positions"].long())
        return torch.view_as_real(z * turn.unsqueeze(1)).reshape(x.shape)

    q, k = turned(st["q"]), turned(st["k"])
    pages, ps, Hkv, D = st["cache_k"].shape
    after = []
    for cache, rows in ((st["cache_k"], k), (st["cache_v"], st["v"].double())):
        flat = cache.double().reshape(pages * ps, Hkv, D)
        flat = flat.index_copy(0, st["slots"], rows)
        after.append(flat.view(pages, ps, Hkv, D))
    return q, k, after[0], after[1]


def _exact_rows(q, k, v):
    """q [n, D] over k / v [L, D], float64: query i sees keys 0 .. L - n + i; blocks of queries."""
    n, L, out = q.shape[0], k.shape[0], []
    for at in range(0, n, 1024):
        some = q[at:at + 1024]
        seen = min(L, L - n + at + some.shape[0])
        s = some @ k[:seen].t() / math.sqrt(q.shape[1])
        allowed = torch.ones(some.shape[0], seen, dtype=torch.bool, device=q.device).tril(L - n + at)
        p = torch.softmax(s.where(allowed, torch.full_like(s, -math.inf)), dim=1)
        out.append(p @ v[:seen])
    return torch.cat(out)


def _exact_attention(st, case):
    q = st["q"]
    rep = case["heads"] // case["kv_heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    new = st["lens"] if case["op"] == "prompt" else st["new"]
    at = 0
    for b, n in enumerate(new):
        if case["op"] == "prompt":
            k, v = st["k"][at:at + n], st["v"][at:at + n]
        else:
            ps = st["cache_k"].shape[1]
            token = torch.arange(st["ctx"][b] + n, device=q.device)
            page = st["block_tables"][b].long()[token // ps]
            k, v = st["cache_k"][page, token % ps], st["cache_v"][page, token % ps]
        for h in range(case["heads"]):
            out[at:at + n, h] = _exact_rows(q[at:at + n, h].double(), k[:, h // rep].double(), v[:, h // rep].double())
        at += n
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(st)
    if case["op"] == "rope":
        return _exact_rope(st)
    return _exact_attention(st, case)
