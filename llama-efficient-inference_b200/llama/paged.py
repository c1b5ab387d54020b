"""Serving over a paged KV cache: packed prompts, chunks and single tokens in one step.

The reference keeps one [max_batch, max_seq] cache per layer and pads every prompt of a batch to the
longest (llama/model.py:195-215, llama/generation.py:6-82).  Here the cache is a pool of pages that
block tables name per request, and a step's new tokens of all requests stand one after another
([tokens, heads, head_dim], no padding).  One step is

  paged_append       pages, block tables, positions, slots from the requests' lengths  (li4_paged_append)
  per layer:
    rope_paged_write   RoPE on q and k, keys and values into their slots           (li4_rope_paged_write)
    prompt_attention   whole prompts, from the packed keys and values              (li4_prompt_attention)
    paged_attention    anything else, from the cache                               (li4_paged_attention)

With PagedKVCache(bits=4) the cache holds keys and values in 4 bits (5 with their parameters): rope_paged_write_int4 and
paged_attention_int4 (li4_rope_paged_write_int4, li4_paged_attention_int4) take the places of their 16-bit forms, and
whole prompts attend to the values that the cache holds.  Requests go on from one another's tokens, sharing full pages, and
end by paged_fork (li4_paged_fork): several answers to a prompt, the steps of a search, PagedKVCache.release.

The lengths live on the GPU: no call reads them on the host, so a step can be captured in a CUDA graph
and replayed while the requests grow.  PagedKVCache holds the pool, Llama.forward_paged runs the model's
blocks over it, Generation.generate_paged is the loop around them.

Every function runs on the current stream of its tensors' device, allocates its outputs (unless they are
given) and its workspace there, and raises RuntimeError subclasses for arguments it does not take.  None has a backward
pass: tensors that require grad are refused outside torch.no_grad(); and none is a registered operator: fake tensors
and calls under a tracer are refused.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch
from torch.utils._python_dispatch import is_in_torch_dispatch_mode

from . import _native as native


class PagedStep(NamedTuple):
    """What paged_append works out for one step (all on the GPU)."""

    cu_seqlens: torch.Tensor  # int32 [requests + 1]: first packed token of each request
    positions: torch.Tensor   # int32 [tokens]
    slots: torch.Tensor       # int64 [tokens]: page * page_size + row; -1: refused or past the last request
    kv_lens: torch.Tensor     # int32 [requests], the step's tokens included
    n_free: torch.Tensor      # int32 [1]
    granted: torch.Tensor     # bool [requests]


class PagedFork(NamedTuple):
    """What paged_fork leaves (all on the GPU)."""

    kv_lens: torch.Tensor  # int32 [requests]
    n_free: torch.Tensor   # int32 [1]
    granted: torch.Tensor  # bool [requests]


class Int4Pages(NamedTuple):
    """Keys or values of a paged cache in 4 bits: groups of 32 dims with a scale s and an offset m stand for c s + m,
    rounded to the type of s and m."""

    codes: torch.Tensor   # uint8 [pages, page_size, kv_heads, head_dim / 2], see pack_codes
    params: torch.Tensor  # float16 or bfloat16 [pages, page_size, kv_heads, head_dim / 32, 2]: (s, m)

    def values(self) -> torch.Tensor:
        """The 16-bit values [pages, page_size, kv_heads, head_dim] (plain tensor operations: for looking, not for steps)."""
        c = unpack_codes(self.codes).unflatten(-1, (-1, 32)).double()
        p = self.params.double()
        return (c * p[..., 0:1] + p[..., 1:2]).to(self.params.dtype).flatten(-2)


_CODE_BITS = (0, 16, 4, 20, 8, 24, 12, 28)  # where in its 32-bit word the code of dim 0 .. 7 begins


def pack_codes(codes: torch.Tensor) -> torch.Tensor:
    """Codes 0 .. 15 [..., head_dim] as the cache holds them, uint8 [..., head_dim / 2]."""
    at = torch.tensor(_CODE_BITS, dtype=torch.int32, device=codes.device)
    return (codes.to(torch.int32).unflatten(-1, (-1, 8)) << at).sum(-1, dtype=torch.int32).view(torch.uint8)


def unpack_codes(packed: torch.Tensor) -> torch.Tensor:
    """The codes [..., head_dim] (int32) of packed rows [..., head_dim / 2]."""
    at = torch.tensor(_CODE_BITS, dtype=torch.int32, device=packed.device)
    return ((packed.contiguous().view(torch.int32).unsqueeze(-1) >> at) & 15).flatten(-2)


MAX_FORK_REQUESTS = 8192  # li4_paged_fork's


def _runs_now(*tensors: torch.Tensor) -> bool:
    """Whether a call on these tensors is made at once on the GPU: plain CUDA tensors, outside of any tracing."""
    return not torch.compiler.is_compiling() and not torch.jit.is_tracing() and not is_in_torch_dispatch_mode() and \
        all(type(t) is torch.Tensor and t.is_cuda for t in tensors)


def _done(what: str, result):
    """The binding's result; a li4_status in its place raises."""
    if type(result) is int:
        native.check(result, what)
    return result


def paged_append(kv_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
                 n_free: torch.Tensor, page_size: int, num_tokens: int, kv_lens_out: Optional[torch.Tensor] = None,
                 n_free_out: Optional[torch.Tensor] = None, max_len: Optional[int] = None) -> PagedStep:
    """One step's bookkeeping (li4_paged_append_within): request b holds kv_lens[b] tokens and appends new_lens[b].

    kv_lens, new_lens int32 [requests]; block_tables int32 [requests, blocks], the entries of the step's fresh
    pages are written; free_pages int32 [capacity] with the free ones in free_pages[:n_free], taken from the top;
    n_free int32 [1]; num_tokens = sum(new_lens), which the host knows.  kv_lens_out / n_free_out may be kv_lens /
    n_free (in place); by default they are new tensors.  A request that does not fit (more than max_len tokens with
    the new ones, table too narrow, too few pages for it and those before it) is refused whole: granted False, length
    kept, slots -1."""
    return PagedStep._make(_done("paged_append", native.ext().paged_append(
        kv_lens, new_lens, block_tables, free_pages, n_free, page_size, num_tokens, kv_lens_out, n_free_out,
        max_len)))


def rope_paged_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                     positions: torch.Tensor, slots: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                     q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                     need_k: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RoPE on packed q [T, heads, d] and k [T, kv_heads, d] and the cache write of k and v (li4_rope_paged_write).

    Pairs (2i, 2i + 1) turn by the angle in row positions[t] of cos / sin (fp32 [positions, d / 2]), in fp32.  The
    turned key and the value of token t go to row slots[t] % page_size of page slots[t] // page_size of cache_k /
    cache_v [pages, page_size, kv_heads, d] (any strides with contiguous rows); negative slots are skipped.
    Returns (turned q, turned k); q_out / k_out may be q / k themselves and overlap nothing else.  need_k = False leaves the packed turned
    keys out (returns None for them): attention over the cache does not read them."""
    return _done("rope_paged_write", native.ext().rope_paged_write(q, k, v, cos, sin, positions, slots, cache_k, cache_v,
                                                                   q_out, k_out, need_k))


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_len: int,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of whole prompts packed one after another (li4_prompt_attention).

    q [T, heads, d], k and v [T, kv_heads, d] in float16 or bfloat16 (d a multiple of 8 up to 128, heads a
    multiple of kv_heads); cu_seqlens int32 [prompts + 1] on the GPU: prompt b is rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1; max_len: the longest prompt, known to the host (it picks the kernel; a wrong value costs
    time, not correctness).  Softmax of scale q k^T (default 1 / sqrt(d)) in fp32.  Rows past the last prompt are
    left as they were in `out`.  out must not overlap q, k or v."""
    return _done("prompt_attention", native.ext().prompt_attention(q, k, v, cu_seqlens, max_len, scale, out))


def paged_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, block_tables: torch.Tensor,
                    kv_lens: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of each request's new tokens over the paged cache (li4_paged_attention).

    q [T, heads, d]: request b's n queries are rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (one token, a few, a
    chunk of a prompt, none; different requests may differ); cache_k / cache_v [pages, page_size, kv_heads, d];
    block_tables int32 [requests, blocks]; kv_lens int32 [requests], the new tokens included (their keys are in the
    cache already): query i sees keys 0 .. kv_len - n + i, and gives zeros where that is none.  Block-table entries
    outside the cache read as zero keys and values.  max_new: the most queries of a request, known to the host (it
    picks the kernels; a wrong value costs time, not correctness).  out must not overlap q or the cache."""
    return _done("paged_attention", native.ext().paged_attention(q, cache_k, cache_v, block_tables, kv_lens, cu_seqlens,
                                                                 max_new, scale, out))


def rope_paged_write_int4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                          positions: torch.Tensor, slots: torch.Tensor, cache_k: Int4Pages, cache_v: Int4Pages,
                          q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                          v_out: Optional[torch.Tensor] = None,
                          need_kv: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """rope_paged_write into a cache in 4 bits (li4_rope_paged_write_int4); head_dim a multiple of 32 up to 128.

    A group of 32 values x gets m = the smallest, s = (the largest - m) / 15 rounded towards zero to the type, and codes
    min(15, (x - m) / s to the nearest, ties to even), 0 where s is 0; a key is turned in 64 bits and rounded first, so
    the codes are a function of the inputs alone.  A group with a value that is not finite reads as NaN.
    Returns (turned q, k, v): k and v packed, as the cache holds them, for prompt_attention.  need_kv = False leaves them
    out (None).  q_out / k_out / v_out may be q / k / v themselves and overlap nothing else."""
    return _done("rope_paged_write_int4", native.ext().rope_paged_write_int4(
        q, k, v, cos, sin, positions, slots, cache_k, cache_v, q_out, k_out, v_out, need_kv))


def paged_attention_int4(q: torch.Tensor, cache_k: Int4Pages, cache_v: Int4Pages, block_tables: torch.Tensor,
                         kv_lens: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_attention over a cache in 4 bits (li4_paged_attention_int4): the same function of the 16-bit values that
    the cache stands for, with the same arguments; cache_k / cache_v are Int4Pages (or pairs) of q's type."""
    return _done("paged_attention_int4", native.ext().paged_attention_int4(
        q, cache_k, cache_v, block_tables, kv_lens, cu_seqlens, max_new, scale, out))


def paged_fork(kv_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor,
               parents: torch.Tensor, page_size: int, pools: Sequence[torch.Tensor] = (),
               kv_lens_out: Optional[torch.Tensor] = None, n_free_out: Optional[torch.Tensor] = None) -> PagedFork:
    """Requests that go on from others, and that end (li4_paged_fork): parents int32 [requests] names for each request
    itself (it stays), another (it holds that one's tokens from now on, as they were before the call) or -1 (it ends).

    Full pages are shared, a last page that is not full is copied into one from the top of the free stack, in every tensor
    of pools ([pages, ...], each page one block of memory).  A request whose copy finds no page, or whose parent is none,
    stays as it was (granted False).  Pages are 0 .. len(free_pages) - 1; other entries of block_tables count as no page and
    are not copied.  Pages that no request holds any more go back on the stack, in the order of requests
    and blocks.  block_tables and free_pages are updated in place; kv_lens_out / n_free_out may be kv_lens / n_free (in
    place), by default they are new tensors; what is written overlaps nothing else, and pools overlap one another at most in
    the same pages.  Sharing is read off the tables: append and this are all there is to call."""
    return PagedFork._make(_done("paged_fork", native.ext().paged_fork(
        kv_lens, block_tables, free_pages, n_free, parents, page_size, pools, kv_lens_out, n_free_out)))


class PagedKVCache:
    """Pages, block tables and lengths of up to max_requests requests of up to max_len tokens each.

    k[i] / v[i] are layer i's pages [num_pages, page_size, kv_heads, head_dim], or with bits = 4 its Int4Pages; each
    (page, head) is contiguous in memory, so the rows a KV head reads of a page are one run.  Request r is row r of
    block_tables and kv_lens for as long as it lives; fork() lets it go on from another, release() returns its pages."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 max_requests: int, max_len: int, dtype: torch.dtype = torch.float16, device="cuda", bits: int = 16):
        if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size}: a power of two from 8 to 1024")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"cache dtype {dtype}: float16 or bfloat16")
        if head_dim % 8 or not 8 <= head_dim <= 128:
            raise ValueError(f"head_dim {head_dim}: a multiple of 8 up to 128")
        if bits not in (4, 16) or (bits == 4 and head_dim % 32):
            raise ValueError(f"a cache of {bits} bits with head_dim {head_dim}: 16, or 4 with head_dim a multiple of 32")
        self.page_size, self.max_len, self.bits = page_size, max_len, bits

        def pages(row, kind):  # a layer's after another
            return [t.transpose(1, 2)
                    for t in torch.zeros(n_layers, num_pages, n_kv_heads, page_size, *row, dtype=kind, device=device)]

        if bits == 16:
            self.k, self.v = pages([head_dim], dtype), pages([head_dim], dtype)
        else:
            self.k, self.v = ([Int4Pages(c, p) for c, p in zip(pages([head_dim // 2], torch.uint8),
                                                               pages([head_dim // 32, 2], dtype))] for _ in range(2))
        i32 = dict(dtype=torch.int32, device=device)
        self.block_tables = torch.zeros(max_requests, -(-max_len // page_size), **i32)
        self.kv_lens = torch.zeros(max_requests, **i32)
        # one entry more than pages: release() drops what it does not return there
        self._stack = torch.cat([torch.arange(num_pages - 1, -1, -1, **i32), torch.zeros(1, **i32)])
        self.free_pages = self._stack[:num_pages]
        self.n_free = torch.full((1,), num_pages, **i32)

    @property
    def pools(self) -> List[torch.Tensor]:
        """All tensors of pages."""
        return self.k + self.v if self.bits == 16 else [t for pair in self.k + self.v for t in pair]

    def append(self, new_lens: torch.Tensor, num_tokens: int) -> PagedStep:
        """Takes pages for new_lens[r] more tokens of every request r (int32 [max_requests], zeros for idle rows);
        num_tokens is their sum.  Updates the cache's lengths, tables and free pages in place.  A request that does not
        fit, or that would hold more than max_len tokens, is refused whole (step.granted)."""
        return paged_append(self.kv_lens, new_lens, self.block_tables, self.free_pages, self.n_free, self.page_size,
                            num_tokens, kv_lens_out=self.kv_lens, n_free_out=self.n_free, max_len=self.max_len)

    def fork(self, parents: torch.Tensor) -> torch.Tensor:
        """Every request r goes on from request parents[r] (int32 [max_requests]): itself, another, or none (-1: it ends);
        see paged_fork.  Updates lengths, tables, free pages and the copied pages in place; returns granted
        bool [max_requests].  No host synchronisation."""
        return paged_fork(self.kv_lens, self.block_tables, self.free_pages, self.n_free, parents, self.page_size,
                          self.pools, kv_lens_out=self.kv_lens, n_free_out=self.n_free).granted

    def release(self, finished: torch.Tensor) -> None:
        """Returns the pages of the requests flagged in finished (bool [max_requests]), those that no other request
        shares, and sets their lengths to 0.  No host synchronisation."""
        n = self.kv_lens.shape[0]
        if _runs_now(self.kv_lens, self.block_tables, self.free_pages, self.n_free, finished) and n <= MAX_FORK_REQUESTS:
            parents = torch.arange(n, dtype=torch.int32, device=self.kv_lens.device).masked_fill_(finished, -1)
            paged_fork(self.kv_lens, self.block_tables, self.free_pages, self.n_free, parents, self.page_size,
                       kv_lens_out=self.kv_lens, n_free_out=self.n_free)  # (nothing is copied: no pools)
        else:
            self._release_by_index(finished)

    def _release_by_index(self, finished: torch.Tensor) -> None:
        """release() in tensor operations, for what paged_fork refuses: off the GPU, fake tensors, tracers, more requests."""
        table, pages = self.block_tables, self.free_pages.shape[0]
        held = torch.div(self.kv_lens + (self.page_size - 1), self.page_size, rounding_mode="floor")
        block = torch.arange(table.shape[1], device=table.device)
        held = (block < held[:, None]) & (table >= 0) & (table < pages)
        page = torch.where(held, table, pages).flatten().long()  # (pages: none)
        # by page the first entry that lets it go, or -1 where a request keeps it
        entry = torch.arange(table.numel(), device=table.device)
        goes = (finished[:, None] & held).flatten()
        first = torch.full((pages + 1,), table.numel(), device=table.device).scatter_reduce_(
            0, page, torch.where(goes, entry, -1), "amin")
        back = goes & (first[page] == entry)
        place = torch.where(back, self.n_free + back.cumsum(0) - 1, self._stack.numel() - 1)
        self._stack.scatter_(0, place, table.flatten())
        self.n_free.add_(back.sum().to(torch.int32))
        self.kv_lens.masked_fill_(finished, 0)


def rope_tables(model) -> Tuple[torch.Tensor, torch.Tensor]:
    """The model's RoPE angles as fp32 cos / sin tables on its device, made again when freqs_cis is another tensor, has been
    written to, or the model has moved."""
    dev, freqs = model.tok_embeddings.weight.device, model.freqs_cis
    version = 0 if freqs.is_inference() else freqs._version  # (inference tensors count no writes)
    made = getattr(model, "_rope_tables", None)
    if made is None or made[0] is not freqs or made[1] != version or made[2].device != dev:
        here = freqs.to(dev)
        made = model._rope_tables = (freqs, version, here.real.float().contiguous(),
                                     here.imag.float().contiguous())
    return made[2], made[3]


def forward_paged(model, tokens: torch.Tensor, step: PagedStep, cache: PagedKVCache, max_new: int,
                  whole_prompts: bool = False) -> torch.Tensor:
    """fp32 logits [requests, vocab] of each request's last token of the step (rows of requests without new tokens
    hold another token's): see Llama.forward_paged."""
    h = hidden_paged(model, tokens, step, cache, max_new, whole_prompts)
    last = (step.cu_seqlens[1:].long() - 1).clamp(0, max(tokens.shape[0] - 1, 0))
    return model._logits(model.norm(h.index_select(0, last)))


def hidden_paged(model, tokens: torch.Tensor, step: PagedStep, cache: PagedKVCache, max_new: int,
                 whole_prompts: bool = False) -> torch.Tensor:
    """The blocks' outputs [tokens, dim], before the last norm: forward_paged without its logits."""
    if tokens.dim() != 1 or tokens.shape[0] == 0:
        raise ValueError(f"forward_paged: a step has at least one token, tokens [T]; got {list(tokens.shape)}")
    cos, sin = rope_tables(model)
    bits = getattr(cache, "bits", 16)
    h = model.tok_embeddings(tokens)
    T = tokens.shape[0]
    for i, layer in enumerate(model.layers):
        att = layer.attention
        x = layer.attention_norm(h)
        q = att.wq(x).view(T, att.n_local_heads, att.head_dim)
        k = att.wk(x).view(T, att.n_local_kv_heads, att.head_dim)
        v = att.wv(x).view(T, att.n_local_kv_heads, att.head_dim)
        if bits == 4:
            q, k, v = rope_paged_write_int4(q, k, v, cos, sin, step.positions, step.slots, cache.k[i], cache.v[i], q_out=q,
                                            k_out=k if whole_prompts else None, v_out=v if whole_prompts else None,
                                            need_kv=whole_prompts)
        else:
            q, k = rope_paged_write(q, k, v, cos, sin, step.positions, step.slots, cache.k[i], cache.v[i], q_out=q,
                                    k_out=k if whole_prompts else None, need_k=whole_prompts)
        if whole_prompts:
            o = prompt_attention(q, k, v, step.cu_seqlens, max_new)
        else:
            attention = paged_attention_int4 if bits == 4 else paged_attention
            o = attention(q, cache.k[i], cache.v[i], cache.block_tables, step.kv_lens, step.cu_seqlens, max_new)
        h = h + att._reduce(att.wo(o.view(T, -1)))
        h = h + layer.feed_forward(layer.ffn_norm(h))
    return h
