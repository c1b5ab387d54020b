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

The lengths live on the GPU: no call reads them on the host, so a step can be captured in a CUDA graph
and replayed while the requests grow.  PagedKVCache holds the pool, Llama.forward_paged runs the model's
blocks over it, Generation.generate_paged is the loop around them.

Every function runs on the current stream of its tensors' device, allocates its outputs (unless they are
given) and its workspace there, and raises RuntimeError subclasses for arguments it does not take.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, NamedTuple, Optional, Tuple

import torch

from . import _native as native

_CODES = {torch.float16: native.LI4_F16, torch.bfloat16: native.LI4_BF16}


class PagedStep(NamedTuple):
    """What paged_append works out for one step (all on the GPU)."""

    cu_seqlens: torch.Tensor  # int32 [requests + 1]: first packed token of each request
    positions: torch.Tensor   # int32 [tokens]
    slots: torch.Tensor       # int64 [tokens]: page * page_size + row; -1: refused or past the last request
    kv_lens: torch.Tensor     # int32 [requests], the step's tokens included
    n_free: torch.Tensor      # int32 [1]
    granted: torch.Tensor     # bool [requests]


def _fail(what: str, message: str):
    raise RuntimeError(f"{what}: {message}")


def _same_device(what: str, **tensors) -> torch.device:
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            _fail(what, f"{name} is on {t.device} (CUDA tensors only)")
        if dev is None:
            dev, first = t.device, name
        elif t.device != dev:
            _fail(what, f"{name} is on {t.device}, {first} is on {dev}")
    return dev


def _int_tensor(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
    if t.dtype != dtype or tuple(t.shape) != shape:
        _fail(what, f"{name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t


def _strides(t: torch.Tensor, dims: int) -> List[int]:
    """Strides of the first `dims` dimensions; a dimension of one element has none."""
    return [t.stride(i) if t.shape[i] > 1 else 0 for i in range(dims)]


def _rows_ok(t: torch.Tensor) -> bool:
    """The kernels' layout: contiguous last dimension, rows on 16-byte boundaries, no repeated rows."""
    if t.numel() == 0:
        return True
    return (t.shape[-1] == 1 or t.stride(-1) == 1) and t.data_ptr() % 16 == 0 and \
        all(t.shape[i] == 1 or (t.stride(i) > 0 and t.stride(i) % 8 == 0) for i in range(t.dim() - 1))


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t itself, or a contiguous copy where its layout is not the kernels'."""
    return t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def _packed(what: str, name: str, t: torch.Tensor, dtype=None) -> None:
    if t.dim() != 3:
        _fail(what, f"{name} must be [tokens, heads, head_dim], got {list(t.shape)}")
    if t.dtype not in _CODES:
        _fail(what, f"{name} must be float16 or bfloat16, got {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        _fail(what, f"{name} is {t.dtype}, q is {dtype}")


def _output(what: str, name: str, t: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    if t is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device or not _rows_ok(t):
        _fail(what, f"{name} must be {like.dtype} {list(like.shape)} on {like.device} with contiguous rows on "
                    "16-byte boundaries")
    return t


def _cache(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, kv_heads: int, head_dim: int) -> None:
    if t.dim() != 4 or t.shape[2] != kv_heads or t.shape[3] != head_dim or t.dtype != dtype:
        _fail(what, f"{name} must be {dtype} [pages, page_size, {kv_heads}, {head_dim}], got {t.dtype} "
                    f"{list(t.shape)}")
    if not _rows_ok(t):
        _fail(what, f"{name}: rows of head_dim values must be contiguous, on 16-byte boundaries")


class _on:
    """The tensors' device as the current one for the launch (nothing to do when it already is)."""

    def __init__(self, device: torch.device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def paged_append(kv_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
                 n_free: torch.Tensor, page_size: int, num_tokens: int, kv_lens_out: Optional[torch.Tensor] = None,
                 n_free_out: Optional[torch.Tensor] = None) -> PagedStep:
    """One step's bookkeeping (li4_paged_append): request b holds kv_lens[b] tokens and appends new_lens[b].

    kv_lens, new_lens int32 [requests]; block_tables int32 [requests, blocks], the entries of the step's fresh
    pages are written; free_pages int32 [capacity] with the free ones in free_pages[:n_free], taken from the top;
    n_free int32 [1]; num_tokens = sum(new_lens), which the host knows.  kv_lens_out / n_free_out may be kv_lens /
    n_free (in place); by default they are new tensors.  A request that does not fit (table too narrow, too few
    pages for it and those before it) is refused whole: granted False, length kept, slots -1."""
    what = "paged_append"
    dev = _same_device(what, kv_lens=kv_lens, new_lens=new_lens, block_tables=block_tables, free_pages=free_pages,
                       n_free=n_free, kv_lens_out=kv_lens_out, n_free_out=n_free_out)
    i32 = torch.int32
    if kv_lens.dim() != 1 or block_tables.dim() != 2 or free_pages.dim() != 1:
        _fail(what, "kv_lens [requests], block_tables [requests, blocks] and free_pages [pages] expected")
    B, width = kv_lens.shape[0], block_tables.shape[1]
    _int_tensor(what, "kv_lens", kv_lens, i32, (B,))
    _int_tensor(what, "new_lens", new_lens, i32, (B,))
    _int_tensor(what, "block_tables", block_tables, i32, (B, width))
    _int_tensor(what, "free_pages", free_pages, i32, (free_pages.shape[0],))
    _int_tensor(what, "n_free", n_free, i32, (1,))
    if width > 1 and block_tables.stride(1) != 1 or B > 1 and block_tables.stride(0) < width:
        _fail(what, "block_tables rows must be contiguous")
    kv_lens, new_lens, free_pages = kv_lens.contiguous(), new_lens.contiguous(), free_pages.contiguous()
    for name, t, like in (("kv_lens_out", kv_lens_out, kv_lens), ("n_free_out", n_free_out, n_free)):
        if t is not None and (t.dtype != i32 or t.shape != like.shape or not t.is_contiguous()):
            _fail(what, f"{name} must be contiguous int32 {list(like.shape)}")
    with _on(dev):
        opt = dict(dtype=i32, device=dev)
        cu = torch.empty(B + 1, **opt)
        positions = torch.empty(num_tokens, **opt)
        slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
        kv_out = torch.empty_like(kv_lens) if kv_lens_out is None else kv_lens_out
        free_out = torch.empty_like(n_free) if n_free_out is None else n_free_out
        granted = torch.empty(B, dtype=torch.bool, device=dev)
        rc = native.lib().li4_paged_append(kv_lens.data_ptr(), new_lens.data_ptr(), B, block_tables.data_ptr(),
                                           block_tables.stride(0) if B > 1 else width, width, free_pages.data_ptr(),
                                           free_pages.shape[0], n_free.data_ptr(), page_size, num_tokens,
                                           cu.data_ptr(), positions.data_ptr(), slots.data_ptr(), kv_out.data_ptr(),
                                           free_out.data_ptr(), granted.data_ptr(), native.stream_ptr(dev))
        native.check(rc, what)
    return PagedStep(cu, positions, slots, kv_out, free_out, granted)


def rope_paged_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                     positions: torch.Tensor, slots: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                     q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                     need_k: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RoPE on packed q [T, heads, d] and k [T, kv_heads, d] and the cache write of k and v (li4_rope_paged_write).

    Pairs (2i, 2i + 1) turn by the angle in row positions[t] of cos / sin (fp32 [positions, d / 2]), in fp32.  The
    turned key and the value of token t go to row slots[t] % page_size of page slots[t] // page_size of cache_k /
    cache_v [pages, page_size, kv_heads, d] (any strides with contiguous rows); negative slots are skipped.
    Returns (turned q, turned k); q_out / k_out may be q / k themselves.  need_k = False leaves the packed turned
    keys out (returns None for them): attention over the cache does not read them."""
    what = "rope_paged_write"
    dev = _same_device(what, q=q, k=k, v=v, cos=cos, sin=sin, positions=positions, slots=slots, cache_k=cache_k,
                       cache_v=cache_v, q_out=q_out, k_out=k_out)
    _packed(what, "q", q)
    _packed(what, "k", k, q.dtype)
    _packed(what, "v", v, q.dtype)
    T, H, D = q.shape
    Hkv = k.shape[1]
    if tuple(k.shape) != (T, Hkv, D) or v.shape != k.shape:
        _fail(what, f"q {list(q.shape)}, k {list(k.shape)} and v {list(v.shape)} do not match")
    _cache(what, "cache_k", cache_k, q.dtype, Hkv, D)
    _cache(what, "cache_v", cache_v, q.dtype, Hkv, D)
    if cache_v.shape != cache_k.shape:
        _fail(what, f"cache_k {list(cache_k.shape)} and cache_v {list(cache_v.shape)} differ")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != D // 2 or cos.dtype != torch.float32 or \
            sin.dtype != torch.float32:
        _fail(what, f"cos / sin must be float32 [positions, {D // 2}], got {list(cos.shape)} / {list(sin.shape)}")
    if not cos.is_contiguous() or cos.data_ptr() % 16 or D % 8:
        cos = cos.clone(memory_format=torch.contiguous_format)
    if not sin.is_contiguous() or sin.data_ptr() % 16:
        sin = sin.clone(memory_format=torch.contiguous_format)
    _int_tensor(what, "positions", positions, torch.int32, (T,))
    _int_tensor(what, "slots", slots, torch.int64, (T,))
    positions, slots = positions.contiguous(), slots.contiguous()
    with _on(dev):
        q_out = _output(what, "q_out", q_out, q)
        k_out = _output(what, "k_out", k_out, k) if need_k or k_out is not None else None
        qr, kr, vr = _readable(q), _readable(k), _readable(v)
        st = _strides(qr, 2) + _strides(kr, 2) + _strides(vr, 2) + _strides(q_out, 2) + \
            (_strides(k_out, 2) if k_out is not None else [0, 0]) + _strides(cache_k, 3) + _strides(cache_v, 3)
        rc = native.lib().li4_rope_paged_write(
            qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), _CODES[q.dtype], T, H, Hkv, D,
            (ctypes.c_int64 * 16)(*st), cos.data_ptr(), sin.data_ptr(), D // 2, cos.shape[0], positions.data_ptr(),
            slots.data_ptr(), q_out.data_ptr(), k_out.data_ptr() if k_out is not None else None, cache_k.data_ptr(),
            cache_v.data_ptr(), cache_k.shape[0], cache_k.shape[1], native.stream_ptr(dev))
        native.check(rc, what)
    return q_out, k_out


def _attention_args(what, q, out, cu_seqlens, max_queries, scale) -> native.Attention:
    a = native.Attention()
    a.q, a.out, a.dtype = q.data_ptr(), out.data_ptr(), _CODES[q.dtype]
    a.n_tokens, a.n_heads, a.head_dim = q.shape
    a.scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    a.stride_qt, a.stride_qh = _strides(q, 2)
    a.stride_ot, a.stride_oh = _strides(out, 2)
    a.cu_seqlens, a.n_seqs, a.max_queries = cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1, max_queries
    return a


def _launch(what, fn, a: native.Attention, dev: torch.device) -> None:
    # The workspace comes from the stream's allocator for this call alone: calls on several streams and captured
    # graphs (each with its own pool) never share one.
    nbytes = native.lib().li4_attention_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    native.check(fn(ctypes.byref(a), ws.data_ptr() if nbytes else None, nbytes, native.stream_ptr(dev)), what)


def _check_queries(what: str, q: torch.Tensor, cu_seqlens: torch.Tensor, kv_heads: int, max_queries: int) -> None:
    _packed(what, "q", q)
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or cu_seqlens.dtype != torch.int32:
        _fail(what, f"cu_seqlens must be int32 [sequences + 1], got {cu_seqlens.dtype} {list(cu_seqlens.shape)}")
    if kv_heads < 1 or q.shape[1] < 1 or q.shape[1] % kv_heads:
        _fail(what, f"{q.shape[1]} query heads over {kv_heads} KV heads")
    if max_queries < 0:
        _fail(what, f"a longest sequence of {max_queries} queries")


def _check_out(what: str, out: torch.Tensor, q: torch.Tensor) -> None:
    if out.numel() and out.data_ptr() == q.data_ptr():
        _fail(what, "out must not be q: rows are read again after others are written")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_len: int,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of whole prompts packed one after another (li4_prompt_attention).

    q [T, heads, d], k and v [T, kv_heads, d] in float16 or bfloat16 (d a multiple of 8 up to 128, heads a
    multiple of kv_heads); cu_seqlens int32 [prompts + 1] on the GPU: prompt b is rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1; max_len: the longest prompt, known to the host (it picks the kernel; a wrong value costs
    time, not correctness).  Softmax of scale q k^T (default 1 / sqrt(d)) in fp32.  Rows past the last prompt are
    left as they were in `out`.  out must not overlap q, k or v."""
    what = "prompt_attention"
    dev = _same_device(what, q=q, k=k, v=v, cu_seqlens=cu_seqlens, out=out)
    _packed(what, "k", k, q.dtype)
    _packed(what, "v", v, q.dtype)
    _check_queries(what, q, cu_seqlens, k.shape[1], max_len)
    if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or v.shape != k.shape:
        _fail(what, f"q {list(q.shape)}, k {list(k.shape)} and v {list(v.shape)} do not match")
    with _on(dev):
        out = _output(what, "out", out, q)
        _check_out(what, out, q)
        qr, kr, vr, cu = _readable(q), _readable(k), _readable(v), cu_seqlens.contiguous()
        a = _attention_args(what, qr, out, cu, max_len, scale)
        a.k, a.v, a.n_kv_heads = kr.data_ptr(), vr.data_ptr(), kr.shape[1]
        a.stride_kt, a.stride_kh = _strides(kr, 2)
        a.stride_vt, a.stride_vh = _strides(vr, 2)
        _launch(what, native.lib().li4_prompt_attention, a, dev)
    return out


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
    what = "paged_attention"
    dev = _same_device(what, q=q, cache_k=cache_k, cache_v=cache_v, block_tables=block_tables, kv_lens=kv_lens,
                       cu_seqlens=cu_seqlens, out=out)
    if cache_k.dim() != 4:
        _fail(what, f"cache_k must be [pages, page_size, kv_heads, head_dim], got {list(cache_k.shape)}")
    _check_queries(what, q, cu_seqlens, cache_k.shape[2], max_new)
    _cache(what, "cache_k", cache_k, q.dtype, cache_k.shape[2], q.shape[2])
    _cache(what, "cache_v", cache_v, q.dtype, cache_k.shape[2], q.shape[2])
    if cache_v.shape != cache_k.shape:
        _fail(what, f"cache_k {list(cache_k.shape)} and cache_v {list(cache_v.shape)} differ")
    B = cu_seqlens.shape[0] - 1
    if block_tables.dim() != 2:
        _fail(what, f"block_tables must be [requests, blocks], got {list(block_tables.shape)}")
    _int_tensor(what, "block_tables", block_tables, torch.int32, (B, block_tables.shape[1]))
    _int_tensor(what, "kv_lens", kv_lens, torch.int32, (B,))
    with _on(dev):
        out = _output(what, "out", out, q)
        _check_out(what, out, q)
        width = block_tables.shape[1]
        if width > 1 and block_tables.stride(1) != 1 or B > 1 and block_tables.stride(0) < width:
            block_tables = block_tables.contiguous()
        qr, cu, lens = _readable(q), cu_seqlens.contiguous(), kv_lens.contiguous()
        a = _attention_args(what, qr, out, cu, max_new, scale)
        a.k, a.v, a.n_kv_heads = cache_k.data_ptr(), cache_v.data_ptr(), cache_k.shape[2]
        a.stride_kp, a.stride_kt, a.stride_kh = _strides(cache_k, 3)
        a.stride_vp, a.stride_vt, a.stride_vh = _strides(cache_v, 3)
        a.kv_lens, a.block_tables = lens.data_ptr(), block_tables.data_ptr()
        a.table_stride, a.table_width = (block_tables.stride(0) if B > 1 else width), width
        a.num_pages, a.page_size = cache_k.shape[0], cache_k.shape[1]
        _launch(what, native.lib().li4_paged_attention, a, dev)
    return out


class PagedKVCache:
    """Pages, block tables and lengths of up to max_requests requests of up to max_len tokens each.

    k[i] / v[i] are layer i's pages [num_pages, page_size, kv_heads, head_dim]; each (page, head) is contiguous in
    memory, so the rows a KV head reads of a page are one run.  Request r is row r of block_tables and kv_lens for as
    long as it lives; release() returns its pages."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 max_requests: int, max_len: int, dtype: torch.dtype = torch.float16, device="cuda"):
        if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size}: a power of two from 8 to 1024")
        if dtype not in _CODES:
            raise ValueError(f"cache dtype {dtype}: float16 or bfloat16")
        if head_dim % 8 or not 8 <= head_dim <= 128:
            raise ValueError(f"head_dim {head_dim}: a multiple of 8 up to 128")
        self.page_size, self.max_len = page_size, max_len
        shape = (n_layers, num_pages, n_kv_heads, page_size, head_dim)
        self.k = [t.transpose(1, 2) for t in torch.zeros(shape, dtype=dtype, device=device)]
        self.v = [t.transpose(1, 2) for t in torch.zeros(shape, dtype=dtype, device=device)]
        i32 = dict(dtype=torch.int32, device=device)
        self.block_tables = torch.zeros(max_requests, -(-max_len // page_size), **i32)
        self.kv_lens = torch.zeros(max_requests, **i32)
        # one entry more than pages: release() drops what it does not return there
        self._stack = torch.cat([torch.arange(num_pages - 1, -1, -1, **i32), torch.zeros(1, **i32)])
        self.free_pages = self._stack[:num_pages]
        self.n_free = torch.full((1,), num_pages, **i32)

    def append(self, new_lens: torch.Tensor, num_tokens: int) -> PagedStep:
        """Takes pages for new_lens[r] more tokens of every request r (int32 [max_requests], zeros for idle rows);
        num_tokens is their sum.  Updates the cache's lengths, tables and free pages in place."""
        return paged_append(self.kv_lens, new_lens, self.block_tables, self.free_pages, self.n_free, self.page_size,
                            num_tokens, kv_lens_out=self.kv_lens, n_free_out=self.n_free)

    def release(self, finished: torch.Tensor) -> None:
        """Returns the pages of the requests flagged in finished (bool [max_requests]) and sets their lengths to 0.
        No host synchronisation."""
        held = torch.div(self.kv_lens + (self.page_size - 1), self.page_size, rounding_mode="floor")
        block = torch.arange(self.block_tables.shape[1], device=self.kv_lens.device)
        back = (finished[:, None] & (block < held[:, None])).flatten()
        place = torch.where(back, self.n_free + back.cumsum(0) - 1, self._stack.numel() - 1)
        self._stack.scatter_(0, place, self.block_tables.flatten())
        self.n_free.add_(back.sum().to(torch.int32))
        self.kv_lens.masked_fill_(finished, 0)


def rope_tables(model) -> Tuple[torch.Tensor, torch.Tensor]:
    """The model's RoPE angles as fp32 cos / sin tables on its device (made once)."""
    dev = model.tok_embeddings.weight.device
    tables = getattr(model, "_rope_tables", None)
    if tables is None or tables[0].device != dev:
        freqs = model.freqs_cis.to(dev)
        tables = model._rope_tables = (freqs.real.float().contiguous(), freqs.imag.float().contiguous())
    return tables


def forward_paged(model, tokens: torch.Tensor, step: PagedStep, cache: PagedKVCache, max_new: int,
                  whole_prompts: bool = False) -> torch.Tensor:
    """fp32 logits [requests, vocab] of each request's last token of the step (rows of requests without new tokens
    hold another token's): see Llama.forward_paged."""
    cos, sin = rope_tables(model)
    h = model.tok_embeddings(tokens)
    T = tokens.shape[0]
    for i, layer in enumerate(model.layers):
        att = layer.attention
        x = layer.attention_norm(h)
        q = att.wq(x).view(T, att.n_local_heads, att.head_dim)
        k = att.wk(x).view(T, att.n_local_kv_heads, att.head_dim)
        v = att.wv(x).view(T, att.n_local_kv_heads, att.head_dim)
        q, k = rope_paged_write(q, k, v, cos, sin, step.positions, step.slots, cache.k[i], cache.v[i], q_out=q,
                                k_out=k if whole_prompts else None, need_k=whole_prompts)
        if whole_prompts:
            o = prompt_attention(q, k, v, step.cu_seqlens, max_new)
        else:
            o = paged_attention(q, cache.k[i], cache.v[i], cache.block_tables, step.kv_lens, step.cu_seqlens, max_new)
        h = h + att._reduce(att.wo(o.view(T, -1)))
        h = h + layer.feed_forward(layer.ffn_norm(h))
    last = (step.cu_seqlens[1:].long() - 1).clamp(0, max(T - 1, 0))
    return model._logits(model.norm(h.index_select(0, last)))
