"""Arguments that the 4-bit cache's entry points, paged_fork and token_logprobs refuse, and the cache's layout (no GPU)."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    import build  # llama-efficient-inference_b200/build.py

    build.build()
    from llama import _native

    return _native


def pages(native, page=16, Hkv=2, D=64, **over):
    G = max(1, D // 32)
    p = native.Int4Pages(codes=16, params=16, stride_cp=page * Hkv * D // 2, stride_ct=D // 2, stride_ch=page * D // 2,
                         stride_pp=page * Hkv * G, stride_pt=G, stride_ph=page * G)
    for name, value in over.items():
        setattr(p, name, value)
    return p


def write(native, dtype=0, T=4, H=4, Hkv=2, D=64, strides=None, rope_stride=None, max_pos=8, n_pages=4, page=16, q=16, cos=16,
          k_out=16, cache=None):
    st = strides or [H * D, D, Hkv * D, D, Hkv * D, D, H * D, D, Hkv * D, D, Hkv * D, D]
    ck = pages(native, D=D) if cache is None else cache
    return native.lib().li4_rope_paged_write_int4(
        q, 16, 16, dtype, T, H, Hkv, D, (ctypes.c_int64 * 12)(*st), cos, 16, D // 2 if rope_stride is None else rope_stride,
        max_pos, 16, 16, 16, k_out, 16, ctypes.byref(ck), ctypes.byref(pages(native, D=D)), n_pages, page, None)


def test_write_refusals(native):
    E = native
    assert write(E, dtype=E.LI4_F32) == E.LI4_ERR_UNSUPPORTED
    for D in (0, 16, 48, 160, 256):
        assert write(E, D=D) == E.LI4_ERR_UNSUPPORTED
    for page in (0, 4, 24, 2048):
        assert write(E, page=page) == E.LI4_ERR_UNSUPPORTED
    assert write(E, T=-1) == E.LI4_ERR_INVALID_ARG
    assert write(E, T=(1 << 30) + 1) == E.LI4_ERR_INVALID_ARG
    assert write(E, Hkv=1 << 62) == E.LI4_ERR_INVALID_ARG
    assert write(E, n_pages=1 << 31) == E.LI4_ERR_INVALID_ARG
    assert write(E, max_pos=0) == E.LI4_ERR_INVALID_ARG
    assert write(E, q=None) == E.LI4_ERR_INVALID_ARG
    assert write(E, cos=None) == E.LI4_ERR_INVALID_ARG
    assert write(E, cache=pages(E, codes=None)) == E.LI4_ERR_INVALID_ARG
    assert write(E, cache=pages(E, params=None)) == E.LI4_ERR_INVALID_ARG
    assert write(E, q=8) == E.LI4_ERR_ALIGNMENT
    assert write(E, k_out=8) == E.LI4_ERR_ALIGNMENT
    assert write(E, cache=pages(E, codes=8)) == E.LI4_ERR_ALIGNMENT
    assert write(E, cache=pages(E, params=18)) == E.LI4_ERR_ALIGNMENT
    assert write(E, cache=pages(E, stride_ct=40)) == E.LI4_ERR_ALIGNMENT
    assert write(E, rope_stride=28) == E.LI4_ERR_INVALID_ARG
    for i in range(12):
        st = [256, 64, 128, 64, 128, 64, 256, 64, 128, 64, 128, 64]
        st[i] += 4
        assert write(E, strides=st) == E.LI4_ERR_ALIGNMENT
    assert write(E, T=0) == E.LI4_OK


def attention(native, ws=1 << 40, k=True, cache=None, **over):
    D, H, Hkv, page = 64, 8, 2, 16
    a = native.Attention(q=16, k=None, v=None, out=16, dtype=0, scale=0.125, stride_qt=H * D, stride_qh=D, stride_ot=H * D,
                         stride_oh=D, cu_seqlens=16, n_seqs=2, n_tokens=8, n_heads=H, n_kv_heads=Hkv, head_dim=D,
                         max_queries=4, kv_lens=16, block_tables=16, table_stride=8, table_width=8, num_pages=20,
                         page_size=page)
    for name, value in over.items():
        setattr(a, name, value)
    ck = pages(native) if cache is None else cache
    return native.lib().li4_paged_attention_int4(ctypes.byref(a), ctypes.byref(ck) if k else None,
                                                 ctypes.byref(pages(native)), 16 if ws else None, ws, None)


def test_attention_refusals(native):
    E = native
    for over, status in [(dict(dtype=E.LI4_F32), E.LI4_ERR_UNSUPPORTED), (dict(head_dim=48), E.LI4_ERR_UNSUPPORTED),
                         (dict(head_dim=160), E.LI4_ERR_UNSUPPORTED), (dict(n_heads=7), E.LI4_ERR_INVALID_ARG),
                         (dict(n_heads=258), E.LI4_ERR_UNSUPPORTED), (dict(scale=float("nan")), E.LI4_ERR_INVALID_ARG),
                         (dict(q=None), E.LI4_ERR_INVALID_ARG), (dict(q=8), E.LI4_ERR_ALIGNMENT), (dict(k=False), E.LI4_ERR_INVALID_ARG),
                         (dict(cache=pages(E, codes=None)), E.LI4_ERR_INVALID_ARG), (dict(cache=pages(E, codes=8)), E.LI4_ERR_ALIGNMENT),
                         (dict(cache=pages(E, stride_ch=8)), E.LI4_ERR_ALIGNMENT), (dict(cache=pages(E, params=2)), E.LI4_ERR_ALIGNMENT),
                         (dict(page_size=24), E.LI4_ERR_UNSUPPORTED), (dict(kv_lens=None), E.LI4_ERR_INVALID_ARG),
                         (dict(block_tables=None), E.LI4_ERR_INVALID_ARG), (dict(table_stride=7), E.LI4_ERR_INVALID_ARG),
                         (dict(num_pages=-1), E.LI4_ERR_INVALID_ARG), (dict(n_tokens=1 << 40), E.LI4_ERR_UNSUPPORTED)]:
        assert attention(E, **over) == status, over
        assert native.last_error()
    assert attention(E, n_seqs=0) == E.LI4_OK
    assert attention(E, n_tokens=0) == E.LI4_OK


def fork(native, B=4, width=8, stride=None, capacity=16, page=16, tables=16, n_free=16, pool=16, step=4096, size=2048, n_pools=1,
         ws=1 << 40, parents=16):
    P, I = ctypes.c_void_p * 1, ctypes.c_int64 * 1
    return native.lib().li4_paged_fork(16, parents, B, tables, width if stride is None else stride, width, 16, capacity, n_free,
                                       page, 16, 16, 16, P(pool), I(step), I(size), n_pools, 16 if ws else None, ws, None)


def test_fork_refusals(native):
    E = native
    for page in (0, 4, 12, 2048):
        assert fork(E, page=page) == E.LI4_ERR_UNSUPPORTED
    assert fork(E, B=-1) == E.LI4_ERR_INVALID_ARG
    assert fork(E, stride=7) == E.LI4_ERR_INVALID_ARG
    assert fork(E, capacity=-1) == E.LI4_ERR_INVALID_ARG
    assert fork(E, B=8193) == E.LI4_ERR_UNSUPPORTED
    assert fork(E, B=8192, width=1 << 19) == E.LI4_ERR_UNSUPPORTED
    assert fork(E, tables=None) == E.LI4_ERR_INVALID_ARG
    assert fork(E, parents=None) == E.LI4_ERR_INVALID_ARG
    assert fork(E, n_free=None) == E.LI4_ERR_INVALID_ARG
    assert fork(E, pool=None) == E.LI4_ERR_ALIGNMENT
    assert fork(E, pool=8) == E.LI4_ERR_ALIGNMENT
    assert fork(E, size=2040) == E.LI4_ERR_ALIGNMENT
    assert fork(E, step=4104) == E.LI4_ERR_ALIGNMENT
    assert fork(E, step=1024) == E.LI4_ERR_INVALID_ARG
    assert fork(E, size=-16) == E.LI4_ERR_INVALID_ARG
    assert fork(E, ws=64) == E.LI4_ERR_WORKSPACE
    assert fork(E, ws=0) == E.LI4_ERR_WORKSPACE
    assert native.lib().li4_paged_fork_workspace_bytes(4, 8, 16) > 0
    for bad in ((0, 8, 16), (8193, 8, 16), (4, -1, 16), (4, 8, -1), (8192, 1 << 40, 1)):
        assert native.lib().li4_paged_fork_workspace_bytes(*bad) == 0


def logprobs(native, dtype=2, rows=2, cols=50, stride=50, top=4, logits=16, tokens=16, out=16, ids=16):
    return native.lib().li4_token_logprobs(logits, dtype, rows, cols, stride, tokens, top, out, 16, ids, 16, None)


def test_logprobs_refusals(native):
    E = native
    assert logprobs(E, dtype=3) == E.LI4_ERR_UNSUPPORTED
    for bad in (dict(rows=-1), dict(cols=0), dict(cols=(1 << 30) + 1), dict(stride=49), dict(logits=None), dict(tokens=None),
                dict(out=None), dict(ids=None), dict(rows=1 << 40)):
        assert logprobs(E, **bad) == E.LI4_ERR_INVALID_ARG, bad
    for bad in (dict(top=33), dict(top=-1), dict(cols=3)):
        assert logprobs(E, **bad) == E.LI4_ERR_UNSUPPORTED, bad
    assert logprobs(E, logits=18) == E.LI4_ERR_ALIGNMENT
    assert logprobs(E, dtype=0, logits=17) == E.LI4_ERR_ALIGNMENT
    assert logprobs(E, rows=0) == E.LI4_OK


def test_codes_round_trip():
    from llama import paged

    c = torch.randint(0, 16, (3, 5, 96), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    packed = paged.pack_codes(c)
    assert packed.dtype == torch.uint8 and packed.shape == (3, 5, 48)
    assert torch.equal(paged.unpack_codes(packed), c)
    word = packed.view(torch.int32)[0, 0, 1].item() & 0xFFFFFFFF  # dims 8 .. 15
    for i in range(4):
        assert word >> 4 * i & 15 == c[0, 0, 8 + 2 * i] and word >> 16 + 4 * i & 15 == c[0, 0, 8 + 2 * i + 1]
    p = paged.Int4Pages(packed.view(1, 3, 5, 48), torch.tensor([0.5, -1.0]).half().expand(1, 3, 5, 3, 2))
    assert torch.equal(p.values(), (c.double() * 0.5 - 1).half().view(1, 3, 5, 96))


def test_cache_of_four_bits():
    from llama.paged import PagedKVCache

    c = PagedKVCache(2, 12, 8, 2, 64, max_requests=3, max_len=64, device="cpu", bits=4)
    assert c.k[0].codes.shape == (12, 8, 2, 32) and c.v[1].params.shape == (12, 8, 2, 2, 2) and len(c.pools) == 8
    for kw in (dict(bits=8), dict(bits=4, head_dim=48)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_layers=1, num_pages=4, page_size=16, n_kv_heads=2, head_dim=64, max_requests=2, max_len=64,
                                   device="cpu"), **kw})


def test_python_refuses_cpu_tensors():
    from llama import logprobs, paged

    i32 = dict(dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    cache = paged.Int4Pages(torch.zeros(2, 16, 4, 32, dtype=torch.uint8), torch.zeros(2, 16, 4, 2, 2, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_attention_int4(q, cache, cache, torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.tensor([0, 2], **i32), 2)
    lens = torch.zeros(2, **i32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_fork(lens, torch.zeros(2, 4, **i32), torch.zeros(8, **i32), torch.zeros(1, **i32), lens, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        logprobs.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long), 2)
