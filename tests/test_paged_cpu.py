"""Arguments the paged-cache entry points refuse (no kernel is launched, no GPU needed)."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    import build  # llama-efficient-inference_b200/build.py

    build.build()
    from llama import _native

    return _native


def append(native, B=4, width=8, stride=None, capacity=16, page=16, T=4, tables=16, n_free=16):
    return native.lib().li4_paged_append(16, 16, B, tables, width if stride is None else stride, width, 16, capacity,
                                         n_free, page, T, 16, 16, 16, 16, 16, 16, None)


def test_append_refusals(native):
    for page in (0, 4, 12, 24, 2048, -16):
        assert append(native, page=page) == native.LI4_ERR_UNSUPPORTED
        assert "page_size" in native.last_error()
    assert append(native, B=-1) == native.LI4_ERR_INVALID_ARG
    assert append(native, T=-1) == native.LI4_ERR_INVALID_ARG
    assert append(native, stride=7) == native.LI4_ERR_INVALID_ARG
    assert append(native, capacity=-1) == native.LI4_ERR_INVALID_ARG
    assert append(native, B=8193) == native.LI4_ERR_UNSUPPORTED
    assert append(native, tables=None) == native.LI4_ERR_INVALID_ARG
    assert append(native, n_free=None) == native.LI4_ERR_INVALID_ARG
    assert append(native, T=(1 << 30) + 1) == native.LI4_ERR_INVALID_ARG


def rope(native, dtype=0, T=4, H=4, Hkv=2, D=64, strides=None, rope_stride=None, max_pos=8, pages=4, page=16, q=16,
         cos=16, cache=16):
    st = strides or [H * D, D, Hkv * D, D, Hkv * D, D, H * D, D, Hkv * D, D] + [page * Hkv * D, D, page * D] * 2
    return native.lib().li4_rope_paged_write(q, 16, 16, dtype, T, H, Hkv, D, (ctypes.c_int64 * 16)(*st), cos, 16,
                                             D // 2 if rope_stride is None else rope_stride, max_pos, 16, 16, 16, 16,
                                             cache, 16, pages, page, None)


def test_rope_write_refusals(native):
    assert rope(native, dtype=native.LI4_F32) == native.LI4_ERR_UNSUPPORTED
    assert rope(native, D=60) == native.LI4_ERR_UNSUPPORTED
    assert rope(native, D=264) == native.LI4_ERR_UNSUPPORTED
    assert rope(native, page=24) == native.LI4_ERR_UNSUPPORTED
    assert rope(native, T=-1) == native.LI4_ERR_INVALID_ARG
    assert rope(native, max_pos=0) == native.LI4_ERR_INVALID_ARG
    assert rope(native, q=None) == native.LI4_ERR_INVALID_ARG
    assert rope(native, cos=None) == native.LI4_ERR_INVALID_ARG
    assert rope(native, cache=None) == native.LI4_ERR_INVALID_ARG
    assert rope(native, q=8) == native.LI4_ERR_ALIGNMENT
    assert rope(native, rope_stride=30) == native.LI4_ERR_ALIGNMENT
    assert rope(native, rope_stride=28) == native.LI4_ERR_INVALID_ARG
    for i in range(16):
        st = [256, 64, 128, 64, 128, 64, 256, 64, 128, 64, 2048, 64, 1024, 2048, 64, 1024]
        st[i] += 4
        assert rope(native, strides=st) == native.LI4_ERR_ALIGNMENT
    assert rope(native, T=0) == native.LI4_OK  # nothing to do, nothing launched


def attention(native, paged, ws=1 << 40, **over):
    D, H, Hkv, page = 64, 8, 2, 16
    a = native.Attention(q=16, k=16, v=16, out=16, dtype=0, scale=0.125, stride_qt=H * D, stride_qh=D,
                         stride_ot=H * D, stride_oh=D, stride_kp=page * Hkv * D, stride_kt=Hkv * D, stride_kh=D,
                         stride_vp=page * Hkv * D, stride_vt=Hkv * D, stride_vh=D, cu_seqlens=16, n_seqs=2, n_tokens=8,
                         n_heads=H, n_kv_heads=Hkv, head_dim=D, max_queries=4, kv_lens=16, block_tables=16,
                         table_stride=8, table_width=8, num_pages=20, page_size=page)
    for name, value in over.items():
        setattr(a, name, value)
    fn = native.lib().li4_paged_attention if paged else native.lib().li4_prompt_attention
    return fn(ctypes.byref(a), 16 if ws else None, ws, None)


@pytest.mark.parametrize("paged", [False, True])
def test_attention_refusals(native, paged):
    E = native
    cases = [(dict(dtype=E.LI4_F32), E.LI4_ERR_UNSUPPORTED), (dict(head_dim=60), E.LI4_ERR_UNSUPPORTED),
             (dict(head_dim=136), E.LI4_ERR_UNSUPPORTED), (dict(n_heads=7), E.LI4_ERR_INVALID_ARG),
             (dict(n_kv_heads=0), E.LI4_ERR_INVALID_ARG), (dict(n_heads=258), E.LI4_ERR_UNSUPPORTED),
             (dict(n_seqs=-1), E.LI4_ERR_INVALID_ARG), (dict(n_tokens=-1), E.LI4_ERR_INVALID_ARG),
             (dict(max_queries=-1), E.LI4_ERR_INVALID_ARG), (dict(scale=float("nan")), E.LI4_ERR_INVALID_ARG),
             (dict(scale=float("inf")), E.LI4_ERR_INVALID_ARG), (dict(q=None), E.LI4_ERR_INVALID_ARG),
             (dict(k=None), E.LI4_ERR_INVALID_ARG), (dict(out=None), E.LI4_ERR_INVALID_ARG),
             (dict(cu_seqlens=None), E.LI4_ERR_INVALID_ARG), (dict(q=8), E.LI4_ERR_ALIGNMENT),
             (dict(out=24), E.LI4_ERR_ALIGNMENT), (dict(stride_qt=516), E.LI4_ERR_ALIGNMENT),
             (dict(stride_vh=-64), E.LI4_ERR_ALIGNMENT), (dict(n_tokens=1 << 40), E.LI4_ERR_UNSUPPORTED)]
    if paged:
        cases += [(dict(page_size=24), E.LI4_ERR_UNSUPPORTED), (dict(page_size=4), E.LI4_ERR_UNSUPPORTED),
                  (dict(kv_lens=None), E.LI4_ERR_INVALID_ARG), (dict(block_tables=None), E.LI4_ERR_INVALID_ARG),
                  (dict(table_stride=7), E.LI4_ERR_INVALID_ARG), (dict(stride_kp=1028), E.LI4_ERR_ALIGNMENT),
                  (dict(num_pages=-1), E.LI4_ERR_INVALID_ARG),
                  (dict(table_width=1 << 40, table_stride=1 << 40), E.LI4_ERR_INVALID_ARG)]
    for over, status in cases:
        assert attention(native, paged, **over) == status, over
        assert native.last_error()
    assert attention(native, paged, n_seqs=0) == E.LI4_OK
    assert attention(native, paged, n_tokens=0) == E.LI4_OK


def test_python_refuses_cpu_tensors():
    from llama import paged

    i32 = dict(dtype=torch.int32)
    lens = torch.zeros(2, **i32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_append(lens, lens, torch.zeros(2, 4, **i32), torch.zeros(8, **i32), torch.zeros(1, **i32), 16, 0)
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    cu = torch.tensor([0, 2], **i32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.prompt_attention(q, q, q, cu, 2)
    cache = torch.zeros(2, 16, 4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_attention(q, cache, cache, torch.zeros(1, 2, **i32), torch.zeros(1, **i32), cu, 2)


def test_cache_refusals():
    from llama.paged import PagedKVCache

    for kw in (dict(page_size=12), dict(page_size=4), dict(dtype=torch.float32), dict(head_dim=60),
               dict(head_dim=136)):
        args = dict(n_layers=1, num_pages=4, page_size=16, n_kv_heads=2, head_dim=64, max_requests=2, max_len=64,
                    device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            PagedKVCache(**args)


def test_release_returns_pages_to_the_stack():
    """PagedKVCache.release is index arithmetic: checked on the CPU against a list."""
    from llama.paged import PagedKVCache

    c = PagedKVCache(1, 12, 8, 1, 8, max_requests=3, max_len=64, device="cpu")
    c.block_tables[0, :3] = torch.tensor([0, 1, 2])
    c.block_tables[1, :2] = torch.tensor([3, 4])
    c.block_tables[2, :1] = torch.tensor([5])  # popped from the top: 0, 1, ...
    c.kv_lens.copy_(torch.tensor([17, 16, 1]))
    c.n_free.fill_(6)
    before = c.free_pages[:6].tolist()
    c.release(torch.tensor([True, False, True]))
    assert c.n_free.item() == 10 and c.kv_lens.tolist() == [0, 16, 0]
    assert c.free_pages[:10].tolist() == before + [0, 1, 2, 5]
    c.release(torch.tensor([True, True, True]))
    assert c.n_free.item() == 12 and sorted(c.free_pages.tolist()) == list(range(12))
