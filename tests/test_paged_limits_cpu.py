"""Arguments that the paged-cache entry points refuse on the host (no kernel is launched, no GPU needed)."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    import build  # llama-efficient-inference_b200/build.py

    build.build()
    from llama import _native

    return _native


def test_append_refuses_a_negative_limit(native):
    def append(max_len, page=16):
        return native.lib().li4_paged_append_within(16, 16, 4, 16, 8, 8, 16, 16, 16, page, 4, max_len, 16, 16, 16, 16,
                                                    16, 16, None)

    assert append(-1) == native.LI4_ERR_INVALID_ARG and "max_len" in native.last_error()
    assert append(10, page=12) == native.LI4_ERR_UNSUPPORTED


def calls(paged, q, k, cache):
    """Every entry point on float tensors, as (name of a tensor, call with that tensor replaced)."""
    i32 = dict(dtype=torch.int32, device=q.device)
    cu, lens, tables = torch.tensor([0, 4], **i32), torch.tensor([4], **i32), torch.zeros(1, 2, **i32)
    cos, pos = torch.zeros(8, 32, device=q.device), torch.zeros(4, **i32)
    slots = torch.zeros(4, dtype=torch.long, device=q.device)
    a = dict(q=q, k=k, v=k.detach().clone(), cache_k=cache, cache_v=cache.detach().clone(), cos=cos, sin=cos.clone())

    def prompt(**x):
        x = {**a, **x}
        return paged.prompt_attention(x["q"], x["k"], x["v"], cu, 4, out=x.get("out"))

    def over_cache(**x):
        x = {**a, **x}
        return paged.paged_attention(x["q"], x["cache_k"], x["cache_v"], tables, lens, cu, 4, out=x.get("out"))

    def rope(**x):
        x = {**a, **x}
        return paged.rope_paged_write(x["q"], x["k"], x["v"], x["cos"], x["sin"], pos, slots, x["cache_k"], x["cache_v"],
                                      q_out=x.get("q_out"), k_out=x.get("k_out"))

    return a, {prompt: ("q", "k", "v"), over_cache: ("q", "cache_k", "cache_v"),
               rope: ("q", "k", "v", "cos", "sin", "cache_k", "cache_v")}


def test_tensors_that_require_grad_are_refused(native):
    """There is no backward pass: a result without a graph would lose the gradient silently."""
    from llama import paged

    q, k = torch.zeros(4, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    a, table = calls(paged, q, k, torch.zeros(2, 16, 2, 64, dtype=torch.float16))
    for call, names in table.items():
        for name in names:
            leaf = a[name].clone().requires_grad_()
            with pytest.raises(RuntimeError, match=f"{name} requires grad"):
                call(**{name: leaf})
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
                call(**{name: leaf})


def test_fake_tensors_and_tracing_are_refused(native):
    """The functions are no registered operators: a tracer would record their outputs as constants."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from llama import paged

    with FakeTensorMode():
        q, k = torch.zeros(4, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
        _, table = calls(paged, q, k, torch.zeros(2, 16, 2, 64, dtype=torch.float16))
        for call in table:
            with pytest.raises(RuntimeError, match="plain tensor"):
                call()
        i32 = dict(dtype=torch.int32)
        with pytest.raises(RuntimeError, match="plain tensor"):
            paged.paged_append(torch.zeros(2, **i32), torch.zeros(2, **i32), torch.zeros(2, 4, **i32),
                               torch.zeros(8, **i32), torch.zeros(1, **i32), 16, 0)
    q, k = torch.zeros(4, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="plain tensor"):
        torch.jit.trace(lambda x: paged.prompt_attention(x, k, k, cu, 4), (q,))


def test_rope_tables_follow_the_model(native):
    """A freqs_cis that is replaced or written to is seen; one that is not is not turned into tables again."""
    from llama.model import Llama, ModelArgs
    from llama.paged import rope_tables

    model = Llama(ModelArgs(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, vocab_size=16, multiple_of=32, max_batch_size=1,
                            max_seq_len=8))
    cos, sin = rope_tables(model)
    assert torch.equal(cos, model.freqs_cis.real.float()) and torch.equal(sin, model.freqs_cis.imag.float())
    assert rope_tables(model)[0] is cos
    model.freqs_cis = model.freqs_cis.conj().resolve_conj().clone()
    assert torch.equal(rope_tables(model)[1], -sin)
    model.freqs_cis.mul_(2)
    assert torch.equal(rope_tables(model)[0], 2 * cos)
    with torch.inference_mode():
        model.freqs_cis = model.freqs_cis.clone()
    assert torch.equal(rope_tables(model)[0], 2 * cos)


def attention_args(native, **over):
    D, H, Hkv, page = 64, 8, 2, 16
    a = native.Attention(q=16, k=16, v=16, out=16, dtype=0, scale=0.125, stride_qt=H * D, stride_qh=D,
                         stride_ot=H * D, stride_oh=D, stride_kp=page * Hkv * D, stride_kt=Hkv * D, stride_kh=D,
                         stride_vp=page * Hkv * D, stride_vt=Hkv * D, stride_vh=D, cu_seqlens=16, n_seqs=2, n_tokens=8,
                         n_heads=H, n_kv_heads=Hkv, head_dim=D, max_queries=4, kv_lens=16, block_tables=16,
                         table_stride=8, table_width=8, num_pages=20, page_size=page)
    for name, value in over.items():
        setattr(a, name, value)
    return a


def test_tables_whose_width_passes_64_bits_are_refused(native):
    for width in (1 << 59, 1 << 60, (1 << 63) - 1):
        a = attention_args(native, table_width=width, table_stride=width)
        assert native.lib().li4_paged_attention(ctypes.byref(a), 16, 1 << 40, None) == native.LI4_ERR_INVALID_ARG
