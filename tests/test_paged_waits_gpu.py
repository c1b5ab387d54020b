"""The bounded waits of the tensor-memory attention kernel run out without a fault, report it and leave the GPU usable."""
import pytest
import torch

from test_paged_gpu import check, cumulative, i32, make_cache, paged, rand  # noqa: F401 (paged: the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture()
def native(paged):  # noqa: F811
    from llama import _native

    _native.device_errors()
    yield _native
    _native.check(_native.lib().li4_debug_set_attention_wait_limit(0), "debug_set_attention_wait_limit")
    _native.device_errors()


@pytest.mark.parametrize("polls", [1, 2, 3, 20, 100, 400])
@pytest.mark.parametrize("d", [64, 128])
def test_waits_that_run_out_set_bit_8_and_nothing_else(paged, native, d, polls):  # noqa: F811
    """No copy lands within a few polls: the call ends by itself, reports bit 8 where a wait ran out, writes nothing past
    its rows, and the next call with the default limit is right."""
    dtype, H, Hkv, lens = torch.float16, 8, 2, [300, 1100, 64]
    T = sum(lens)
    q, k, v = rand((T + 5, H, d), dtype, 1), rand((T + 5, Hkv, d), dtype, 2), rand((T + 5, Hkv, d), dtype, 3)
    cu = i32(cumulative(lens))
    want = paged.prompt_attention(q, k, v, cu, max(lens))
    native.check(native.lib().li4_debug_set_attention_wait_limit(polls), "debug_set_attention_wait_limit")
    out = torch.full((T + 5, H, d), 7.0, dtype=dtype, device="cuda")
    for _ in range(3):
        paged.prompt_attention(q, k, v, cu, max(lens), out=out)
    torch.cuda.synchronize()
    flags = native.device_errors()
    assert flags in (0, 256) and (flags == 256 or polls > 3)
    assert bool((out[T:] == 7).all())
    native.check(native.lib().li4_debug_set_attention_wait_limit(0), "debug_set_attention_wait_limit")
    for _ in range(2):
        assert torch.equal(paged.prompt_attention(q, k, v, cu, max(lens))[:T], want[:T])
    assert native.device_errors() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_waits_run_out_over_a_paged_cache_with_care(paged, native, d):  # noqa: F811
    """The same over pages, cut ranges and items that are run again (a NaN value)."""
    dtype, H, Hkv, kv, new = torch.bfloat16, 8, 2, [5000, 300], [200, 100]
    ck, cv, tables, keys, values = make_cache(kv, Hkv, d, 16, dtype, 4)
    cv[int(tables[0, 0]), 0, :, 3] = float("nan")
    q = rand((sum(new), H, d), dtype, 5)
    args = (q, ck, cv, tables, i32(kv), i32(cumulative(new)), max(new))
    want = paged.paged_attention(*args)
    for polls in (1, 5, 40, 200, 1000):
        native.check(native.lib().li4_debug_set_attention_wait_limit(polls), "debug_set_attention_wait_limit")
        paged.paged_attention(*args)
        torch.cuda.synchronize()
        assert native.device_errors() in (0, 256)
    native.check(native.lib().li4_debug_set_attention_wait_limit(0), "debug_set_attention_wait_limit")
    got = paged.paged_attention(*args)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    check(got[200:], q[200:], keys[1:], values[1:], [100])
    assert native.device_errors() == 0
