"""The same call gives the same bits, whatever ran on the GPU before it."""
import pytest
import torch

from test_paged_gpu import TYPES, cumulative, i32, paged, rand  # noqa: F401 (paged: the fixture)
from test_paged_int4_gpu import layout

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hkv,D", [(7, 1, 128), (40, 8, 64), (20, 1, 128), (10, 2, 96), (9, 1, 32), (12, 4, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_a_tile_without_a_query(paged, H, Hkv, D, dtype):  # noqa: F811
    """Groups of heads that do not divide 128 leave rows of a tile without a query: what shared memory holds there, here
    queries of other calls with scores of many sizes, changes nothing."""
    shape = [(1682, 40), (809, 130), (300, 1), (64, 33)]
    q, ck, cv, table, lens, cu, most, _ = layout(paged, shape, H, Hkv, D, 16, dtype, 61)
    k16, v16 = (torch.nan_to_num(c.values(), 0.0) for c in (ck, cv))
    n = 300
    packed = [rand((n, heads, D), dtype, 62 + i) for i, heads in enumerate((H, Hkv, Hkv))]
    calls = {"int4": lambda: paged.paged_attention_int4(q, ck, cv, table, lens, cu, most),
             "paged": lambda: paged.paged_attention(q, k16, v16, table, lens, cu, most),
             "prompt": lambda: paged.prompt_attention(*packed, i32([0, n]), n)}
    wide = [rand((2000, heads, D), dtype, 65 + i) for i, heads in enumerate((32, 8, 8))]
    cu_wide = i32(cumulative([500, 700, 800]))
    for name, call in calls.items():
        want = None
        for grow in (0.0, 0.1, 1.0, 5.0, 30.0, 300.0):
            for _ in range(3):
                paged.prompt_attention(wide[0] * grow, wide[1], wide[2], cu_wide, 800)
                got = call()
                want = got.clone() if want is None else want
                assert torch.equal(got, want), (name, grow, int((got != want).sum()))
