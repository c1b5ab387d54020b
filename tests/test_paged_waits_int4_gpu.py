"""Bounded waits of attention over a 4-bit cache: a call whose waits ran out says so."""
import math

import pytest
import torch

from test_paged_gpu import TYPES, paged  # noqa: F401 (paged: the fixture)
from test_paged_int4_gpu import layout

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_call_says_when_its_waits_ran_out(paged, dtype, D, bad):  # noqa: F811
    """Without bit 8 the outputs are those of the default limit, with NaN values (items are run again) too; limits of a few
    polls, less than any copy takes, always set it."""
    from llama import _native as native

    shape = [(5000, 200), (300, 100), (70, 1)]
    q, ck, cv, table, lens, cu, most, _ = layout(paged, shape, 8, 2, D, 16, dtype, 41)
    if bad:
        cv.params[table[0, 0].long(), 0, 1, 0] = math.nan
    want = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
    assert native.device_errors() == 0
    try:
        for polls in (1, 2, 5, 20, 50, 100, 150, 200, 300, 400, 800, 2000):
            native.check(native.lib().li4_debug_set_attention_wait_limit(polls), "debug_set_attention_wait_limit")
            for _ in range(4):
                got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
                flags = native.device_errors()
                assert flags in (0, 256)
                if flags == 0:
                    assert torch.equal(torch.isnan(got), torch.isnan(want)), polls
                    assert torch.equal(got.nan_to_num(), want.nan_to_num()), polls
                    assert polls > 2
    finally:
        native.check(native.lib().li4_debug_set_attention_wait_limit(0), "debug_set_attention_wait_limit")
        native.device_errors()
