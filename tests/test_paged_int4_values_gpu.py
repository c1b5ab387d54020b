"""Groups of a 4-bit cache whose values c s + m are not finite, for some codes or for all: what each query gets is what the
same values of a 16-bit cache would give it.

Tolerances are those of test_paged_gpu.check, and one more for bf16 values near 2^128.  Before the division by their sum
the weights are 2^t exp(x - max) with t from 0 to 8 (the maximum in use may lag by that), so a sum of weighted values held in 32
bits is at most 2^8 Z S, Z = sum exp(x - max), S = sum p |v|: where that bound is below 2^127 no addition or rounding can pass the
largest fp32 value, above it an output may be infinite (or a NaN, of two such sums joined) though its quotient is not."""
import math

import pytest
import torch

from test_paged_gpu import TYPES, paged  # noqa: F401 (paged: the fixture)
from test_paged_int4_gpu import layout
from test_paged_nonfinite_gpu import close

pytestmark = pytest.mark.gpu


def overflows(got, q, k, v):
    """Outputs that are not finite where 2^8 Z S allows it."""
    n, H, D = q.shape
    L, rep = k.shape[0], H // k.shape[1]
    seen = torch.arange(L, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (L - n)
    x = torch.einsum("nhd,lhd->hnl", q.double(), k.double().repeat_interleave(rep, 1)) / math.sqrt(D)
    x = x.masked_fill(~seen, -math.inf)
    Z = torch.exp(x - x.amax(-1, keepdim=True)).sum(-1)
    S = torch.einsum("hnl,lhd->nhd", torch.softmax(x, -1), v.double().abs().repeat_interleave(rep, 1))
    return ~torch.isfinite(got) & (2.0 ** 8 * Z.t()[..., None] * S >= 2.0 ** 127)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (4, 2, 128), (6, 2, 96), (9, 1, 32), (8, 1, 128), (32, 1, 64)])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 40, 200])
def test_values_past_the_type(paged, n, H, Hkv, D, dtype):  # noqa: F811
    """A scale whose multiples pass the largest value, beside codes whose values are finite; an infinite offset; both signs;
    a NaN: queries that see the key get its infinities, the finite values of its group by their weights, all others none."""
    big = torch.finfo(dtype).max
    L = n + 30
    for key in sorted({L - 1, L - 1 - n // 2, 30}):
        for s, m in ((big / 4, 1.0), (-big / 4, 2.0), (big / 14, 0.0), (1.0, math.inf), (0.5, -math.inf), (math.nan, 0.0), (math.inf, 0.0)):
            q, ck, cv, table, lens, cu, most, (keys, _) = layout(paged, [(L, n), (45, 1)], H, Hkv, D, 16, dtype, 71)
            group = 1 % (D // 32)
            cv.params[table[0, key // 16].long(), key % 16, Hkv - 1, group] = torch.tensor((s, m), dtype=dtype, device="cuda")
            values = cv.values()[table[0, :-(-L // 16)].long()].flatten(0, 1)[:L]
            got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
            bad = ~torch.isfinite(values[key])  # [Hkv, D]
            assert int(bad.sum()) <= 32
            skip = torch.zeros(n, H, D, dtype=torch.bool, device="cuda")
            first = max(0, key - (L - n))
            skip[first:] = bad.repeat_interleave(H // Hkv, 0)
            want = values[key].repeat_interleave(H // Hkv, 0).expand(n - first, H, D)
            seen = skip[first:]
            same = (got[:n][first:] == want) | (torch.isnan(got[:n][first:]) & torch.isnan(want))
            assert bool(same[seen].all()), (key, s, m)
            clean = values.clone()
            clean[key][bad] = 0
            close(got[:n], q[:n], keys[0], clean, skip | overflows(got[:n], q[:n], keys[0], clean))
