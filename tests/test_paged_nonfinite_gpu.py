"""NaN and infinities in the caches and the packed keys and values: who sees them, who does not, and what they cost.

Tolerances are those of test_paged_gpu.check."""
import math

import pytest
import torch

from test_paged_gpu import TYPES, cumulative, i32, make_cache, paged, rand  # noqa: F401 (paged: the fixture)

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def close(got, q, k, v, skip=None):
    """test_paged_gpu.check for one sequence, a head's rows at a time: got, q [n, H, d], k / v [L, Hkv, d]; outputs where
    skip [n, H, d] is true are not looked at."""
    n, H, d = q.shape
    L, rep, dtype = k.shape[0], q.shape[1] // k.shape[1], q.dtype
    scale, u = 1.0 / math.sqrt(d), torch.finfo(q.dtype).eps / 2
    seen = torch.arange(L, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (L - n)
    for h in range(H):
        qh, kh, vh = q[:, h].double(), k[:, h // rep].double(), v[:, h // rep].double()
        p = torch.softmax((qh @ kh.t() * scale).masked_fill(~seen, -math.inf), 1)
        o, S = p @ vh, p @ vh.abs()
        A = ((qh.abs() @ kh.abs().t()) * seen).amax(1, keepdim=True) * scale
        delta = (d + 8) * 2.0 ** -23 * A + 2.0 ** -21
        tol = u * o.abs() + (u + 2 * delta + (L / 16 + 64) * 2.0 ** -22) * S + 1e-30
        if dtype == torch.float16:
            tol = tol + 2.0 ** -25 * (seen.double() @ vh.abs() + 1)
        good = (got[:, h].double() - o).abs() <= tol
        assert bool((good if skip is None else good | skip[:, h]).all()), (h, n, L, (~good).nonzero()[:4].tolist())


def split_check(got, q, k, v, row, dim):
    """One sequence of n queries over L keys whose value row `row` is not finite in `dim`: outputs that see it are not
    finite, all others are right."""
    n, L = q.shape[0], k.shape[0]
    first = max(0, row - (L - n))  # the first query that sees it
    assert not bool(torch.isfinite(got[first:, :, dim]).any())
    clean = v.clone()
    clean[row, :, dim] = 0
    skip = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    skip[first:, :, dim] = True
    close(got, q, k, clean, skip)


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (8, 1), (3, 3), (100, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_bad_value_anywhere_in_a_prompt(paged, dtype, H, Hkv, d, bad):  # noqa: F811
    n = 270
    q, k, v0 = rand((n, H, d), dtype, 1), rand((n, Hkv, d), dtype, 2), rand((n, Hkv, d), dtype, 3)
    for row, dim in ((0, 0), (1, d - 1), (127, 7), (128, 8), (200, d // 2), (268, 3), (269, 33)):
        v = v0.clone()
        v[row, :, dim] = bad
        got = paged.prompt_attention(q, k, v, i32([0, n]), n)
        split_check(got, q, k, v, row, dim)


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,L", [(1, 300), (2, 700), (4, 64), (8, 5000), (70, 71), (130, 3001), (300, 300)])
@pytest.mark.parametrize("page", [8, 64])
def test_a_bad_value_in_a_cache(paged, page, n, L, d, bad):  # noqa: F811
    """Single tokens, a few, chunks; contexts that are cut into ranges."""
    dtype, H, Hkv = torch.float16, 8, 2
    ck, cv, tables, keys, values = make_cache([L], Hkv, d, page, dtype, 5)
    k, v0 = keys[0], values[0]
    q = rand((n, H, d), dtype, 6)
    for row in sorted({0, L - n - 1, L - n, L - n + 1, L - n // 2 - 1, L - 2, L - 1}):
        if not 0 <= row < L:
            continue
        v = v0.clone()
        v[row, :, 5] = bad
        place = int(tables[0, row // page]), row % page
        cv[place[0], place[1], :, 5] = bad
        got = paged.paged_attention(q, ck, cv, tables, i32([L]), i32([0, n]), n)
        cv[place[0], place[1]] = v0[row]
        split_check(got, q, k, v, row, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,d", [(8, 2, 64), (3, 3, 128), (16, 1, 128), (12, 4, 72)])
def test_bad_values_in_some_of_many_prompts(paged, H, Hkv, d, dtype):  # noqa: F811
    """Several items per CTA, with and without bad values in turn, some with many of both signs; one KV head's bad values
    are no other's."""
    lens = [(37 * b) % 290 for b in range(70)]
    T = sum(lens)
    q, k, v0 = rand((T, H, d), dtype, 20), rand((T, Hkv, d), dtype, 21), rand((T, Hkv, d), dtype, 22)
    v, clean, at, rep = v0.clone(), v0.clone(), cumulative(lens), H // Hkv
    skip = torch.zeros(T, H, d, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for i in range((0, 0, 1, 0, 7)[b % 5] if n else 0):
            j, h, dim = (n - 1 - 11 * i - b) % n, (b + i) % Hkv, (5 * b + 3 * i) % d
            v[at[b] + j, h, dim] = (NAN, INF, -INF)[(b + i) % 3]
            clean[at[b] + j, h, dim] = 0
            skip[at[b] + j:at[b + 1], h * rep:(h + 1) * rep, dim] = True
    got = paged.prompt_attention(q, k, v, i32(at), max(lens))
    assert not bool((torch.isfinite(got) & skip).any())
    for b, n in enumerate(lens):
        if n:
            part = slice(at[b], at[b + 1])
            close(got[part], q[part], k[part], clean[part], skip[part])


@pytest.mark.parametrize("d", [64, 128])
def test_a_whole_hidden_stretch_of_bad_values(paged, d):  # noqa: F811
    """Every later value is NaN: rows that see none of them are right."""
    dtype, n, H, Hkv, cut = torch.bfloat16, 400, 4, 1, 150
    q, k, v = rand((n, H, d), dtype, 7), rand((n, Hkv, d), dtype, 8), rand((n, Hkv, d), dtype, 9)
    v[cut:] = NAN
    v[cut::3] = INF
    got = paged.prompt_attention(q, k, v, i32([0, n]), n)
    close(got[:cut], q[:cut], k[:cut], v[:cut])
    assert not bool(torch.isfinite(got[cut:]).any())


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [2, 333])
def test_bad_scores_make_their_rows_nan(paged, n, d, bad):  # noqa: F811
    """A NaN score (or an infinite one: infinity - infinity) makes every output of its row NaN and touches no other row,
    wherever the key stands (which of the kernel's exponentials takes it)."""
    dtype, H, Hkv, L = torch.float16, 4, 2, 400
    q0, k0, v = rand((n, H, d), dtype, 10), rand((L, Hkv, d), dtype, 11), rand((L, Hkv, d), dtype, 12)
    v[:, :, 4] = 1  # (the outputs of an infinite probability would be infinite here)
    page = 16
    tables = torch.arange(L // page, dtype=torch.int32, device="cuda")[None]
    at = [L - n + i for i in (0, n // 2, n - 1)] + [0, 1, 6, 7, 130, 135]
    for j in at:
        k = k0.clone()
        q = q0.abs() if bad == INF else q0
        k[j] = bad
        got = paged.paged_attention(q, k.view(-1, page, Hkv, d), v.view(-1, page, Hkv, d), tables, i32([L]), i32([0, n]), n)
        first = max(0, j - (L - n))
        assert bool(torch.isnan(got[first:]).all()), j
        if first:
            close(got[:first], q[:first], k[:L - n + first], v[:L - n + first])
    # a query row that is NaN is NaN alone
    q = q0.clone()
    q[n // 2, 1] = NAN
    got = paged.paged_attention(q, k0.view(-1, page, Hkv, d), v.view(-1, page, Hkv, d), tables, i32([L]), i32([0, n]), n)
    assert bool(torch.isnan(got[n // 2, 1]).all())
    rows = [i for i in range(n) if i != n // 2]
    assert bool(torch.isfinite(got[rows]).all()) and bool(torch.isfinite(got[n // 2, [0, 2, 3]]).all())


def elapsed(call, reps=5):
    call()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    for _ in range(reps):
        call()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / reps


@pytest.mark.parametrize("d", [64, 128])
def test_a_bad_value_costs_little_and_hurts_no_other_prompt(paged, d):  # noqa: F811
    """A NaN in the first value of a long prompt, and one in the middle, beside a clean prompt: the clean one's outputs
    do not move by a bit, every wait holds, and the call takes about twice a clean call's time (a CTA's first two items run
    twice; 1.6 to 2 measured).  Redoing whole rows took hundreds; 6 is allowed here, as the clocks move between calls."""
    dtype, lens, H, Hkv = torch.float16, [6000, 700], 8, 2
    T = sum(lens)
    q, k, v = rand((T, H, d), dtype, 13), rand((T, Hkv, d), dtype, 14), rand((T, Hkv, d), dtype, 15)
    cu = i32(cumulative(lens))
    want = paged.prompt_attention(q, k, v, cu, max(lens))
    clean = elapsed(lambda: paged.prompt_attention(q, k, v, cu, max(lens)))
    for row in (0, 3000, 5999):
        w = v.clone()
        w[row, :, 9] = NAN
        got = paged.prompt_attention(q, k, w, cu, max(lens))
        assert torch.equal(got[lens[0]:], want[lens[0]:])
        assert bool(torch.isnan(got[row:lens[0], :, 9]).all())
        others = [x for x in range(d) if x != 9]
        assert torch.equal(got[:row - row % 512], want[:row - row % 512])
        assert bool(torch.isfinite(got[:lens[0]][..., others]).all()) and bool(torch.isfinite(got[:row]).all())
        assert elapsed(lambda: paged.prompt_attention(q, k, w, cu, max(lens))) < 6 * clean


def test_a_bad_value_costs_little_over_long_contexts(paged):  # noqa: F811
    """Requests of a few tokens over long contexts, the first value and one that the last query alone sees NaN."""
    dtype, H, Hkv, d, page, n = torch.float16, 8, 1, 64, 64, 4
    lens = [30000] * 40
    ck, cv, tables, keys, values = make_cache(lens[:1], Hkv, d, page, dtype, 16)
    tables = tables[:, :-1].expand(40, -1).contiguous()
    q = rand((40 * n, H, d), dtype, 17)
    args = (tables, i32(lens), i32(cumulative([n] * 40)), n)
    want = paged.paged_attention(q, ck, cv, *args)
    clean = elapsed(lambda: paged.paged_attention(q, ck, cv, *args))
    bad = cv.clone(memory_format=torch.preserve_format)
    bad[int(tables[0, 0]), 0, :, 2] = NAN
    bad[int(tables[0, 29999 // page]), 29999 % page, :, 4] = INF
    got = paged.paged_attention(q, ck, bad, *args).view(40, n, H, d)
    assert bool(torch.isnan(got[..., 2]).all()) and not bool(torch.isfinite(got[:, -1, :, 4]).any())
    same = [x for x in range(d) if x not in (2, 4)]
    u = torch.finfo(dtype).eps
    ref = want.view(40, n, H, d)
    # (the last key's step sums in another order: a rounding of the type at most)
    assert bool(((got - ref)[..., same].abs() <= u * ref[..., same].abs() + 2.0 ** -14).all())
    assert bool(((got - ref)[:, :-1, :, 4].abs() <= u * ref[:, :-1, :, 4].abs() + 2.0 ** -14).all())
    assert elapsed(lambda: paged.paged_attention(q, ck, bad, *args)) < 6 * clean
    assert math.isfinite(clean)
