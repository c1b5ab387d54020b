"""The paged-cache operators on the GPU against plain implementations in 64 bits.

Attention tolerance, per output o of a query that sees L keys (u = eps / 2 of the 16-bit type, S = sum_j
p_j |v_j| with the softmax's p, A = max_j scale sum_d |q_d k_jd|):
  the final rounding                                     u |o|
  probabilities rounded to the type                      u S   (and, fp16 alone, 2^-25 sum_j |v_j| below its
                                                               subnormal step, as every p is at most 1 x the sum)
  scores: fp32 sums of exact products over d dims, the product with the scale and the exponent's
  argument move ln p by delta <= (d + 8) 2^-23 A + 2^-21; numerator and sum both     2 delta S
  fp32 sums over the keys, a step per 16 keys and the joins of parts                 (L / 16 + 64) 2^-23 2 S
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def paged():
    import build

    build.build()
    from llama import paged

    return paged


def rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def oracle_rows(q, k, v, scale):
    """q [n, d], k / v [L, d] float64 -> (out, S, A, sum |v|) with query i seeing keys 0 .. L - n + i."""
    n, L = q.shape[0], k.shape[0]
    out = torch.zeros_like(q)
    S, A, V = torch.zeros_like(q), torch.zeros(n, 1, dtype=q.dtype, device=q.device), torch.zeros_like(q)
    for i in range(n):
        seen = L - n + i + 1
        if seen <= 0:
            continue
        p = torch.softmax(k[:seen] @ q[i] * scale, 0)
        out[i], S[i], V[i] = p @ v[:seen], p @ v[:seen].abs(), v[:seen].abs().sum(0)
        A[i] = (k[:seen].abs() @ q[i].abs()).max() * abs(scale)
    return out, S, A, V


def check(got, q, keys, values, lens, scale=None):
    """got, q [T, H, d]; keys / values: per sequence [L, Hkv, d]; lens: queries per sequence."""
    dtype, d = q.dtype, q.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(dtype).eps / 2
    at = 0
    for b, n in enumerate(lens):
        k, v = keys[b], values[b]
        rep = q.shape[1] // k.shape[1]
        for h in range(q.shape[1]):
            o, S, A, V = oracle_rows(q[at:at + n, h].double(), k[:, h // rep].double(), v[:, h // rep].double(), scale)
            delta = (d + 8) * 2.0 ** -23 * A + 2.0 ** -21
            tol = u * o.abs() + (u + 2 * delta + (k.shape[0] / 16 + 64) * 2.0 ** -22) * S + 1e-30
            if dtype == torch.float16:
                tol = tol + 2.0 ** -25 * (V + 1)
            err = (got[at:at + n, h].double() - o).abs()
            assert bool((err <= tol).all()), (b, h, n, k.shape[0], float((err / tol).max()))
        at += n


HEADS = [(32, 8, 64), (8, 2, 128), (4, 4, 64), (7, 1, 128), (6, 2, 32), (12, 4, 80), (2, 1, 8), (40, 8, 64),
         (16, 1, 64), (5, 1, 112), (128, 1, 64), (100, 1, 24)]
PROMPTS = [[1], [2, 1], [33], [128], [0, 5, 0, 17, 0], [129, 127, 1, 64], [300, 3, 257]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", PROMPTS, ids=str)
@pytest.mark.parametrize("H,Hkv,d", HEADS[:6])
def test_prompt_attention(paged, H, Hkv, d, lens, dtype):
    T = sum(lens)
    q, k, v = rand((T, H, d), dtype, 1), rand((T, Hkv, d), dtype, 2), rand((T, Hkv, d), dtype, 3)
    got = paged.prompt_attention(q, k, v, i32(cumulative(lens)), max(lens))
    check(got, q, list(k.split(lens)), list(v.split(lens)), lens)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,d", HEADS[6:])
def test_prompt_attention_other_heads(paged, H, Hkv, d, dtype):
    lens = [70, 1, 140]
    T = sum(lens)
    q, k, v = rand((T, H, d), dtype, 1), rand((T, Hkv, d), dtype, 2), rand((T, Hkv, d), dtype, 3)
    got = paged.prompt_attention(q, k, v, i32(cumulative(lens)), max(lens))
    check(got, q, list(k.split(lens)), list(v.split(lens)), lens)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_attention_long_against_tiles(paged, d):
    """A prompt of several thousand tokens, every 97th query of it."""
    n, H, Hkv, dtype = 4133, 4, 1, torch.bfloat16
    q, k, v = rand((n, H, d), dtype, 4), rand((n, Hkv, d), dtype, 5), rand((n, Hkv, d), dtype, 6)
    got = paged.prompt_attention(q, k, v, i32([0, n]), n)
    for i in list(range(0, n, 97)) + [n - 1]:
        check(got[i:i + 1], q[i:i + 1], [k[:i + 1]], [v[:i + 1]], [1])


def test_prompt_attention_very_long(paged):
    n, dtype = 70001, torch.float16
    q, k, v = rand((n, 2, 64), dtype, 4), rand((n, 1, 64), dtype, 5), rand((n, 1, 64), dtype, 6)
    got = paged.prompt_attention(q, k, v, i32([0, n]), n)
    for i in [0, 1, 127, 128, 4095, 32768, 65535, 65536, 69999, 70000]:
        check(got[i:i + 1], q[i:i + 1], [k[:i + 1]], [v[:i + 1]], [1])


@pytest.mark.parametrize("claim", [1, 50])
def test_prompt_attention_many_prompts(paged, claim):
    """More sequences than one round of the item search looks at, some of them empty."""
    lens = [(7 * b) % 50 for b in range(150)]
    T = sum(lens)
    q, k, v = rand((T, 4, 32), torch.bfloat16, 7), rand((T, 2, 32), torch.bfloat16, 8), rand((T, 2, 32), torch.bfloat16, 9)
    got = paged.prompt_attention(q, k, v, i32(cumulative(lens)), claim)
    check(got, q, list(k.split(lens)), list(v.split(lens)), lens)


def test_two_prompt_batches_at_once(paged):
    """Calls on two streams at the same time give what they give alone."""
    batches = []
    for i in range(2):
        lens = [900 + 100 * i, 333, 1500]
        T = sum(lens)
        q, k, v = (rand((T, h, 128), torch.float16, 60 + 3 * i + h) for h in (8, 2, 2))
        batches.append((q, k, v, i32(cumulative(lens)), 1500))
    want = [paged.prompt_attention(*b) for b in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged.prompt_attention(*batches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("d", [64, 128])
def test_long_chunk_is_cut_and_joined_alike_every_time(paged, d):
    """Few items over many keys: ranges of keys on different SMs, joined in order."""
    ck, cv, tables, keys, values = make_cache([9001, 40], 2, d, 32, torch.bfloat16, 70)
    q = rand((170, 8, d), torch.bfloat16, 71)
    args = (q, ck, cv, tables, i32([9001, 40]), i32([0, 130, 170]), 130)
    got = paged.paged_attention(*args)
    check(got, q, keys, values, [130, 40])
    for _ in range(3):
        assert torch.equal(got, paged.paged_attention(*args))


def test_no_bounded_wait_ran_out(paged):
    from llama import _native

    assert _native.device_errors() == 0


def test_prompt_attention_wrong_max_len_is_only_slower(paged):
    lens = [200, 31]
    q, k, v = (rand((231, h, 64), torch.float16, 7 + h) for h in (8, 2, 2))
    cu = i32(cumulative(lens))
    want = paged.prompt_attention(q, k, v, cu, 200)
    for claim in (0, 1, 10000):
        got = paged.prompt_attention(q, k, v, cu, claim)
        check(got, q, list(k.split(lens)), list(v.split(lens)), lens)
    assert torch.equal(want, paged.prompt_attention(q, k, v, cu, 200))


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_attention_strided_rows_and_rows_past_the_end(paged, dtype):
    lens, H, Hkv, d, extra = [45, 100], 8, 2, 64, 13
    T = sum(lens) + extra
    qkv = rand((T, (H + 2 * Hkv) * d), dtype, 8)
    qkv[sum(lens):] = float("nan")  # what lies behind the last sequence is nobody's
    q = qkv[:, :H * d].view(T, H, d)
    k, v = qkv[:, H * d:(H + Hkv) * d].view(T, Hkv, d), qkv[:, (H + Hkv) * d:].view(T, Hkv, d)
    wide = torch.full((T, H, 2 * d), 7.0, dtype=dtype, device="cuda")
    out = wide[..., :d]
    got = paged.prompt_attention(q, k, v, i32(cumulative(lens)), 100, out=out)
    assert got is out
    n = sum(lens)
    check(out[:n], q[:n], list(k[:n].split(lens)), list(v[:n].split(lens)), lens)
    assert bool((wide[n:] == 7).all()) and bool((wide[..., d:] == 7).all())
    # rows of the output that start 16 bytes past a 32-byte sector
    odd_out = torch.full((T, H, d + 16), 7.0, dtype=dtype, device="cuda")
    assert torch.equal(paged.prompt_attention(q, k, v, i32(cumulative(lens)), 100, out=odd_out[..., 8:8 + d])[:n], out[:n])
    assert bool((odd_out[n:] == 7).all()) and bool((odd_out[..., :8] == 7).all()) and bool((odd_out[..., 8 + d:] == 7).all())
    # other layouts: heads outermost, a misaligned first element, a broadcast key head
    q2 = q[:n].transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(n * Hkv * d + 1, dtype=dtype, device="cuda")[1:].view(n, Hkv, d)
    odd.copy_(k[:n])
    got2 = paged.prompt_attention(q2, odd, v[:n], i32(cumulative(lens)), 100)
    assert torch.equal(got2, out[:n])
    one = k[:n, :1].expand(n, Hkv, d)
    check(paged.prompt_attention(q2, one, v[:n], i32(cumulative(lens)), 100), q2, list(one.split(lens)),
          list(v[:n].split(lens)), lens)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_attention_scales_and_growing_scores(paged, dtype, scale):
    """Scores that grow along the keys make the running maximum move in every tile."""
    n, H, Hkv, d = 700, 4, 2, 64
    q, k, v = rand((n, H, d), dtype, 9), rand((n, Hkv, d), dtype, 10), rand((n, Hkv, d), dtype, 11)
    k = (k.float() * torch.linspace(0.05, 3, n, device="cuda")[:, None, None]).to(dtype)
    got = paged.prompt_attention(q, k, v, i32([0, n]), n, scale=scale)
    check(got, q, [k], [v], [n], scale=scale)


def poisoned(shape, dtype):
    t = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
    t[::3] = float("inf")
    return t


def make_cache(lens_kv, Hkv, d, page, dtype, seed, layout="heads", spare=3, slack=2):
    """A cache whose unused rows, pages and table entries are poison; returns (k pages, v pages, tables, keys, values)."""
    blocks = [-(-n // page) for n in lens_kv]
    num = sum(blocks) + spare
    order = list(range(num))
    random.Random(seed).shuffle(order)
    tables = torch.full((len(lens_kv), max(blocks + [0]) + slack), -1, dtype=torch.int32, device="cuda")
    tables[:, -1] = 1 << 30
    shape = (num, Hkv, page, d) if layout == "heads" else (num, page, Hkv, d)
    ck, cv = poisoned(shape, dtype), poisoned(shape, dtype)
    if layout == "heads":
        ck, cv = ck.transpose(1, 2), cv.transpose(1, 2)
    keys, values, at = [], [], 0
    for b, n in enumerate(lens_kv):
        pages = order[at:at + blocks[b]]
        at += blocks[b]
        tables[b, :blocks[b]] = i32(pages)
        k, v = rand((n, Hkv, d), dtype, seed + 2 * b + 1), rand((n, Hkv, d), dtype, seed + 2 * b + 2)
        for j, p in enumerate(pages):
            part = slice(j * page, min(n, (j + 1) * page))
            ck[p, :part.stop - part.start] = k[part]
            cv[p, :part.stop - part.start] = v[part]
        keys.append(k)
        values.append(v)
    return ck, cv, tables, keys, values


STEPS = [  # (new tokens, tokens of the cache with them) per request
    [(1, 1)], [(1, 300)], [(1, 17), (1, 1), (0, 40), (1, 700)], [(2, 65), (4, 4), (3, 1000)],
    [(64, 64), (1, 513), (33, 200)], [(150, 411), (1, 2), (0, 0), (129, 129)], [(5, 3), (7, 0), (40, 12)],
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", STEPS, ids=str)
@pytest.mark.parametrize("H,Hkv,d,page", [(32, 8, 64, 16), (8, 2, 128, 64), (7, 1, 128, 8), (6, 2, 32, 256),
                                          (4, 4, 64, 128), (12, 4, 80, 32), (24, 1, 128, 1024)])
def test_paged_attention(paged, H, Hkv, d, page, step, dtype):
    new, kv = [s[0] for s in step], [s[1] for s in step]
    ck, cv, tables, keys, values = make_cache(kv, Hkv, d, page, dtype, 20)
    q = rand((sum(new), H, d), dtype, 12)
    got = paged.paged_attention(q, ck, cv, tables, i32(kv), i32(cumulative(new)), max(new))
    check(got, q, keys, values, new)


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_attention_long_contexts_share_the_gpu(paged, d, new):
    """Very different lengths in one step: shares that cut sequences and shares that hold several."""
    kv = [9000, 3, 1, 130, 5000, 77, 256, 12001]
    ck, cv, tables, keys, values = make_cache(kv, 2, d, 16, torch.float16, 21)
    q = rand((len(kv) * new, 8, d), torch.float16, 13)
    args = (q, ck, cv, tables, i32(kv), i32(cumulative([new] * len(kv))), new)
    got = paged.paged_attention(*args)
    check(got, q, keys, values, [new] * len(kv))
    for _ in range(3):
        assert torch.equal(got, paged.paged_attention(*args))


def test_paged_attention_many_requests(paged):
    kv = [1 + (37 * b) % 211 for b in range(400)]
    ck, cv, tables, keys, values = make_cache(kv, 1, 64, 8, torch.float16, 22)
    q = rand((400, 2, 64), torch.float16, 14)
    got = paged.paged_attention(q, ck, cv, tables, i32(kv), i32(cumulative([1] * 400)), 1)
    check(got, q, keys, values, [1] * 400)


@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_layouts_agree(paged, new):
    kv, H, Hkv, d = [100, 260], 8, 4, 64
    a = make_cache(kv, Hkv, d, 16, torch.bfloat16, 23)
    b = make_cache(kv, Hkv, d, 16, torch.bfloat16, 23, layout="rows")
    q = rand((2 * new, H, d), torch.bfloat16, 15)
    rest = (i32(kv), i32([0, new, 2 * new]), new)
    assert torch.equal(paged.paged_attention(q, *a[:3], *rest), paged.paged_attention(q, *b[:3], *rest))


@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_pages_outside_the_cache_read_as_zeros(paged, new):
    kv, H, Hkv, d, page = [90], 4, 1, 64, 16
    ck, cv, tables, keys, values = make_cache(kv, Hkv, d, page, torch.float16, 24)
    tables[0, 1], tables[0, 3] = -5, ck.shape[0]
    for t in (keys[0], values[0]):
        t[page:2 * page] = 0
        t[3 * page:4 * page] = 0
    q = rand((new, H, d), torch.float16, 16)
    got = paged.paged_attention(q, ck, cv, tables, i32(kv), i32([0, new]), new)
    check(got, q, keys, values, [new])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [3, 90, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_not_seen_do_not_matter(paged, dtype, n, bad):
    """A NaN or infinity in value row j reaches the queries that see j and no other."""
    H, Hkv, d, j = 4, 2, 64, n - 2
    q, k, v = rand((n, H, d), dtype, 17), rand((n, Hkv, d), dtype, 18), rand((n, Hkv, d), dtype, 19)
    v[j, :, 5] = bad
    k[n - 1] = bad
    got = paged.prompt_attention(q, k, v, i32([0, n]), n)
    check(got[:j], q[:j], [k[:j]], [v[:j]], [j])
    assert not bool(torch.isfinite(got[j, :, 5]).any())
    # the same keys in a cache
    page = 16
    ck = torch.zeros(-(-n // page), page, Hkv, d, dtype=dtype, device="cuda")
    cv = torch.zeros_like(ck)
    ck.view(-1, Hkv, d)[:n], cv.view(-1, Hkv, d)[:n] = k, v
    tables = torch.arange(ck.shape[0], dtype=torch.int32, device="cuda")[None]
    got = paged.paged_attention(q, ck, cv, tables, i32([n]), i32([0, n]), n)
    check(got[:j], q[:j], [k[:j]], [v[:j]], [j])
    assert not bool(torch.isfinite(got[j, :, 5]).any())


@pytest.mark.parametrize("new", [1, 70])
def test_offsets_past_32_bits(paged, new):
    """Pages whose rows start more than 2^31 elements into the cache."""
    page, Hkv, d, H = 64, 8, 128, 8
    num = (1 << 31) // (page * Hkv * d) + 40
    ck = torch.zeros(num, page, Hkv, d, dtype=torch.float16, device="cuda")
    cv = torch.zeros_like(ck)
    n, pages = 150, [num - 1, num - 30, num - 17]
    k, v = rand((n, Hkv, d), torch.float16, 25), rand((n, Hkv, d), torch.float16, 26)
    q, kr = rand((n, H, d), torch.float16, 27), torch.empty_like(k)
    slots = torch.tensor([pages[j // page] * page + j % page for j in range(n)], device="cuda")
    cos, sin = torch.ones(n, d // 2, device="cuda"), torch.zeros(n, d // 2, device="cuda")
    paged.rope_paged_write(q, k, v, cos, sin, torch.arange(n, dtype=torch.int32, device="cuda"), slots, ck, cv, k_out=kr)
    assert torch.equal(kr, k) and torch.equal(ck[num - 1], k[:page]) and torch.equal(cv[num - 17, :22], v[128:])
    got = paged.paged_attention(q[n - new:], ck, cv, i32([pages]), i32([n]), i32([0, new]), new)
    check(got, q[n - new:], [k], [v], [new])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("H,Hkv,d,page", [(32, 8, 64, 16), (3, 1, 128, 8), (4, 4, 40, 32), (2, 2, 256, 64)])
def test_rope_paged_write(paged, H, Hkv, d, page, T, dtype):
    """Two products and a sum of fp32 (each off by 2^-24 of its terms), one rounding to the type."""
    qkv = rand((T, (H + 2 * Hkv) * d), dtype, 30)
    q, k = qkv[:, :H * d].view(T, H, d), qkv[:, H * d:(H + Hkv) * d].view(T, Hkv, d)
    v = qkv[:, (H + Hkv) * d:].view(T, Hkv, d)
    P = 500
    angle = torch.rand(P, d // 2, device="cuda", generator=torch.Generator(device="cuda").manual_seed(31)) * 6.28
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, P, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(32)).int()
    num = -(-T // page) + 2
    slots = torch.randperm(num * page, device="cuda", generator=torch.Generator(device="cuda").manual_seed(33))[:T]
    slots = slots.contiguous()
    if T > 2:
        slots[1] = -1
    ck, cv = torch.full((num, page, Hkv, d), 3.0, dtype=dtype, device="cuda"), \
        torch.full((num, Hkv, page, d), 4.0, dtype=dtype, device="cuda").transpose(1, 2)
    want_k, want_v = ck.clone(), cv.clone()
    src = qkv.clone()
    q_rot, k_rot = paged.rope_paged_write(q, k, v, cos, sin, pos, slots, ck, cv)
    assert torch.equal(src, qkv)
    u = torch.finfo(dtype).eps / 2
    for x, got in ((q, q_rot), (k, k_rot)):
        c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]
        a, b = x[..., 0::2].double(), x[..., 1::2].double()
        want = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
        mag = torch.stack([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1).flatten(-2)
        tol = u * want.abs() + 2.0 ** -22 * mag + 2.0 ** -24 * (dtype == torch.float16)
        assert bool(((got.double() - want).abs() <= tol).all())
    keep = slots >= 0
    want_k[slots[keep] // page, slots[keep] % page] = k_rot[keep]
    want_v[slots[keep] // page, slots[keep] % page] = v[keep]
    assert torch.equal(ck, want_k) and torch.equal(cv, want_v)
    # in place, and without the packed keys
    none_q, none_k = paged.rope_paged_write(q, k, v, cos, sin, pos, slots, ck, cv, need_k=False)
    assert none_k is None and torch.equal(none_q, q_rot)
    paged.rope_paged_write(q, k, v, cos, sin, pos, slots, ck, cv, q_out=q, k_out=k)
    assert torch.equal(q, q_rot) and torch.equal(k, k_rot) and torch.equal(ck, want_k)


def test_rope_paged_write_reports_bad_positions_and_slots(paged):
    from llama import _native

    _native.device_errors()
    q, k = rand((3, 2, 64), torch.float16, 34), rand((3, 1, 64), torch.float16, 35)
    cos = torch.ones(4, 32, device="cuda")
    ck = torch.zeros(2, 16, 1, 64, dtype=torch.float16, device="cuda")
    cv = torch.zeros_like(ck)
    good = torch.tensor([0, 1, 31], device="cuda")
    paged.rope_paged_write(q, k, k, cos, cos, i32([0, 3, 1]), good, ck, cv)
    assert _native.device_errors() == 0
    before = ck.clone()
    for pos, slots in (([0, 4, 1], good), ([-1, 0, 0], good), ([0, 0, 0], torch.tensor([0, 32, 1 << 40], device="cuda"))):
        ck.copy_(before)
        paged.rope_paged_write(q, k, k, cos, cos, i32(pos), slots, ck, cv)
        assert _native.device_errors() == 128
    assert _native.device_errors() == 0


def append_oracle(ctx, new, tables, stack, n_free, page, T):
    tables, stack, asked, cu = [list(r) for r in tables], list(stack[:n_free]), 0, [0]
    positions, slots, lens, granted = [], [], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        held, want = -(-c // page), -(-(c + n) // page)
        fits = want <= len(tables[b])
        asked += want - held if fits else 0
        ok = fits and (want == held or asked <= n_free)
        if ok:
            for j in range(held, want):
                tables[b][j] = stack.pop()
        for p in range(c, c + n):
            positions.append(p)
            slots.append(tables[b][p // page] * page + p % page if ok else -1)
        cu.append(cu[-1] + n)
        lens.append(c + n if ok else c)
        granted.append(ok)
    positions += [0] * (T - len(positions))
    slots += [-1] * (T - len(slots))
    return tables, cu, positions, slots, lens, [len(stack)], granted


APPENDS = [  # requests, longest context, most new tokens, page size, blocks per table, free pages (None: plenty)
    (1, 0, 1, 16, 4, None), (5, 40, 3, 8, 8, None), (64, 500, 1, 16, 40, None), (33, 100, 70, 8, 24, None),
    (7, 30, 900, 32, 32, None), (300, 64, 40, 16, 8, None), (20, 100, 60, 16, 12, 9), (20, 100, 60, 16, 6, None),
    (8192, 20, 2, 8, 4, None), (6, 4000, 4000, 1024, 8, 3), (0, 0, 0, 16, 4, None),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_paged_append(paged, case, in_place):
    B, ctx_hi, new_hi, page, width, pages = case
    rng = random.Random(B * 7 + page)
    ctx = [min(rng.randint(0, ctx_hi), width * page) for _ in range(B)]
    new = [rng.choice([0, new_hi, rng.randint(0, new_hi)]) for _ in range(B)]
    held = [-(-c // page) for c in ctx]
    need = sum(-(-(c + n) // page) - h for c, n, h in zip(ctx, new, held))
    free = need + 5 if pages is None else pages
    ids = list(range(sum(held) + free))
    rng.shuffle(ids)
    tables, at = [], 0
    for h in held:
        tables.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    stack = ids[at:] + [-9] * 4
    T = sum(new) + 3
    tt = i32(tables).view(B, width)
    kv, nf = i32(ctx), i32([free])
    out = dict(kv_lens_out=kv, n_free_out=nf) if in_place else {}
    step = paged.paged_append(kv, i32(new), tt, i32(stack), nf, page, T, **out)
    w_tables, w_cu, w_pos, w_slots, w_lens, w_free, w_ok = append_oracle(ctx, new, tables, stack, free, page, T)
    assert step.cu_seqlens.tolist() == w_cu
    assert step.granted.tolist() == w_ok
    assert step.kv_lens.tolist() == w_lens and step.n_free.tolist() == w_free
    assert step.positions.tolist() == w_pos
    assert step.slots.tolist() == w_slots
    assert tt.tolist() == w_tables
    if in_place:
        assert step.kv_lens is kv and step.n_free is nf
    else:
        assert kv.tolist() == ctx and nf.tolist() == [free]


def test_paged_append_refuses_lengths_out_of_range(paged):
    """Lengths that are negative or whose sums pass 32 bits take nothing and hurt no one before them."""
    big = 1 << 29
    tables = torch.full((9, 6), -1, dtype=torch.int32, device="cuda")
    ctx = [3, 0, -4, 0, 0, 0, 0, 7, big]
    new = [2, big, 1, big, big, big, -9, big, 2 * big]
    nf = i32([5])
    step = paged.paged_append(i32(ctx), i32(new), tables, i32([4, 5, 6, 7, 8]), nf, 16, 2)
    assert step.granted.tolist() == [True] + [False] * 8
    assert step.kv_lens.tolist() == [5] + ctx[1:] and step.n_free.tolist() == [5]
    assert step.positions.tolist() == [3, 4] and bool((tables == -1).all())
    assert step.cu_seqlens[:2].tolist() == [0, 2] and step.slots.tolist() == [-16 + 3, -16 + 4]
    # more tokens than the host counted: the first requests that fit are served
    tables = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    step = paged.paged_append(i32([0, 0, 0]), i32([3, 4, 5]), tables, i32([1, 2, 3]), i32([3]), 16, 8)
    assert step.granted.tolist() == [True, True, False] and step.n_free.tolist() == [1]
    assert step.slots.tolist() == [48, 49, 50, 32, 33, 34, 35, -1]


def test_paged_append_table_rows_with_a_stride(paged):
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    step = paged.paged_append(i32([0, 0, 0]), i32([17, 0, 5]), wide[:, :6], i32(list(range(8))), i32([8]), 16, 22)
    assert wide[:, 0].tolist() == [7, -1, 5] and wide[0, 1].item() == 6 and bool((wide[:, 6:] == -1).all())
    assert step.slots.tolist() == [112 + i for i in range(16)] + [96] + [80 + i for i in range(5)]


def test_refusals_launch_nothing(paged):
    q, k = rand((4, 4, 64), torch.float16, 40), rand((4, 2, 64), torch.float16, 41)
    cu = i32([0, 4])
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.float16, device="cuda")
    tables, lens = i32([[0, 1]]), i32([4])
    bad = [
        lambda: paged.prompt_attention(q.float(), k.float(), k.float(), cu, 4),
        lambda: paged.prompt_attention(q, k.bfloat16(), k, cu, 4),
        lambda: paged.prompt_attention(q, k[:3], k[:3], cu, 4),
        lambda: paged.prompt_attention(q, k, k[:, :1], cu, 4),
        lambda: paged.prompt_attention(q[:, :3].contiguous(), k, k, cu, 4),
        lambda: paged.prompt_attention(q, k, k, cu.long(), 4),
        lambda: paged.prompt_attention(q, k, k, cu.cpu(), 4),
        lambda: paged.prompt_attention(q, k, k, cu, -1),
        lambda: paged.prompt_attention(q, k, k, cu, 4, out=q),
        lambda: paged.prompt_attention(q, k, k, cu, 4, out=torch.empty(4, 4, 32, dtype=q.dtype, device="cuda")),
        lambda: paged.prompt_attention(q[0], k, k, cu, 4),
        lambda: paged.prompt_attention(rand((4, 4, 136), torch.float16, 1), rand((4, 2, 136), torch.float16, 1),
                                       rand((4, 2, 136), torch.float16, 1), cu, 4),
        lambda: paged.paged_attention(q, cache.transpose(2, 3), cache, tables, lens, cu, 4),
        lambda: paged.paged_attention(q, cache[:, :12], cache[:, :12], tables, lens, cu, 4),
        lambda: paged.paged_attention(q, cache, cache[:1], tables, lens, cu, 4),
        lambda: paged.paged_attention(q, cache, cache, tables.long(), lens, cu, 4),
        lambda: paged.paged_attention(q, cache, cache, tables, lens[:0], cu, 4),
        lambda: paged.paged_attention(q, cache.bfloat16(), cache.bfloat16(), tables, lens, cu, 4),
        lambda: paged.paged_append(lens.long(), lens, tables, lens, lens, 16, 4),
        lambda: paged.paged_append(lens, lens, tables, lens, i32([1, 2]), 16, 4),
        lambda: paged.paged_append(lens, lens, tables, lens, lens, 12, 4),
        lambda: paged.rope_paged_write(q, k, k, torch.zeros(4, 31, device="cuda"), torch.zeros(4, 31, device="cuda"),
                                       i32([0] * 4), torch.zeros(4, dtype=torch.long, device="cuda"), cache, cache),
        lambda: paged.rope_paged_write(q, k, k, torch.zeros(4, 32, device="cuda"), torch.zeros(4, 32, device="cuda"),
                                       i32([0] * 4).long(), torch.zeros(4, dtype=torch.long, device="cuda"), cache, cache),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_empty_calls(paged):
    q, k = rand((0, 4, 64), torch.float16, 42), rand((0, 2, 64), torch.float16, 43)
    assert paged.prompt_attention(q, k, k, i32([0]), 0).shape == q.shape
    assert paged.prompt_attention(q, k, k, i32([0, 0, 0]), 0).shape == q.shape
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.float16, device="cuda")
    assert paged.paged_attention(q, cache, cache, i32([[0]]), i32([0]), i32([0, 0]), 0).shape == q.shape
    # no pages at all, tokens without keys: zeros
    q = rand((3, 4, 64), torch.float16, 44)
    none = torch.zeros(0, 16, 2, 64, dtype=torch.float16, device="cuda")
    got = paged.paged_attention(q, none, none, torch.zeros(1, 0, dtype=torch.int32, device="cuda"), i32([9]), i32([0, 3]), 3)
    assert bool((got == 0).all())


def test_other_streams_and_graphs(paged):
    """A captured step replays with the lengths of the day; two graphs on two streams do not disturb each other."""
    H, Hkv, d, page = 8, 2, 64, 16
    kv0 = [700, 20, 333]
    ck, cv, tables, keys, values = make_cache([1000, 900, 800], Hkv, d, page, torch.float16, 50)
    q = rand((3, H, d), torch.float16, 51)
    lens = i32(kv0)
    cu = i32([0, 1, 2, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.paged_attention(q, ck, cv, tables, lens, cu, 1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged.paged_attention(q, ck, cv, tables, lens, cu, 1))
        graphs.append(g)
    for kv in ([700, 20, 333], [1, 900, 512], [1000, 3, 800]):
        lens.copy_(i32(kv))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for o in outs:
            check(o, q, [k[:n] for k, n in zip(keys, kv)], [v[:n] for v, n in zip(values, kv)], [1, 1, 1])


# ---------------------------------------------------------------------------------------------
# the operators together: the model's steps over the paged cache against its padded forward
# ---------------------------------------------------------------------------------------------
def tiny_model(dim=256, heads=4, kv_heads=1, seed=0):
    from llama.model import Llama, ModelArgs

    args = ModelArgs(dim=dim, n_layers=2, n_heads=heads, n_kv_heads=kv_heads, vocab_size=500, multiple_of=128,
                     max_batch_size=4, max_seq_len=256)
    torch.manual_seed(seed)
    torch.set_default_dtype(torch.float16)
    try:
        with torch.device("cuda"):
            model = Llama(args)
    finally:
        torch.set_default_dtype(torch.float32)
    with torch.no_grad():
        for name, p in model.named_parameters():
            p.copy_(1.0 + 0.1 * torch.randn_like(p) if name.endswith("norm.weight") else 0.05 * torch.randn_like(p))
    return model.eval()


@pytest.mark.parametrize("heads,kv_heads,page", [(4, 1, 16), (4, 4, 8), (2, 1, 64)])
def test_model_steps_over_the_paged_cache(paged, heads, kv_heads, page):
    """Prompts of three requests, chunks and single tokens, one request ending and another taking its pages: the
    logits of every step against Llama.forward on that request alone.  Both run the same fp16 modules; the
    attention and RoPE roundings differ by a few steps of fp16 on values the 2 blocks pass on, so logits agree
    within 1% of their range (a wrong key, position or page moves them by its whole)."""
    model = tiny_model(heads=heads, kv_heads=kv_heads)
    rng = random.Random(1)
    texts = [[rng.randrange(500) for _ in range(200)] for _ in range(4)]
    cache = model.paged_cache(num_pages=-(-200 // page) * 3 + 3, page_size=page, max_requests=3)
    with pytest.raises(ValueError):
        model.forward_paged(torch.zeros(0, dtype=torch.long, device="cuda"), None, cache, 0)
    fed, owner = [0, 0, 0], [0, 1, 2]

    def step(new, whole=False):
        tokens = [t for r, n in enumerate(new) for t in texts[owner[r]][fed[r]:fed[r] + n]]
        plan = cache.append(i32(new), len(tokens))
        logits = model.forward_paged(torch.tensor(tokens, device="cuda"), plan, cache, max(new), whole_prompts=whole)
        for r, n in enumerate(new):
            fed[r] += n
            if n:
                model.reset_cache()
                want = model(torch.tensor([texts[owner[r]][:fed[r]]], device="cuda"), 0)[0, -1]
                assert bool(plan.granted[r])
                assert float((logits[r] - want).abs().max()) <= 1e-2 * float(want.abs().max())

    with torch.no_grad():
        step([37, 1, 90], whole=True)
        step([1, 1, 1])
        step([1, 64, 1])
        step([0, 1, 1])
        cache.release(torch.tensor([False, False, True], device="cuda"))
        fed[2], owner[2] = 0, 3
        step([1, 1, 130])
        step([50, 2, 3])
        cache.release(torch.tensor([True, True, True], device="cuda"))
        assert int(cache.n_free) == cache.free_pages.numel()
        assert sorted(cache.free_pages.tolist()) == list(range(cache.free_pages.numel()))


class Letters:
    """A tokenizer of one token per character."""

    pad_id, eos_id = 0, 1

    def encode(self, text, bos, eos):
        return [2] + [3 + ord(c) % 490 for c in text]

    def decode(self, ids):
        return " ".join(map(str, ids))


@pytest.mark.parametrize("quantized", [False, True])
def test_generate_paged(paged, quantized):
    """Every greedy token of every answer is the best of Llama.forward's logits for the text before it, up to 2% of
    their range (the two paths round at different places); the captured step gives the eager loop's answers."""
    from llama import quantize

    model = tiny_model(seed=3)
    if quantized:
        quantize.quantize_model(model, 128)
        quantize.set_dequant_impl("v4")
    try:
        prompts, tok = ["a", "some longer prompt " * 5, "of three", "the fourth"], Letters()
        got = model.generate_paged(tok, prompts, 12, 0.0, 1.0, "cuda", page_size=8)
        again = model.generate_paged(tok, prompts, 12, 0.0, 1.0, "cuda", page_size=32, cuda_graph=True)
        assert [len(g["generation"].split()) for g in got] == [12] * 4 or all(g["generation"] for g in got)
        for text, a, b in zip(prompts, got, again):
            for answer in (a, b):
                ids = tok.encode(text, True, False)
                gen = [int(x) for x in answer["generation"].split()]
                with torch.no_grad():
                    model.reset_cache()
                    logits = model(torch.tensor([ids + gen], device="cuda"), 0)[0].float()
                for i, t in enumerate(gen):
                    row = logits[len(ids) - 1 + i]
                    assert float(row.max() - row[t]) <= 2e-2 * float(row.max() - row.min())
        sampled = model.generate_paged(tok, prompts, 5, 0.8, 0.9, "cuda")
        assert len(sampled) == 4
        with pytest.raises(ValueError):
            model.generate_paged(tok, prompts, 5, 0.8, 0.9, "cuda", cuda_graph=True)
        with pytest.raises(ValueError):
            model.generate_paged(tok, ["x" * 600], 5, 0.0, 0.9, "cuda")
    finally:
        quantize.set_dequant_impl("v1")
