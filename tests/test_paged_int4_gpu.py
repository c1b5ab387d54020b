"""The paged cache in 4 bits on the GPU: its write against the definition (codes and parameters to the bit), its attention
against 64 bits over the values that the cache stands for, with the tolerance derived in test_paged_gpu.py (unpacking adds
no error: a value is c s + m rounded once, as it is in the oracle)."""
import itertools
import math
import random

import pytest
import torch

from test_paged_gpu import check, cumulative, i32, rand

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def paged():
    import build

    build.build()
    from llama import paged

    return paged


def quantized(x):
    """Codes (int64), s and m of rows [..., d] of 16-bit values, by the definition, in float64."""
    g = x.double().unflatten(-1, (-1, 32))
    fine = torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(fine, g, 0.0)
    m, top = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    want = (top - m) / 15
    # towards zero: the significand cut to the type's digits, on the subnormals' grid below the smallest exponent
    digits, least = {torch.float16: (11, -24), torch.bfloat16: (8, -133)}[x.dtype]
    power = torch.frexp(want)[1]
    unit = torch.exp2((power - digits).clamp(min=least).double())
    s = (want / unit).floor() * unit
    t = torch.where(s > 0, (g - m) / torch.where(s > 0, s, 1.0), 0.0)
    c = t.round().clamp(max=15)
    s, m, c = torch.where(fine, s, math.nan), torch.where(fine, m, math.nan), torch.where(fine, c, 0.0)
    return c.flatten(-2).long(), s.squeeze(-1).to(x.dtype), m.squeeze(-1).to(x.dtype)


def new_cache(paged, pages, ps, Hkv, D, dtype, seed, by_head=True):
    """An Int4Pages of random codes and parameters."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages, Hkv, ps) if by_head else (pages, ps, Hkv)
    codes = torch.randint(0, 256, shape + (D // 2,), generator=gen, device="cuda", dtype=torch.uint8)
    s = torch.rand(shape + (D // 32, 1), generator=gen, device="cuda") * 0.3
    m = torch.randn(shape + (D // 32, 1), generator=gen, device="cuda") * 0.3 - 7.5 * s
    params = torch.cat([s, m], -1).to(dtype)
    if by_head:
        codes, params = codes.transpose(1, 2), params.transpose(1, 2)
    return paged.Int4Pages(codes, params)


def tables(D, positions=4096):
    inv = 500000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    angles = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return angles.cos().float(), angles.sin().float()


def turned(k, cos, sin, pos):
    """Keys turned in 64 bits, rounded to 32 and then to the type."""
    x, y = k.double()[..., 0::2], k.double()[..., 1::2]
    c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]
    return torch.stack([x * c - y * s, x * s + y * c], -1).flatten(-2).float().to(k.dtype)


def same(a, b):
    return bool(((a == b) | ((a != a) & (b != b))).all())


def check_write(paged, k, v, ck, cv, slots, before, ps):
    """The cache's rows at slots hold k and v, all others what they held."""
    for x, cache, (codes0, params0) in ((k, ck, before[0]), (v, cv, before[1])):
        want_c, s, m = quantized(x)
        keep = (slots >= 0) & (slots < cache.codes.shape[0] * ps)
        page, row = slots[keep] // ps, slots[keep] % ps
        codes0[page, row] = paged.pack_codes(want_c[keep])
        params0[page, row] = torch.stack([s[keep], m[keep]], -1)
        assert torch.equal(cache.codes, codes0)
        assert same(cache.params, params0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D,T", [(4, 2, 64, 1), (32, 8, 64, 16), (8, 1, 128, 37), (3, 3, 32, 5), (6, 2, 96, 130),
                                       (1, 1, 32, 1), (32, 8, 128, 700)])
@pytest.mark.parametrize("by_head", [True, False])
def test_write(paged, H, Hkv, D, T, dtype, by_head):
    ps, pages = 16, T // 16 + 4
    wide = rand((T, (H + 2 * Hkv) * D), dtype, 1, 3.0)
    q, k, v = (t.unflatten(1, (-1, D)) for t in wide.split([H * D, Hkv * D, Hkv * D], 1))
    cos, sin = tables(D)
    gen = torch.Generator(device="cuda").manual_seed(2)
    pos = torch.randint(0, 4096, (T,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * ps, generator=gen, device="cuda")[:T].clone()
    slots[::5] = torch.where(torch.arange(len(slots[::5]), device="cuda") % 2 == 1, -1, slots[::5])
    ck, cv = (new_cache(paged, pages, ps, Hkv, D, dtype, 3 + i, by_head) for i in range(2))
    before = [(c.codes.clone(), c.params.clone()) for c in (ck, cv)]
    scratch = torch.zeros(pages, ps, Hkv, D, dtype=dtype, device="cuda")
    want_q, _ = paged.rope_paged_write(q, k, v, cos, sin, pos, slots, scratch, scratch.clone())
    got_q, got_k, got_v = paged.rope_paged_write_int4(q, k, v, cos, sin, pos, slots, ck, cv)
    assert torch.equal(got_q, want_q)
    kt = turned(k, cos, sin, pos)
    check_write(paged, kt, v, ck, cv, slots, [(a.clone(), b.clone()) for a, b in before], ps)
    for x, got in ((kt, got_k), (v, got_v)):
        c, s, m = quantized(x)
        want = (c.unflatten(-1, (-1, 32)) * s.double().unsqueeze(-1) + m.double().unsqueeze(-1)).flatten(-2)
        # rounded once: half a step of the type, and its subnormal grid
        step = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** (-25 if dtype == torch.float16 else -134)
        assert bool(((got.double() - want).abs() <= step).all())
        # and no value is further off than half a step of its group, what the scale lost by its cut, and that rounding
        off = (x.double() - want).abs().unflatten(-1, (-1, 32))
        limit = s.double() * (0.5 + 16 * torch.finfo(dtype).eps) + 16 * 2.0 ** -24
        assert bool((off <= limit.unsqueeze(-1) + step.unflatten(-1, (-1, 32))).all())
    # the same without the packed keys and values, and onto the inputs
    for kw in (dict(need_kv=False), dict(k_out=k, v_out=v, q_out=q)):
        for c, b in zip((ck, cv), before):
            c.codes.copy_(b[0])
            c.params.copy_(b[1])
        r = paged.rope_paged_write_int4(q, k, v, cos, sin, pos, slots, ck, cv, **kw)
        if "need_kv" in kw:
            check_write(paged, kt, v, ck, cv, slots, [(a.clone(), b.clone()) for a, b in before], ps)
            assert r[1] is None and r[2] is None and torch.equal(r[0], want_q)
        else:
            assert torch.equal(q, want_q) and same(k, got_k) and same(v, got_v)


@pytest.mark.parametrize("dtype", TYPES)
def test_write_awkward_values(paged, dtype):
    """Groups of one value, subnormals, the largest values, borders between codes, what is not finite."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal / 128
    D, rows = 64, []
    ramp = torch.arange(32, dtype=torch.float64)
    for group in (ramp * 0, ramp * 0 - 3, ramp, ramp / 2, -ramp * tiny, ramp * tiny, (ramp - 16) * big / 16, ramp % 2 * big,
                  ramp % 2 * 15, torch.cat([ramp[:16], ramp[:16] + 0.5]).clamp(max=15), ramp * 1e-4 + 7, ramp ** 3 - 500,
                  torch.where(torch.arange(32) == 7, math.nan, 1.0).double(),
                  torch.where(torch.arange(32) == 9, math.inf, 2.0).double(),
                  torch.where(torch.arange(32) == 31, -math.inf, 2.0).double()):
        rows.append(torch.cat([group, torch.linspace(-1, 1, 32, dtype=torch.float64)]))
    gen = torch.Generator().manual_seed(5)
    for e in range(-24, 15, 3):  # many exponents, values on a coarse grid: quotients on borders
        rows.append(torch.randint(-15, 16, (D,), generator=gen).double() * 2.0 ** e)
        rows.append(torch.randn(D, generator=gen, dtype=torch.float64) * 2.0 ** e)
    x = torch.stack(rows).to(dtype).cuda()[:, None]
    T = x.shape[0]
    cos, sin = tables(D)
    pos, slots = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.arange(T, device="cuda").flip(0)
    ck, cv = (new_cache(paged, 8, 8, 1, D, dtype, 7 + i) for i in range(2))
    before = [(c.codes.clone(), c.params.clone()) for c in (ck, cv)]
    _, k, v = paged.rope_paged_write_int4(x, x, x, cos, sin, pos, slots, ck, cv)
    keys = x.clone()  # position 0 turns nothing, but a pair with an infinity or a NaN is not finite after it
    pairs = keys.unflatten(-1, (-1, 2))
    pairs[~torch.isfinite(pairs).all(-1)] = math.nan
    check_write(paged, keys, x, ck, cv, slots, before, 8)
    assert bool(torch.isnan(v[12:15, :, :32]).all()) and bool(torch.isfinite(v[:12]).all())
    assert bool(torch.isnan(k[12:15, :, :32]).all()) and bool(torch.isfinite(k[:12]).all())


def test_write_bad_places(paged):
    """Slots past the cache are skipped and positions clamped, both with bit 7; a skipped token's position sets nothing."""
    from llama import _native

    D, dtype = 64, torch.float16
    q, k, v = rand((3, 2, D), dtype, 1), rand((3, 1, D), dtype, 2), rand((3, 1, D), dtype, 3)
    cos, sin = tables(D, 10)
    ck, cv = (new_cache(paged, 2, 8, 1, D, dtype, 7 + i) for i in range(2))
    codes = ck.codes.clone()
    for pos, slot, bit in (([0, 99, -5], [-1, -1, -1], 0), ([0, 1, 2], [16, 1 << 40, -1], 128)):
        paged.rope_paged_write_int4(q, k, v, cos, sin, i32(pos), torch.tensor(slot, device="cuda"), ck, cv)
        assert _native.device_errors() == bit
        assert torch.equal(ck.codes, codes)
    paged.rope_paged_write_int4(q, k, v, cos, sin, i32([10, -1, 3]), torch.arange(3, device="cuda"), ck, cv)
    assert _native.device_errors() == 128
    want, _, _ = quantized(turned(k, cos, sin, i32([9, 0, 3])))
    assert torch.equal(paged.unpack_codes(ck.codes[0, :3]), want)


def layout(paged, shape, H, Hkv, D, ps, dtype, seed=0, by_head=True):
    """A cache, tables and queries for [(tokens the cache holds with the new ones, new tokens)]; the keys and values."""
    rng = random.Random(seed)
    need = [-(-L // ps) for L, _ in shape]
    pages, width = sum(need) + 3, max(need + [1]) + 1
    order = rng.sample(range(pages), pages)
    table = torch.full((len(shape), width), 1 << 30, dtype=torch.int32)  # entries past a request's pages are never used
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    ck, cv = (new_cache(paged, pages, ps, Hkv, D, dtype, seed + 1 + i, by_head) for i in range(2))
    for c in (ck, cv):  # pages of nobody and rows past the end hold what must not be seen
        for p in order[at:]:
            c.params[p] = math.nan
        for b, (L, _) in enumerate(shape):
            if L % ps:
                c.params[table[b, need[b] - 1].long(), L % ps:] = math.nan
    table = table.cuda()
    rows = []
    for c in (ck, cv):
        values = c.values()
        rows.append([values[table[b, :n].long()].flatten(0, 1)[:L] for b, (n, (L, _)) in enumerate(zip(need, shape))])
    q = rand((sum(n for _, n in shape), H, D), dtype, seed + 9)
    cu, lens = i32(cumulative([n for _, n in shape])), i32([L for L, _ in shape])
    return q, ck, cv, table, lens, cu, max([n for _, n in shape] + [0]), rows


HEADS = [(32, 8, 64), (8, 2, 128), (7, 1, 128), (6, 2, 32), (12, 4, 96), (4, 4, 64), (40, 8, 64), (128, 1, 64), (9, 1, 32)]
SHAPES = [[(1, 1)], [(576, 1)], [(17, 1), (0, 0), (5, 5), (300, 2)], [(500, 200), (6, 1)], [(70, 70)], [(3, 5), (0, 2), (40, 1)],
          [(2049, 3), (129, 129), (128, 1)]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("H,Hkv,D", HEADS)
def test_attention(paged, H, Hkv, D, shape, dtype):
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, H, Hkv, D, 16, dtype)
    got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
    check(got, q, keys, values, [n for _, n in shape])


@pytest.mark.parametrize("ps", [8, 32, 128, 1024])
@pytest.mark.parametrize("by_head", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_page_sizes(paged, D, ps, by_head):
    shape = [(1500, 1), (333, 2), (1025, 300), (8, 1)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 8, 2, D, ps, torch.float16, 3, by_head)
    for max_new in (most, 1):  # a claim that is too small picks other kernels
        got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, max_new, scale=0.1)
        check(got, q, keys, values, [n for _, n in shape], 0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 4, 300])
def test_attention_long(paged, n, dtype):
    """A long context: parts of it joined."""
    shape = [(20011, n), (31, 1), (9000, 1)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 4, 1, 128, 64, dtype, 5)
    got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
    some = sorted({0, n // 2, n - 1})
    for i in some:
        L = shape[0][0] - n + i + 1
        check(got[i:i + 1], q[i:i + 1], [keys[0][:L]], [values[0][:L]], [1])
    check(got[n:], q[n:], keys[1:], values[1:], [1, 1])


def test_attention_many_requests(paged):
    shape = [((37 * b) % 400 + 1, 1) for b in range(300)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 8, 2, 64, 16, torch.float16, 6)
    check(paged.paged_attention_int4(q, ck, cv, table, lens, cu, most), q, keys, values, [1] * 300)


@pytest.mark.parametrize("n", [1, 4, 60])
def test_attention_entries_outside_the_cache(paged, n):
    """They read as zero keys and values."""
    shape = [(200, n), (100, 1)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 8, 2, 64, 16, torch.bfloat16, 8)
    table[0, 3], table[0, 7], table[1, 0] = -1, ck.codes.shape[0], 2 ** 31 - 1
    for rows in (keys, values):
        rows[0][48:64] = 0
        rows[0][112:128] = 0
        rows[1][:16] = 0
    check(paged.paged_attention_int4(q, ck, cv, table, lens, cu, most), q, keys, values, [n, 1])
    # no page at all
    empty = [paged.Int4Pages(c.codes[:0], c.params[:0]) for c in (ck, cv)]
    got = paged.paged_attention_int4(q, *empty, table, lens, cu, most)
    assert bool((got == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [3, 50, 200])
def test_attention_groups_that_are_not_finite(paged, n, D, dtype):
    """A group's NaN reaches the queries that see its key, in that group's dims (a key's: in all), and no others."""
    shape = [(n + 30, n), (45, 1)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 4, 2, D, 16, dtype, 11)
    clean = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
    for what, key in itertools.product(("value", "key"), (30 + n - 1, 30 + n // 2)):
        cache = cv if what == "value" else ck
        at = (table[0, key // 16].long(), key % 16, 1, 1)
        for bad in ((math.nan, math.nan), (1.0, math.inf), (math.inf, 0.0)):
            saved = cache.params[at].clone()
            cache.params[at] = torch.tensor(bad, dtype=dtype, device="cuda")
            got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
            cache.params[at] = saved
            hit = torch.zeros_like(clean, dtype=torch.bool)
            dims = slice(32, 64) if what == "value" else slice(None)
            hit[key - 30:n, 2:, dims] = True  # KV head 1's queries
            assert bool((~torch.isfinite(got[hit])).all()), (what, key, bad)
            assert bool(torch.isfinite(got[~hit]).all()), (what, key, bad)
            check(torch.where(hit, 0, got)[:, :2], q[:, :2], [r[:, :1] for r in keys], [r[:, :1] for r in values], [n, 1])


def test_attention_odd_places(paged):
    """Params off the alignment of a whole row, strides of other tensors, an output's rows behind the last sequence."""
    shape = [(150, 1), (40, 9), (64, 1)]
    for D in (64, 128):
        q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 4, 2, D, 16, torch.float16, 13)
        pages, ps, Hkv, G, _ = ck.params.shape
        moved = []
        for c in (ck, cv):
            room = torch.zeros(pages * ps * Hkv * (2 * G + 2) + 2, dtype=torch.float16, device="cuda")[2:]
            params = room.view(pages, ps, Hkv, 2 * G + 2)[..., :2 * G].unflatten(-1, (G, 2))
            params.copy_(c.params)
            codes = torch.zeros(pages, ps, Hkv, D // 2 + 16, dtype=torch.uint8, device="cuda")[..., :D // 2]
            codes.copy_(c.codes)
            moved.append(paged.Int4Pages(codes, params))
        T = q.shape[0]
        wide = torch.zeros(T + 4, 4, D + 8, dtype=torch.float16, device="cuda")
        wide[:T, :, :D] = q
        out = torch.full((T + 4, 4, D), 7.0, dtype=torch.float16, device="cuda")
        got = paged.paged_attention_int4(wide[..., :D], *moved, table, lens, cu, most, out=out)
        assert got.data_ptr() == out.data_ptr() and bool((out[T:] == 7).all())
        check(out[:T], q, keys, values, [n for _, n in shape])


def test_attention_captured_and_on_streams(paged):
    """Two captured graphs and eager calls on other streams at once; the lengths grow between the replays."""
    shapes = [[(5000, 1), (70, 1)], [(900, 130), (33, 1)]]
    made = [layout(paged, s, 8, 2, 64, 16, torch.float16, 20 + i) for i, s in enumerate(shapes)]
    graphs, outs = [], []
    for q, ck, cv, table, lens, cu, most, _ in made:
        paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged.paged_attention_int4(q, ck, cv, table, lens, cu, most))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    eager = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for (q, ck, cv, table, lens, cu, most, _), s in zip(made, streams[2:]):
            with torch.cuda.stream(s):
                eager.append(paged.paged_attention_int4(q, ck, cv, table, lens, cu, most))
    torch.cuda.synchronize()
    for i, (q, ck, cv, table, lens, cu, most, (keys, values)) in enumerate(made):
        check(outs[i], q, keys, values, [n for _, n in shapes[i]])
        for e in eager[i::2]:
            assert torch.equal(e, outs[i])
    lens = made[0][4]
    lens.sub_(7)
    graphs[0].replay()
    torch.cuda.synchronize()
    q, keys, values = made[0][0], *made[0][7]
    check(outs[0], q, [k[:-7] for k in keys], [v[:-7] for v in values], [1, 1])


def test_refusals(paged):
    D, dtype = 64, torch.float16
    q, k, v = rand((3, 4, D), dtype, 1), rand((3, 2, D), dtype, 2), rand((3, 2, D), dtype, 3)
    cos, sin = tables(D, 16)
    ck, cv = (new_cache(paged, 4, 16, 2, D, dtype, 7 + i) for i in range(2))
    pos, slots = i32([0, 1, 2]), torch.arange(3, device="cuda")
    table, lens, cu = i32([[0, 1]]), i32([20]), i32([0, 3])

    def write(**kw):
        a = dict(q=q, k=k, v=v, cos=cos, sin=sin, positions=pos, slots=slots, cache_k=ck, cache_v=cv)
        return paged.rope_paged_write_int4(**{**a, **kw})

    def attend(**kw):
        a = dict(q=q, cache_k=ck, cache_v=cv, block_tables=table, kv_lens=lens, cu_seqlens=cu, max_new=3)
        return paged.paged_attention_int4(**{**a, **kw})

    write(), attend()
    pages = paged.Int4Pages
    odd = ck.codes.flatten()
    for call in (write, attend):
        for cache in (ck.codes, (ck.codes,), pages(ck.codes.short(), ck.params), pages(ck.codes[..., :16], ck.params),
                      pages(ck.codes, ck.params.bfloat16()), pages(ck.codes, ck.params[:, :, :, :1]), pages(ck.codes[:3], ck.params),
                      pages(ck.codes.cpu(), ck.params), pages(ck.codes, None), pages(ck.codes[:, :8], ck.params[:, :8]),
                      pages(ck.codes[:, :, :1], ck.params[:, :, :1]),
                      pages(odd.as_strided((3, 16, 2, 32), (1024, 32, 512, 1), 8), ck.params[:3])):
            with pytest.raises((RuntimeError, TypeError)):
                call(cache_k=cache)
    with pytest.raises(RuntimeError, match="overlap"):
        write(q_out=k.new_empty(3, 4, D), k_out=v)
    with pytest.raises(RuntimeError, match="overlap"):
        write(v_out=k)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(out=q)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(out=ck.codes.transpose(1, 2).flatten()[:1536].view(dtype).view(3, 4, D))
    with pytest.raises(RuntimeError, match="multiple of 32"):
        attend(q=rand((3, 4, 48), dtype, 1))
    with pytest.raises(RuntimeError, match="requires grad"):
        attend(q=q.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        write(k=k.bfloat16())
