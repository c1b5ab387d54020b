"""Limits of the paged serving path on the GPU: what is refused, and that a refusal is the only thing that happens."""
import pytest
import torch

from test_paged_gpu import i32, paged, rand, tiny_model  # noqa: F401 (paged: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,max_len", [(16, 20), (16, 16), (8, 1), (1024, 37), (32, 95)])
def test_no_request_grows_past_max_len(paged, page, max_len):  # noqa: F811
    """max_len that is no multiple of the page size: the last page's other rows are never given out."""
    cache = paged.PagedKVCache(1, 40, page, 1, 8, max_requests=3, max_len=max_len)
    step = cache.append(i32([max_len, max_len + 1, max_len - 1]), 3 * max_len)
    assert step.granted.tolist() == [True, False, True]
    assert cache.kv_lens.tolist() == [max_len, 0, max_len - 1]
    assert bool((step.slots[max_len:2 * max_len + 1] == -1).all()) and bool((step.slots[2 * max_len + 1:] >= 0).all())
    free = int(cache.n_free)
    step = cache.append(i32([1, 1, 1]), 3)
    assert step.granted.tolist() == [False, True, True]
    assert cache.kv_lens.tolist() == [max_len, 1, max_len]
    step = cache.append(i32([1, 0, 1]), 2)
    assert step.granted.tolist() == [False, True, False]
    assert cache.kv_lens.tolist() == [max_len, 1, max_len] and int(cache.n_free) >= free - 2


def test_append_takes_a_limit(paged):  # noqa: F811
    tables = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    args = (i32([0, 5, 9]), i32([10, 5, 2]), tables, i32([0, 1, 2, 3, 4, 5]), i32([6]), 8, 17)
    step = paged.paged_append(*args, max_len=10)
    assert step.granted.tolist() == [True, True, False] and step.n_free.tolist() == [3]
    assert step.kv_lens.tolist() == [10, 10, 9]
    assert paged.paged_append(*args, max_len=11).granted.tolist() == [True, True, True]
    assert paged.paged_append(*args).granted.tolist() == [True, True, True]
    assert paged.paged_append(*args, max_len=1 << 62).granted.tolist() == [True, True, True]
    assert paged.paged_append(*args, max_len=0).granted.tolist() == [False, False, False]
    for bad in (-1, 1.5):
        with pytest.raises(RuntimeError):
            paged.paged_append(*args, max_len=bad)


def test_the_model_s_positions_stay_inside_its_rope_table(paged):  # noqa: F811
    """A cache as long as the RoPE table, which ends inside a page: tokens past it are refused, not clamped (the error
    words are looked at after every test)."""
    model = tiny_model()
    rows = model.freqs_cis.shape[0]
    cache = model.paged_cache(num_pages=2, page_size=1024, max_requests=1, max_len=rows)
    tokens = torch.randint(0, 500, (rows,), device="cuda")
    step = cache.append(i32([rows]), rows)
    assert step.granted.tolist() == [True]
    assert bool(torch.isfinite(model.forward_paged(tokens, step, cache, rows)).all())
    step = cache.append(i32([1]), 1)
    assert step.granted.tolist() == [False] and step.slots.tolist() == [-1]
    assert cache.kv_lens.tolist() == [rows]


def test_refused_tokens_set_no_error(paged):  # noqa: F811
    """Refused requests through the append and the RoPE write: one at the end of its table and of the RoPE table, one of
    a negative length.  Their tokens have positions outside the table and are skipped; nothing is reported."""
    from llama import _native

    page, H, Hkv, d, rows = 16, 4, 2, 64, 32
    kv, new, T = i32([rows, -5, 3]), i32([2, 2, 1]), 5
    tables = i32([[0, 1], [2, 3], [4, 5]])
    step = paged.paged_append(kv, new, tables, i32([6, 7]), i32([2]), page, T)
    assert step.granted.tolist() == [False, False, True] and step.slots.tolist() == [-1, -1, -1, -1, 4 * page + 3]
    q, k, v = rand((T, H, d), torch.float16, 1), rand((T, Hkv, d), torch.float16, 2), rand((T, Hkv, d), torch.float16, 3)
    angle = torch.rand(rows, d // 2, device="cuda")
    ck = torch.zeros(8, page, Hkv, d, dtype=torch.float16, device="cuda")
    cv = torch.zeros_like(ck)
    paged.rope_paged_write(q, k, v, angle.cos(), angle.sin(), step.positions, step.slots, ck, cv)
    assert _native.device_errors() == 0
    assert torch.equal(cv[4, 3], v[4]) and int((cv != 0).any(-1).sum()) == Hkv
    # a bad position that would be written is reported
    bad = step.positions.clone()
    bad[4] = rows
    paged.rope_paged_write(q, k, v, angle.cos(), angle.sin(), bad, step.slots, ck, cv)
    assert _native.device_errors() == 128


def prompts_in(model, cache, lens, seed):
    """Random prompts of the given lengths (0: the request stays idle) through the cache; the requests' next tokens."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(0, 500, (sum(lens),), device="cuda", generator=gen)
    step = cache.append(i32(lens), sum(lens))
    assert bool(step.granted.all())
    return model.forward_paged(tokens, step, cache, max(lens), whole_prompts=True).argmax(-1)


def eager_steps(model, cache, tok, active, steps):
    """Tokens of a loop over the active requests that stops feeding a request once it is refused."""
    tok, history = tok.clone(), []
    for _ in range(steps):
        step = cache.append(i32([int(a) for a in active]), sum(active))
        rows = [r for r, a in enumerate(active) if a]
        best = model.forward_paged(tok[rows], step, cache, 1).argmax(-1)
        for r in rows:
            if bool(step.granted[r]):
                tok[r] = best[r]
        history.append(tok.clone())
    return torch.stack(history)


def test_captured_steps_say_which_requests_were_refused(paged):  # noqa: F811
    """Pages run out, and a request reaches max_len, in the middle of the replays: the refused request keeps its token and
    length and granted says so; the others go on as in an eager loop."""
    from llama.generation import PagedDecodeGraph

    model = tiny_model(seed=1)
    lens, steps = [5, 17, 8], 12
    with torch.no_grad():
        caches = [model.paged_cache(num_pages=6, page_size=8, max_requests=3, max_len=24) for _ in range(2)]
        first = [prompts_in(model, c, lens, 2) for c in caches]
        assert torch.equal(*first)
        want = eager_steps(model, caches[0], first[0], [True] * 3, steps)
        graph = PagedDecodeGraph(model, caches[1], first[1])
        assert graph.granted.tolist() == [True] * 3
        got, granted = [], []
        for _ in range(steps):
            graph.replay()
            got.append(graph.tok.clone())
            granted.append(graph.granted.tolist())
    assert torch.equal(torch.stack(got), want)
    assert caches[1].kv_lens.tolist() == caches[0].kv_lens.tolist()
    for r, n in enumerate(lens):
        served = int(caches[1].kv_lens[r]) - n
        assert [g[r] for g in granted] == [i < served for i in range(steps)]
        assert all(int(t[r]) == int(got[served - 1][r]) for t in got[served:])
    assert not all(granted[-1]) and caches[1].kv_lens.max() <= 24


def test_captured_steps_leave_idle_requests_idle(paged):  # noqa: F811
    from llama.generation import PagedDecodeGraph

    model = tiny_model(seed=2)
    lens = [0, 9, 0, 30, 1]
    with torch.no_grad():
        caches = [model.paged_cache(num_pages=20, page_size=8, max_requests=5) for _ in range(2)]
        first = [prompts_in(model, c, lens, 3) for c in caches]
        want = eager_steps(model, caches[0], first[0], [n > 0 for n in lens], 6)
        graph = PagedDecodeGraph(model, caches[1], first[1])
        for i in range(6):
            graph.replay()
            assert torch.equal(graph.tok, want[i])
        assert caches[1].kv_lens.tolist() == [0, 15, 0, 36, 7] and bool(graph.granted.all())
        with pytest.raises(ValueError):
            PagedDecodeGraph(model, model.paged_cache(num_pages=4, page_size=8, max_requests=2), first[0][:2])


def test_outputs_that_overlap_their_inputs_are_refused(paged):  # noqa: F811
    from test_paged_limits_cpu import calls

    T, H, Hkv, d, page = 4, 4, 2, 64, 16
    dtype = torch.float16
    pool = torch.zeros(1 << 16, dtype=dtype, device="cuda")

    def at(start, shape):
        n = 1
        for x in shape:
            n *= x
        return pool[start:start + n].view(shape)

    Q, K, C = (T, H, d), (T, Hkv, d), (2, page, Hkv, d)
    q, k, cache = at(8192, Q), at(16384, K), at(24576, C)
    a, table = calls(paged, q, k, cache)
    prompt, over_cache, rope = table
    v, cache_v = at(32768, K), at(40960, C)
    bad = [(prompt, dict(out=at(8192 + 8, Q))), (prompt, dict(out=at(8192 - 8, Q))), (prompt, dict(out=q)),
           (prompt, dict(out=at(16384 + K[0] * Hkv * d - 8, Q))), (prompt, dict(out=at(16384 - 8, Q))),
           (prompt, dict(v=v, out=at(32768 + 64, Q))), (over_cache, dict(out=at(24576 + 1024, Q))),
           (over_cache, dict(cache_v=cache_v, out=at(40960 + 2048, Q))), (over_cache, dict(out=at(8192 + 64, Q))),
           (rope, dict(q_out=at(8192 + 8, Q))), (rope, dict(q_out=at(16384, Q))), (rope, dict(k_out=at(8192, K))),
           (rope, dict(v=v, k_out=v)), (rope, dict(q_out=at(24576, Q))), (rope, dict(cache_v=cache_v, k_out=at(40960, K))),
           (rope, dict(q_out=at(49152, Q), k_out=at(49152 + 64, K))),
           # the same memory in another order
           (rope, dict(q_out=at(8192, (H, T, d)).transpose(0, 1)))]
    for i, (call, over) in enumerate(bad):
        with pytest.raises(RuntimeError, match="overlap"):
            call(**over)
            pytest.fail(f"call {i} was not refused")
    # what touches without overlapping, in place, and parts of one wide row
    prompt(out=at(8192 + T * H * d, Q))
    prompt(out=at(16384 - T * H * d, Q))
    rope(q_out=q, k_out=k)
    rope(q_out=q)
    wide = rand((T, (2 * H + 3 * Hkv) * d), dtype, 1)
    parts, start = [], 0
    for heads in (H, Hkv, Hkv, H, Hkv):
        parts.append(wide[:, start:start + heads * d].view(T, heads, d))
        start += heads * d
    prompt(q=parts[0], k=parts[1], v=parts[2], out=parts[3])
    rope(q=parts[0], k=parts[1], v=parts[2], q_out=parts[3], k_out=parts[4])
    rope(q=parts[0], k=parts[1], v=parts[2], q_out=parts[0], k_out=parts[1])
    # heads interleaved in pairs of rows: q and the output take turns
    turns = rand((T, H, 2, d), dtype, 2)
    prompt(q=turns[:, :, 0], out=turns[:, :, 1])
    torch.cuda.synchronize()


def test_claims_whose_products_pass_64_bits(paged):  # noqa: F811
    """A longest sequence or a table width near 2^62 counts as a long one; it does not wrap to a short one."""
    import ctypes

    from llama import _native as native
    from test_paged_limits_cpu import attention_args

    def need(**over):
        return native.lib().li4_attention_workspace_bytes(ctypes.byref(attention_args(native, **over)))

    for kv_lens in (None, 16):
        long = need(kv_lens=kv_lens, table_width=128, max_queries=1 << 28)
        assert long > need(kv_lens=kv_lens, table_width=128, max_queries=4)
        for claim in (1 << 30, 1 << 61, 1 << 62, (1 << 63) - 1):
            assert need(kv_lens=kv_lens, table_width=128, max_queries=claim) == long
    wide = need(max_queries=100, table_width=1 << 26)
    for width in (1 << 59, 1 << 60, (1 << 63) - 1):
        assert need(max_queries=100, table_width=width) == wide
    q, k = rand((70, 4, 64), torch.float16, 1), rand((70, 2, 64), torch.float16, 2)
    cu = i32([0, 70])
    want = paged.prompt_attention(q, k, k, cu, 70)
    for claim in (1 << 61, 1 << 62, (1 << 63) - 1):
        assert torch.equal(paged.prompt_attention(q, k, k, cu, claim), want)
