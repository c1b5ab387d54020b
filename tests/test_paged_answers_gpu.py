"""The 4-bit cache, forked requests and token log probabilities as a serving loop uses them together."""
import math
import random

import pytest
import torch

from test_paged_gpu import Letters, check, i32, paged, rand, tiny_model  # noqa: F401 (paged: the fixture)
from test_paged_int4_gpu import layout, quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads,kv_heads,page", [(4, 1, 16), (8, 4, 8), (2, 1, 64)])
def test_steps_agree_however_a_text_is_cut(paged, heads, kv_heads, page, bits):  # noqa: F811
    """A text in one step, in chunks, token by token, forked on the way: the same keys and values are in the cache (those
    of 4 bits are what whole prompts attend to as well), so the last token's logits agree as two fp16 paths do: within
    1% of their range."""
    model = tiny_model(heads=heads, kv_heads=kv_heads)
    rng = random.Random(2)
    text = [rng.randrange(500) for _ in range(150)]

    def run(cuts, fork_at=None):
        cache = model.paged_cache(num_pages=3 * -(-200 // page) + 4, page_size=page, max_requests=3, bits=bits)
        row, fed = 0, 0
        with torch.no_grad():
            for n in cuts:
                new = [0, 0, 0]
                new[row] = n
                plan = cache.append(i32(new), n)
                tokens = torch.tensor(text[fed:fed + n], device="cuda")
                logits = model.forward_paged(tokens, plan, cache, n, whole_prompts=fed == 0)[row]
                fed += n
                if fork_at is not None and fed >= fork_at and row == 0:  # the rest on another row; its parent goes on elsewhere
                    assert bool(cache.fork(i32([0, -1, 0])).all())
                    other = cache.append(i32([3, 0, 0]), 3)
                    model.forward_paged(torch.tensor([7, 8, 9], device="cuda"), other, cache, 3)
                    row = 2
            cache.release(torch.ones(3, dtype=torch.bool, device="cuda"))
            assert sorted(cache.free_pages[:int(cache.n_free)].tolist()) == list(range(cache.free_pages.numel()))
        return logits

    want = run([150])
    for cuts, fork_at in (([100, 50], None), ([60, 40, 1, 1, 48], None), ([1] * 150, None), ([37, 1, 1, 111], 38), ([64, 86], 64)):
        got = run(cuts, fork_at)
        assert float((got - want).abs().max()) <= 1e-2 * float(want.abs().max()), (cuts, fork_at)
    if bits == 4:  # and not those of the unquantized keys and values, nor far from them
        model.reset_cache()
        with torch.no_grad():
            plain = model(torch.tensor([text], device="cuda"), 0)[0, -1]
        assert float(torch.corrcoef(torch.stack([plain, want]))[0, 1]) > 0.9


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("cuda_graph", [False, True])
def test_generate_samples_with_logprobs(paged, bits, cuda_graph):  # noqa: F811
    """Greedy: the samples of a prompt are its one answer; the log probabilities are those of Llama.forward's logits for
    the text so far, up to twice the 2% that two paths' logits may differ by (16 bits)."""
    model = tiny_model(seed=3)
    prompts, tok = ["a", "some longer prompt " * 5, "of three", "the fourth"], Letters()
    args = (tok, prompts, 9, 0.0, 1.0, "cuda")
    one = model.generate_paged(*args, page_size=8, kv_bits=bits)
    got = model.generate_paged(*args, page_size=8, kv_bits=bits, samples=3, logprobs=4, cuda_graph=cuda_graph)
    assert len(one) == 4 and len(got) == 12 and "logprobs" not in one[0]
    for r, answer in enumerate(got):
        lp = answer["logprobs"]
        gen = [int(x) for x in answer["generation"].split()]
        if not cuda_graph:
            assert answer["generation"] == one[r // 3]["generation"]
        assert lp["tokens"] == gen and len(lp["logprobs"]) == len(lp["entropy"]) == len(lp["top"]) == len(gen)
        ids = tok.encode(prompts[r // 3], True, False)
        with torch.no_grad():
            model.reset_cache()
            logits = model(torch.tensor([ids + gen], device="cuda"), 0)[0].float()
        want = torch.log_softmax(logits.double(), 1)[len(ids) - 1:]
        room = 4e-2 * float(logits.max() - logits.min())
        for i, t in enumerate(gen):
            assert lp["top"][i][0] == (t, lp["logprobs"][i]) and len(lp["top"][i]) == 4
            assert [v for _, v in lp["top"][i]] == sorted((v for _, v in lp["top"][i]), reverse=True)
            assert 0 <= lp["entropy"][i] <= math.log(500) + 1e-5
            if bits == 16:
                assert abs(lp["logprobs"][i] - float(want[i, t])) <= room
    if not cuda_graph:
        sampled = model.generate_paged(tok, prompts, 5, 0.8, 0.9, "cuda", samples=5, kv_bits=bits, logprobs=0)
        assert len(sampled) == 20 and all(t == [] for a in sampled for t in a["logprobs"]["top"])
        with pytest.raises(ValueError):
            model.generate_paged(tok, prompts, 5, 0.0, 0.9, "cuda", samples=0)
        with pytest.raises(ValueError):
            model.generate_paged(tok, prompts, 5, 0.0, 0.9, "cuda", kv_bits=8)


def test_score_paged(paged):  # noqa: F811
    """Within twice the 2% that two paths' logits may differ by; blocks of few rows give the same."""
    model = tiny_model(seed=4)
    texts, tok = ["a", "", "some text that is longer " * 4, "of three"], Letters()
    got = model.score_paged(tok, texts, "cuda", top=2)
    again = model.score_paged(tok, texts, "cuda", top=2, rows=7, page_size=64)
    four = model.score_paged(tok, texts, "cuda", kv_bits=4)
    for text, a, b, c in zip(texts, got, again, four):
        ids = tok.encode(text, True, False)
        assert a["tokens"] == b["tokens"] == c["tokens"] == ids[1:]
        if len(ids) == 1:
            assert a == {"tokens": [], "logprobs": [], "entropy": [], "top": []}
            continue
        with torch.no_grad():
            model.reset_cache()
            logits = model(torch.tensor([ids], device="cuda"), 0)[0].float()
        want = torch.log_softmax(logits.double(), 1)
        room = 4e-2 * float(logits.max() - logits.min())
        for i, t in enumerate(ids[1:]):
            assert abs(a["logprobs"][i] - float(want[i, t])) <= room and abs(b["logprobs"][i] - a["logprobs"][i]) <= room
            assert len(a["top"][i]) == 2 and c["top"][i] == [] and math.isfinite(c["logprobs"][i])


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 90])
def test_attention_scales_and_growing_scores(paged, n, dtype, scale):  # noqa: F811
    """Scores that grow along the keys make the running maximum move all the time."""
    shape = [(1700, n), (130, 1)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 4, 2, 64, 16, dtype, 31)
    grow = torch.linspace(0.05, 3, 1700, device="cuda")
    for j in range(0, 1700, 16):  # a request's keys grow by their parameters
        page = table[0, j // 16].long()
        rows = min(16, 1700 - j)
        ck.params[page, :rows] = (ck.params[page, :rows].float() * grow[j:j + rows, None, None, None]).to(dtype)
    keys = list(keys)
    keys[0] = ck.values()[table[0, :107].long()].flatten(0, 1)[:1700]
    got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most, scale=scale)
    check(got, q, keys, values, [n, 1], scale=scale)


@pytest.mark.parametrize("new", [1, 70])
def test_offsets_past_32_bits(paged, new):  # noqa: F811
    """Pages whose codes start more than 2^32 bytes, and whose params more than 2^30 pairs, into the cache."""
    page, Hkv, D, H = 64, 8, 128, 8
    num = (1 << 32) // (page * Hkv * D // 2) * 4 + 40
    gen = dict(device="cuda")
    params = torch.zeros(num, page, Hkv, D // 32, 2, dtype=torch.float16, **gen)
    codes = torch.zeros(num, page, Hkv, D // 2, dtype=torch.uint8, **gen)
    cache = paged.Int4Pages(codes, params)
    assert params.numel() // 2 > 1 << 30
    n, pages = 150, [num - 1, num - 30, num - 17]
    k, q = rand((n, Hkv, D), torch.float16, 25), rand((n, H, D), torch.float16, 27)
    slots = torch.tensor([pages[j // page] * page + j % page for j in range(n)], device="cuda")
    cos, sin = torch.ones(n, D // 2, device="cuda"), torch.zeros(n, D // 2, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    _, kr, vr = paged.rope_paged_write_int4(q, k, k, cos, sin, pos, slots, cache, cache)  # (turned by nothing: the same rows)
    assert torch.equal(kr, vr)
    want, _, _ = quantized(k)
    assert torch.equal(paged.unpack_codes(codes[num - 1]), want[:page]) and torch.equal(paged.unpack_codes(codes[num - 17, :22]), want[128:])
    got = paged.paged_attention_int4(q[n - new:], cache, cache, i32([pages]), i32([n]), i32([0, new]), new)
    check(got, q[n - new:], [kr], [kr], [new])


@pytest.mark.parametrize("D", [64, 128])
def test_waits_that_run_out_over_a_4_bit_cache(paged, D):  # noqa: F811
    """A few polls are too few: the call ends by itself with bit 8, or is right; the next one with the default limit is
    right, with items that are run again (a NaN value) too."""
    from llama import _native as native

    shape = [(5000, 200), (300, 100), (70, 1)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 8, 2, D, 16, torch.bfloat16, 41)
    out = torch.full((q.shape[0] + 4, 8, D), 7.0, dtype=torch.bfloat16, device="cuda")
    try:
        for bad in (False, True):
            if bad:
                cv.params[table[0, 0].long(), 0, 1, 0] = math.nan
            want = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
            for polls in (1, 2, 5, 20, 100, 400, 2000):
                native.check(native.lib().li4_debug_set_attention_wait_limit(polls), "debug_set_attention_wait_limit")
                for _ in range(2):
                    wide = torch.zeros(q.shape[0] + 4, 8, D, dtype=torch.bfloat16, device="cuda")
                    wide[:q.shape[0]] = q
                    paged.paged_attention_int4(wide, ck, cv, table, lens, cu, most, out=out)
                torch.cuda.synchronize()
                assert native.device_errors() in (0, 256)
                assert bool((out[q.shape[0]:] == 7).all())
            native.check(native.lib().li4_debug_set_attention_wait_limit(0), "debug_set_attention_wait_limit")
            got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
            assert native.device_errors() == 0
        check(got[200:], q[200:], keys[1:], values[1:], [100, 1])
    finally:
        native.check(native.lib().li4_debug_set_attention_wait_limit(0), "debug_set_attention_wait_limit")
        native.device_errors()


def test_every_group_is_not_finite_in_many_items(paged):  # noqa: F811
    """NaN values in every request: all items of a launch are run with care, short ones one after another."""
    shape = [(40 + b % 3, 40) for b in range(200)]
    q, ck, cv, table, lens, cu, most, (keys, values) = layout(paged, shape, 4, 2, 64, 16, torch.float16, 51)
    clean = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
    for b, (L, n) in enumerate(shape):  # the last key: the last query alone sees it
        cv.params[table[b, (L - 1) // 16].long(), (L - 1) % 16, b % 2, b % 2] = math.nan
    got = paged.paged_attention_int4(q, ck, cv, table, lens, cu, most)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for b in range(200):
        hit[40 * b + 39, 2 * (b % 2):2 * (b % 2) + 2, 32 * (b % 2):32 * (b % 2) + 32] = True
    assert bool(torch.isnan(got[hit]).all()) and bool(torch.isfinite(got[~hit]).all())
    assert torch.allclose(got[~hit].float(), clean[~hit].float(), atol=2e-3, rtol=2e-3)
