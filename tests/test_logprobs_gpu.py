"""token_logprobs on the GPU against 64 bits.

Tolerance (u = 2^-24).  t = (x - b) log2(e) carries three roundings, the constant's among them: 3 u |t| absolute; a
2^t the unit's 2^-22 and ln 2 x 3 u |t|.  The base b lies up to 4 below the largest value.  With E = 4 + sum p |ln p'| (p' against
the largest) the sum S is off by
  d = 2^-22 + 3 u E + n u,   n = 8 + V / 4096 + 24 the longest chain of additions (a tile's values, tiles, joins),
relatively, log p by d + 3 u (|x - b| + log S + 4), and the entropy, whose W = sum 2^t t meets the same errors in weights of
|t|, by d (1 + 2 E) + 2 sum p (|ln p'| + 4)^2 3 u + 3 u (log S + E)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def logprobs():
    import build

    build.build()
    from llama import logprobs

    return logprobs


def rows(T, V, dtype, seed, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(T, V, generator=gen, device="cuda") * scale).to(dtype)


def check(logprobs, x, tokens, top):
    V = x.shape[1]
    r = logprobs.token_logprobs(x, tokens, top)
    d = x.double()
    p = torch.log_softmax(d, 1)
    b = d.amax(1)
    away = (b[:, None] - d).clamp(max=1e6)
    weight = p.exp()
    E, E2 = (weight * away).sum(1) + 4, (weight * (away + 4) ** 2).sum(1)
    u = 2.0 ** -24
    off = 2.0 ** -22 + 3 * u * E + (32 + V / 4096) * u
    log_s = torch.logsumexp(d, 1) - b + 4
    if tokens is not None:
        at = tokens.clamp(0, V - 1)[:, None]
        want = p.gather(1, at).view(-1)
        tol = off + 3 * u * (away.gather(1, at).view(-1) + log_s)
        bad = (tokens < 0) | (tokens >= V)
        assert bool(torch.isnan(r.logprobs[bad]).all())
        err = (r.logprobs.double() - want)[~bad].abs()
        fine = (err <= tol[~bad]) | (want[~bad] == r.logprobs[~bad])
        assert bool(fine.all()), float((err / tol[~bad]).max())
    else:
        assert r.logprobs is None
    H = -torch.where(weight > 0, weight * p, 0.0).sum(1)
    tol = off * (1 + 2 * E) + 6 * u * E2 + 3 * u * (log_s + E)
    assert bool(((r.entropy.double() - H).abs() <= tol).all()), float(((r.entropy.double() - H).abs() / tol).max())
    if top == 0:
        assert r.top_tokens is None and r.top_logprobs is None
        return r
    order = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_tokens, order)
    want = p.gather(1, order)
    tol = off[:, None] + 3 * u * (away.gather(1, order) + log_s[:, None])
    # (a difference of the lowest and the largest value, -6.8e38, is -infinity in 32 bits)
    assert bool((((r.top_logprobs.double() - want).abs() <= tol) | (r.top_logprobs == want.float())).all())
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(1, 1), (1, 2), (3, 7), (5, 33), (2, 100), (4, 1000), (3, 2047), (2, 8193), (1, 128256), (7, 32003),
                                 (300, 5001), (40, 128256)])
def test_rows(logprobs, T, V, dtype):
    x = rows(T, V, dtype, T + V)
    tokens = (torch.arange(T, device="cuda") * 7919) % V
    for top in (0, 1, 5, 20, 32):
        if top <= V:
            check(logprobs, x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 4096, 40001])
def test_equal_and_rising_values(logprobs, V, dtype):
    """Values that leave the candidates' room: all equal, rising with the index, of few levels."""
    level = torch.arange(V, device="cuda") % 3
    x = torch.stack([torch.zeros(V, device="cuda"), torch.arange(V, device="cuda") / V * 60.0, level.float(), -level.float(),
                     torch.where(level == 0, -0.0, 0.0), torch.arange(V, 0, -1, device="cuda") / V]).to(dtype)
    tokens = torch.tensor([0, V - 1, V // 2, 1, 2, 0], device="cuda")
    for top in (1, 7, 32):
        check(logprobs, x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_masked_values(logprobs, dtype, low):
    """Few tokens allowed, the others -infinity or the type's lowest value; one allowed; a token that is not."""
    V = 33333
    low = -math.inf if low == "-inf" else torch.finfo(dtype).min
    for allowed in ([5], [0, V - 1], [3, 17, 900, 20000, 20001], list(range(0, V, 100))):
        x = torch.full((3, V), low, device="cuda").to(dtype)
        x[:, allowed] = rows(3, len(allowed), dtype, 3)
        check(logprobs, x, torch.tensor([allowed[0], allowed[-1], 1], device="cuda"), 32)


def test_lowest_everywhere_and_far_apart(logprobs):
    V = 20000
    for dtype in TYPES:
        m = torch.finfo(dtype)
        x = torch.full((2, V), m.min, dtype=dtype, device="cuda")
        x[1, 77] = m.max
        r = check(logprobs, x, torch.tensor([9, 77], device="cuda"), 3)
        assert abs(r.entropy[0].item() - math.log(V)) < 1e-5 and r.entropy[1].item() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(logprobs, dtype):
    """NaN, +infinity and nothing but -infinity: NaN statistics, the likeliest still in order; other rows untouched."""
    V = 9001
    x = rows(6, V, dtype, 5)
    clean = x.clone()
    x[1, 400] = math.nan
    x[2, 8000] = math.inf
    x[3] = -math.inf
    x[4, 1::2] = math.nan
    tokens = torch.tensor([1, 2, 3, 4, 5, 6], device="cuda")
    r = logprobs.token_logprobs(x, tokens, 9)
    for row in (1, 2, 3, 4):
        assert math.isnan(r.logprobs[row].item()) and math.isnan(r.entropy[row].item())
        assert bool(torch.isnan(r.top_logprobs[row]).all())
    want = torch.sort(clean.double(), dim=1, descending=True, stable=True).indices
    assert r.top_tokens[1].tolist() == [400] + [i for i in want[1].tolist() if i != 400][:8]
    assert r.top_tokens[2].tolist() == [8000] + [i for i in want[2].tolist() if i != 8000][:8]
    assert r.top_tokens[3].tolist() == list(range(9))
    assert r.top_tokens[4].tolist() == list(range(1, 18, 2))
    for row in (0, 5):
        check(logprobs, x[row:row + 1], tokens[row:row + 1], 9)


@pytest.mark.parametrize("dtype", TYPES)
def test_places_and_strides(logprobs, dtype):
    """Rows on any boundary of their type, rows apart, rows of no order, tokens outside the vocabulary."""
    room = rows(1, 9 * 1201 + 40, dtype, 8).flatten()
    for start in range(9):
        x = room[start:start + 9 * 1201].view(9, 1201)
        check(logprobs, x[:, :1000], torch.tensor([-1, 0, 999, 1000, 5, -100, 1 << 40, 7, 8], device="cuda"), 6)
    check(logprobs, rows(700, 20, dtype, 9).t(), torch.arange(20, device="cuda"), 4)
    check(logprobs, rows(1, 500, dtype, 9).expand(4, 500), torch.arange(4, device="cuda"), 4)
    r = logprobs.token_logprobs(rows(0, 50, dtype, 1), torch.zeros(0, dtype=torch.long, device="cuda"), 3)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 3)
    r = logprobs.token_logprobs(rows(2, 50, dtype, 1), None, 3, entropy=False)
    assert r.logprobs is None and r.entropy is None and r.top_tokens.shape == (2, 3)


def test_captured_and_on_streams(logprobs):
    x = rows(64, 128256, torch.float32, 3)
    tokens = torch.arange(64, device="cuda")
    want = check(logprobs, x, tokens, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = logprobs.token_logprobs(x, tokens, 8)
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            if i % 3 == 0:
                g.replay()
            else:
                eager.append(logprobs.token_logprobs(x, tokens, 8))
    torch.cuda.synchronize()
    for r in [held] + eager:
        for a, b in zip(r, want):
            assert torch.equal(a, b)
    x.copy_(rows(64, 128256, torch.float32, 4))
    g.replay()
    fresh = logprobs.token_logprobs(x, tokens, 8)
    for a, b in zip(held, fresh):
        assert torch.equal(a, b)


def test_refusals(logprobs):
    x, tokens = rows(2, 50, torch.float16, 1), torch.zeros(2, dtype=torch.long, device="cuda")
    for a in ((x.double(), tokens, 1), (x[0], tokens, 1), (x, tokens.int(), 1), (x, tokens[:1], 1), (x, tokens, 33), (x, tokens, -1),
              (x[:, :5], tokens, 6), (x[:, :0], tokens, 0), (x.cpu(), tokens, 1), (x, tokens.cpu(), 1), (x, tokens, "1"),
              (x.clone().requires_grad_(), tokens, 1)):
        with pytest.raises(RuntimeError):
            logprobs.token_logprobs(*a)
