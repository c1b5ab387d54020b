"""paged_fork on the GPU against a list of pages per request."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    import build

    build.build()
    from llama import paged

    return paged


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Lists:
    """The definition: which pages each request holds, the free stack, what each page's rows are."""

    def __init__(self, lens, tables, stack, ps, width, content):
        self.lens, self.tables, self.stack, self.ps, self.width = list(lens), [list(t) for t in tables], list(stack), ps, width
        self.content = list(content)

    def fork(self, parents):
        old = [(n, list(t)) for n, t in zip(self.lens, self.tables)]
        top, asked, granted, copies = len(self.stack), 0, [], []
        for r, p in enumerate(parents):
            if p == r or p == -1:
                granted.append(True)
                if p == -1:
                    self.lens[r], self.tables[r] = 0, []
                continue
            if not 0 <= p < len(parents) or not 0 <= old[p][0] <= self.width * self.ps:
                granted.append(False)
                continue
            n, pages = old[p]
            part = n % self.ps != 0
            asked += part
            granted.append(not part or asked <= top)
            if granted[-1]:
                self.lens[r], self.tables[r] = n, list(pages)
                if part:
                    self.tables[r][-1] = self.stack.pop()
                    copies.append((pages[-1], self.tables[r][-1]))
        before = list(self.content)
        for a, b in copies:
            self.content[b] = before[a]
        held = {p for t in self.tables for p in t}
        for _, pages in old:
            for p in pages:
                if p not in held and p not in self.stack:
                    self.stack.append(p)
        return granted


def make(rng, B, ps, width, spare, shared=True):
    """Requests with some shared leading pages, a shuffled stack."""
    lens = [rng.choice([0, rng.randrange(1, width * ps + 1), ps * rng.randrange(0, width + 1)]) for _ in range(B)]
    tables, number = [], 0
    for r, n in enumerate(lens):
        pages = -(-n // ps)
        own = []
        if shared and r and rng.random() < 0.5:
            other = rng.randrange(r)
            own = tables[other][:rng.randrange(0, min(lens[other], n) // ps + 1)]
        fresh = pages - len(own)
        tables.append(own + list(range(number, number + fresh)))
        number += fresh
    pool = number + spare
    names = rng.sample(range(pool), pool)
    return lens, [[names[p] for p in t] for t in tables], [names[p] for p in range(number, pool)], pool


def run(paged, rng, B, ps, width, spare, rounds=3, parents_of=None, pools=True):
    lens, tables, stack, pool = make(rng, B, ps, width, spare)
    content = torch.randint(0, 1 << 15, (pool,), device="cuda", dtype=torch.int16)
    half = content.view(torch.float16)[:, None, None, None].expand(pool, ps, 2, 8).contiguous()
    by_head = content[:, None, None, None].expand(pool, 3, ps, 4).contiguous().transpose(1, 2)
    gapped = content.view(torch.uint8).view(pool, 2)[:, :1].repeat(1, 64)[:, None].expand(pool, 2, 64).contiguous()[:, 0]
    all_pools = [half, by_head, gapped] if pools else []
    oracle = Lists(lens, tables, stack, ps, width, content.tolist())
    kv = i32(lens)
    bt = torch.full((B, width + 2), -7, dtype=torch.int32, device="cuda")[:, :width]
    for r, t in enumerate(tables):
        bt[r, :len(t)] = i32(t)
    free = torch.full((pool,), -9, dtype=torch.int32, device="cuda")
    free[:len(stack)] = i32(stack)
    n_free = i32([len(stack)])
    for _ in range(rounds):
        parents = parents_of(rng, B) if parents_of else [rng.choice([r, rng.randrange(B), -1]) if rng.random() < 0.9 else r for r in range(B)]
        before_free, height = free.clone(), n_free.item()
        granted = oracle.fork(parents)
        got = paged.paged_fork(kv, bt, free, n_free, i32(parents), ps, all_pools, kv_lens_out=kv, n_free_out=n_free)
        assert got.granted.tolist() == granted
        assert kv.tolist() == oracle.lens and got.kv_lens.data_ptr() == kv.data_ptr()
        assert n_free.item() == len(oracle.stack)
        assert free[:len(oracle.stack)].tolist() == oracle.stack
        above = max(height, len(oracle.stack))
        assert torch.equal(free[above:], before_free[above:])
        for r, t in enumerate(oracle.tables):
            assert bt[r, :len(t)].tolist() == t, r
        held = sorted({p for t in oracle.tables for p in t})
        if pools and held:
            want = torch.tensor(oracle.content, dtype=torch.int16, device="cuda")[held]
            assert torch.equal(half.view(torch.int16)[held], want[:, None, None, None].expand(-1, ps, 2, 8))
            assert torch.equal(by_head[held], want[:, None, None, None].expand(-1, ps, 3, 4))
            assert torch.equal(gapped[held], want.view(torch.uint8).view(-1, 2)[:, :1].expand(-1, 64))


@pytest.mark.parametrize("B,ps,width,spare", [(1, 8, 3, 2), (2, 16, 4, 5), (7, 8, 5, 3), (33, 16, 9, 40), (64, 8, 40, 64),
                                              (300, 32, 6, 300), (1000, 8, 17, 400), (513, 16, 1, 3)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_fork(paged, B, ps, width, spare, seed):
    run(paged, random.Random(seed), B, ps, width, spare)


def test_fork_many_requests(paged):
    run(paged, random.Random(9), 8192, 8, 5, 3000, rounds=2)


def test_fork_all_onto_one_and_places_changed(paged):
    run(paged, random.Random(4), 40, 16, 8, 200, parents_of=lambda rng, B: [5] * B)
    run(paged, random.Random(5), 40, 16, 8, 200, parents_of=lambda rng, B: [(r + 1) % B for r in range(B)])
    run(paged, random.Random(6), 40, 16, 8, 200, parents_of=lambda rng, B: [-1] * B)
    run(paged, random.Random(7), 40, 16, 8, 0, parents_of=lambda rng, B: [(r * 7) % B for r in range(B)])
    run(paged, random.Random(8), 12, 16, 8, 9, parents_of=lambda rng, B: [rng.choice([-2, 12, 1 << 30, -(1 << 31), r]) for r in range(B)])
    run(paged, random.Random(8), 12, 16, 8, 9, pools=False)


def test_fork_new_outputs_and_odd_lengths(paged):
    """kv_lens and n_free stay without outputs for them; lengths that fit no table are refused as parents."""
    kv, bt = i32([20, -3, 1000, 9]), i32([[0, 1], [2, 3], [4, 5], [6, 7]])
    free, n_free = i32([10, 11, 12] + [0] * 10), i32([3])
    got = paged.paged_fork(kv, bt, free, n_free, i32([0, 0, 1, 2]), 16)
    assert kv.tolist() == [20, -3, 1000, 9] and n_free.item() == 3
    assert got.granted.tolist() == [True, True, False, False]
    assert got.kv_lens.tolist() == [20, 20, 1000, 9]
    assert got.n_free.item() == 2 and bt.tolist() == [[0, 1], [0, 12], [4, 5], [6, 7]]
    # a length past the table holds what the table has; its pages come back when it ends
    got = paged.paged_fork(got.kv_lens, bt, free, got.n_free, i32([0, 1, -1, 3]), 16)
    assert got.kv_lens.tolist() == [20, 20, 0, 9]
    assert free[:got.n_free.item()].tolist() == [10, 11, 4, 5]


def test_fork_entries_that_are_no_page(paged):
    kv, bt = i32([20, 0, 0]), i32([[-5, 99], [0, 0], [0, 0]])
    free, n_free = i32([1, 2, 3, 0]), i32([3])
    pool = torch.arange(4, device="cuda", dtype=torch.int32)[:, None].repeat(1, 4)
    got = paged.paged_fork(kv, bt, free, n_free, i32([-1, 0, 1]), 16, [pool])
    assert got.kv_lens.tolist() == [0, 20, 0] and got.n_free.item() == 2
    assert bt[1].tolist() == [-5, 3] and free[:2].tolist() == [1, 2]
    assert torch.equal(pool, torch.arange(4, device="cuda", dtype=torch.int32)[:, None].repeat(1, 4))


def test_fork_captured(paged):
    """A captured step of a search, replayed: the same as eager calls on a copy."""
    rng = random.Random(3)
    lens, tables, stack, pool = make(rng, 16, 8, 6, 64, shared=False)
    made = []
    for _ in range(2):
        bt = torch.zeros(16, 6, dtype=torch.int32, device="cuda")
        for r, t in enumerate(tables):
            bt[r, :len(t)] = i32(t)
        free = torch.zeros(pool, dtype=torch.int32, device="cuda")
        free[:len(stack)] = i32(stack)
        made.append([i32(lens), bt, free, i32([len(stack)]), torch.arange(pool * 16, device="cuda", dtype=torch.float32).view(pool, 16)])
    parents = i32(range(16))

    def step(kv, bt, free, n_free, data):
        return paged.paged_fork(kv, bt, free, n_free, parents, 8, [data], kv_lens_out=kv, n_free_out=n_free).granted

    step(*made[0]), step(*made[1])  # (parents are the requests themselves: nothing changes)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        granted = step(*made[0])
    for i in range(6):
        parents.copy_(i32([rng.randrange(16) for _ in range(16)]))
        g.replay()
        want = step(*made[1])
        assert torch.equal(granted, want)
        for a, b in zip(*made):
            assert torch.equal(a, b)


def test_cache_fork_append_release(paged):
    """PagedKVCache over a life of requests: after everything ends every page is free, once."""
    rng = random.Random(11)
    for bits in (16, 4):
        cache = paged.PagedKVCache(2, 120, 8, 2, 64, max_requests=10, max_len=80, bits=bits)
        for _ in range(25):
            new = [rng.choice([0, 0, 1, 5, 9]) for _ in range(10)]
            cache.append(i32(new), sum(new))
            cache.fork(i32([rng.choice([r, r, rng.randrange(10), -1]) for r in range(10)]))
            lens, tables = cache.kv_lens.tolist(), cache.block_tables.tolist()
            held = [t[:-(-n // 8)] for n, t in zip(lens, tables)]
            free = cache.free_pages[:cache.n_free.item()].tolist()
            used = {p for t in held for p in t}
            assert len(set(free)) == len(free) and not used & set(free) and len(used) + len(free) == 120
            last = [t[-1] for n, t in zip(lens, held) if n % 8]  # pages that requests append to are shared by none
            for p in last:
                assert sum(t.count(p) for t in held) == 1
        cache.release(torch.ones(10, dtype=torch.bool, device="cuda"))
        assert cache.n_free.item() == 120 and sorted(cache.free_pages.tolist()) == list(range(120))


@pytest.mark.parametrize("bits", [16, 4])
def test_cache_without_pages(paged, bits):
    """Nothing is granted, and ending requests that hold nothing is no error."""
    cache = paged.PagedKVCache(1, 0, 8, 2, 32, max_requests=3, max_len=16, bits=bits)
    assert not cache.append(i32([1, 0, 2]), 3).granted[0]
    cache.release(torch.ones(3, dtype=torch.bool, device="cuda"))
    assert cache.fork(i32([1, 1, -1])).tolist() == [True] * 3
    assert cache.n_free.item() == 0 and cache.kv_lens.tolist() == [0, 0, 0]


def test_cache_whose_tensors_are_replaced(paged):
    """fork copies in the tensors that the cache holds when it is called."""
    cache = paged.PagedKVCache(1, 4, 8, 1, 32, max_requests=2, max_len=16)
    cache.append(i32([3, 0]), 3)
    cache.k[0] = torch.full_like(cache.k[0], 2.0)
    cache.k[0][cache.block_tables[0, 0].long()] = 5.0
    cache.fork(i32([0, 0]))
    assert (cache.k[0][cache.block_tables[1, 0].long()] == 5.0).all()
    assert (cache.k[0] == 5.0).sum().item() == 2 * 8 * 32


def test_refusals(paged):
    kv, bt, free, n_free, parents = i32([1, 2]), i32([[0], [1]]), i32([2, 3, 0, 0]), i32([2]), i32([0, 0])
    pool = torch.zeros(4, 16, device="cuda")

    def fork(**kw):
        a = dict(kv_lens=kv, block_tables=bt, free_pages=free, n_free=n_free, parents=parents, page_size=8, pools=[pool])
        return paged.paged_fork(**{**a, **kw})

    for kw in (dict(page_size=12), dict(parents=parents.long()), dict(parents=parents[:1]), dict(kv_lens=kv.cpu()), dict(pools=pool),
               dict(pools=[pool[:3]]), dict(pools=[pool[:, ::2]]), dict(pools=[pool[:, :3]]), dict(pools=[torch.zeros(4, 4, 2, device="cuda")[:, :2, :1]]),
               dict(pools=[pool.cpu()]), dict(pools=[None]), dict(n_free=i32([1, 2])), dict(block_tables=bt[:1]), dict(pools=7),
               dict(pools=[pool[:1].expand(4, 16)]), dict(kv_lens_out=kv.long()), dict(pools=[torch.zeros(66, device="cuda")[1:65].view(4, 16)])):
        with pytest.raises((RuntimeError, TypeError)):
            fork(**kw)
    assert fork().granted.tolist() == [True, True]
    none = paged.paged_fork(kv[:0], bt[:0], free, n_free, parents[:0], 8)
    assert none.n_free.item() == n_free.item() and none.granted.numel() == 0
