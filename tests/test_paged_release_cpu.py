"""PagedKVCache.release off the GPU: shared pages, fake tensors, compiled."""
import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from llama.paged import PagedKVCache


def shared_cache(rng, requests, pages, page=8, width=6, device="cpu"):
    """A cache whose requests hold random pages, some of them in common, as forks leave them."""
    c = PagedKVCache(1, pages, page, 1, 32, max_requests=requests, max_len=width * page, device=device)
    order, tables, lens = rng.sample(range(pages), pages), [], []
    for r in range(requests):
        lens.append(rng.choice([0, rng.randrange(1, width * page + 1)]))
        n = -(-lens[-1] // page)
        own = list(tables[rng.randrange(r)][:rng.randrange(0, width)]) if r and rng.random() < 0.6 else []
        own = own[:lens[-1] // page]
        own += [order.pop() for _ in range(n - len(own))]
        tables.append(own)
        c.block_tables[r, :n] = torch.tensor(own, dtype=torch.int32)
    c.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    c.free_pages[:len(order)] = torch.tensor(order, dtype=torch.int32)
    c.n_free.fill_(len(order))
    return c, lens, tables, order


def released(lens, tables, free, finished):
    lens, free = list(lens), list(free)
    kept = {p for t, f in zip(tables, finished) if not f for p in t}
    for r, f in enumerate(finished):
        if f:
            free += [p for p in tables[r] if p not in kept and p not in free]
            lens[r] = 0
    return lens, free


@pytest.mark.parametrize("seed", range(8))
def test_shared_pages(seed):
    rng = random.Random(seed)
    c, lens, tables, free = shared_cache(rng, 9, 60)
    for _ in range(3):
        finished = [rng.random() < 0.4 for _ in range(9)]
        c.release(torch.tensor(finished))
        lens, free = released(lens, tables, free, finished)
        tables = [[] if n == 0 else t for n, t in zip(lens, tables)]
        assert c.kv_lens.tolist() == lens and c.n_free.item() == len(free)
        assert c.free_pages[:len(free)].tolist() == free


def test_one_flag_for_all():
    c, lens, tables, free = shared_cache(random.Random(1), 5, 40)
    c.release(torch.tensor([True]))
    lens, free = released(lens, tables, free, [True] * 5)
    assert c.kv_lens.tolist() == lens and c.free_pages[:c.n_free.item()].tolist() == free


def test_fake_tensors():
    """A cache of fake CUDA tensors (sizes are planned with them, without a GPU)."""
    with FakeTensorMode():
        c = PagedKVCache(2, 12, 8, 2, 64, max_requests=3, max_len=64, device="cuda")
        c.release(torch.zeros(3, dtype=torch.bool, device="cuda"))
        assert c.kv_lens.shape == (3,) and c.kv_lens.device.type == "cuda"


def test_compiled():
    """A graph of the call does what the call does."""
    finished = torch.tensor([True, False, True, False, True])
    made = [shared_cache(random.Random(3), 5, 40)[0] for _ in range(2)]
    made[0].release(finished)
    torch.compile(made[1].release, backend="eager", fullgraph=True)(finished)
    n = int(made[0].n_free)
    for a, b in ((made[0].kv_lens, made[1].kv_lens), (made[0].n_free, made[1].n_free), (made[0].free_pages[:n], made[1].free_pages[:n])):
        assert torch.equal(a, b)
