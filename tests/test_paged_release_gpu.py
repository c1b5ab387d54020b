"""PagedKVCache.release on the GPU: by paged_fork and by index arithmetic, whatever the layers' tensors are."""
import random

import pytest
import torch

from test_paged_fork_gpu import i32, paged  # noqa: F401 (paged: the fixture)
from test_paged_release_cpu import released, shared_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(6))
def test_both_ways(paged, seed):  # noqa: F811
    made = [shared_cache(random.Random(seed), 40, 300, device="cuda") for _ in range(3)]
    rng = random.Random(seed)
    _, lens, tables, free = made[0]
    for _ in range(3):
        finished = [rng.random() < 0.3 for _ in range(40)]
        flags = torch.tensor(finished, device="cuda")
        made[0][0].release(flags)
        made[1][0]._release_by_index(flags)
        torch.compile(made[2][0].release, backend="eager", fullgraph=True)(flags)
        lens, free = released(lens, tables, free, finished)
        tables = [[] if n == 0 else t for n, t in zip(lens, tables)]
        for c, *_ in made:
            assert c.kv_lens.tolist() == lens and c.free_pages[:c.n_free.item()].tolist() == free


def test_layers_of_any_strides(paged):  # noqa: F811
    """Layer tensors whose pages are no blocks of memory, which the write and the attention take, or start anywhere."""
    cache = paged.PagedKVCache(1, 12, 8, 2, 64, max_requests=3, max_len=32)
    wide = torch.zeros(12, 8, 2, 128, dtype=torch.float16, device="cuda")
    cache.k[0], cache.v[0] = wide[..., :64], torch.zeros(12 * 8 * 2 * 64 + 4, dtype=torch.float16, device="cuda")[4:].view(12, 8, 2, 64)
    cache.append(i32([9, 20, 3]), 32)
    cache.release(torch.tensor([True, False, True], device="cuda"))
    assert cache.kv_lens.tolist() == [0, 20, 0] and cache.n_free.item() == 9
    cache.release(torch.tensor([True], device="cuda"))
    assert cache.kv_lens.tolist() == [0, 0, 0] and sorted(cache.free_pages.tolist()) == list(range(12))


def test_many_requests(paged):  # noqa: F811
    """More requests than paged_fork takes."""
    cache = paged.PagedKVCache(1, 9100, 8, 1, 32, max_requests=9000, max_len=16)
    cache.block_tables[:, 0] = torch.arange(9000, dtype=torch.int32, device="cuda") + 100
    cache.kv_lens.fill_(5)
    cache.free_pages[:100] = torch.arange(100, dtype=torch.int32, device="cuda")
    cache.n_free.fill_(100)
    flags = torch.arange(9000, device="cuda") % 3 == 0
    cache.release(flags)
    assert cache.n_free.item() == 3100 and cache.free_pages[100:3100].tolist() == list(range(100, 9100, 3))
    assert torch.equal(cache.kv_lens, torch.where(flags, 0, 5).int())


def test_captured(paged):  # noqa: F811
    cache, lens, tables, free = shared_cache(random.Random(2), 8, 60, device="cuda")
    flags = torch.zeros(8, dtype=torch.bool, device="cuda")
    cache.release(flags)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.release(flags)
    for finished in ([False, True] * 4, [True] * 8):
        flags.copy_(torch.tensor(finished))
        g.replay()
        lens, free = released(lens, tables, free, finished)
        tables = [[] if n == 0 else t for n, t in zip(lens, tables)]
        assert cache.kv_lens.tolist() == lens and cache.free_pages[:cache.n_free.item()].tolist() == free
