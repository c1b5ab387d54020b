"""paged_fork over pools that share memory without harm, and the refusals of what would corrupt it."""
import pytest
import torch

from test_paged_fork_gpu import i32, paged  # noqa: F401 (paged: the fixture)

pytestmark = pytest.mark.gpu


def state():
    """Two requests of 20 and 9 tokens in pages of 8, which become three: the second goes on from the first, the third from
    the second."""
    return dict(kv_lens=i32([20, 9, 0]), block_tables=i32([[4, 0, 2], [5, 1, 0], [0, 0, 0]]), free_pages=i32([7, 3, 6, 0, 0, 0, 0, 0]),
                n_free=i32([3]), parents=i32([0, 0, 1]), page_size=8)


COPIES = ((2, 6), (1, 3))  # page, its copy


def expect(before, after):
    want = before.clone()
    for a, b in COPIES:
        want[b] = before[a]
    assert torch.equal(after, want)


def test_interleaved_pools(paged):  # noqa: F811
    """Keys and values of all layers in one block per page; the parameters behind the codes; the same pool twice, a part of it."""
    whole = torch.randint(0, 1 << 15, (8, 3, 2, 64), dtype=torch.int16, device="cuda")
    for pools in ([whole[:, i, j] for i in range(3) for j in range(2)], [whole[:, 0, 0], whole[:, 2, 1]], [whole, whole],
                  [whole.flatten(1)[:, 8:200], whole[:, 0]], [whole[:, 0], whole[:, 0, 1, 8:], whole[:, 1:]],
                  [whole.flatten(1)[:, 64:], whole.flatten(1)[:, :64]]):
        whole.random_(0, 1 << 15)
        before = whole.clone()
        got = paged.paged_fork(**state(), pools=pools)
        assert got.granted.tolist() == [True, True, True] and got.kv_lens.tolist() == [20, 20, 9]
        want = before.clone()
        for p in pools:
            there = torch.as_strided(want, p.shape, p.stride(), p.storage_offset())
            was = torch.as_strided(before, p.shape, p.stride(), p.storage_offset())
            for a, b in COPIES:
                there[b] = was[a]
        assert torch.equal(whole, want)
        assert not torch.equal(whole, before)


def test_pools_after_one_another(paged):  # noqa: F811
    """Layers that follow one another, in any order of the list, with and without a gap."""
    whole = torch.randint(0, 1 << 15, (70, 9, 64), dtype=torch.int16, device="cuda")
    for pools in (list(whole[:, :8]), list(whole[:, 1:].flip(0).unbind()), [whole[i, 1:] for i in range(0, 70, 3)]):
        before = [p.clone() for p in pools]
        paged.paged_fork(**state(), pools=pools)
        for a, b in zip(before, pools):
            expect(a, b)


def test_refusals(paged):  # noqa: F811
    s = state()
    block = torch.zeros(40, dtype=torch.int32, device="cuda")
    pool = torch.zeros(12, 64, dtype=torch.int16, device="cuda")
    for kw in (dict(kv_lens_out=s["parents"]), dict(kv_lens_out=s["free_pages"][2:5]), dict(kv_lens_out=s["block_tables"][1]),
               dict(n_free_out=s["kv_lens"][:1]), dict(n_free_out=s["free_pages"][7:]), dict(kv_lens_out=block[3:6], n_free_out=block[5:6]),
               dict(kv_lens=block[:3], kv_lens_out=block[1:4]), dict(pools=[pool[:8], pool[1:9]]), dict(pools=[pool[:8], pool.flatten()[8:520].view(8, 64)]),
               dict(pools=[s["free_pages"].view(torch.int16).view(8, 2).repeat(1, 4), pool[:8], pool[4:]])):
        with pytest.raises(RuntimeError, match="overlap"):
            paged.paged_fork(**{**s, **kw})
    assert s["kv_lens"].tolist() == [20, 9, 0] and s["n_free"].item() == 3 and s["free_pages"].tolist() == [7, 3, 6, 0, 0, 0, 0, 0]


def test_pools_without_pages(paged):  # noqa: F811
    """Without pages there is nothing to copy, whatever the strides of the empty tensors say."""
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    odd = torch.zeros(1, 1, 1, device="cuda").expand(1, 3, 8)[:0]
    got = paged.paged_fork(i32([0, 0]), torch.zeros(2, 0, dtype=torch.int32, device="cuda"), empty, i32([0]), i32([1, -1]), 8, [odd, odd[:, ::2]])
    assert got.granted.tolist() == [True, True] and got.n_free.item() == 0
