"""paged_fork where its warps cannot keep their entries of the tables between the passes (more than 16256 held entries: they
are read again), and over more pools than one launch copies."""
import random

import pytest
import torch

from test_paged_fork_gpu import i32, make, paged, run  # noqa: F401 (paged: the fixture)

pytestmark = pytest.mark.gpu

KEPT = 128 * 4 * 32 - 128  # li4_fork.cu: warps x groups x 32 entries less a warp's rounding


def mixed(rng, B):
    return [rng.choice([r, r, rng.randrange(B), -1]) for r in range(B)]


PARENTS = {"mixed": mixed, "exchanged": lambda rng, B: [B - 1 - r for r in range(B)], "all end": lambda rng, B: [-1] * B,
           "onto few": lambda rng, B: [r % 3 if r >= 3 else r for r in range(B)], "none there": lambda rng, B: [B + r % 2 for r in range(B)]}


@pytest.mark.parametrize("parents", PARENTS)
@pytest.mark.parametrize("B,width,spare", [(150, 600, 150), (6000, 12, 4000), (24, 3000, 7), (150, 600, 0)])
def test_long_lines(paged, B, width, spare, parents):  # noqa: F811
    lens, *_ = make(random.Random(17), B, 8, width, spare)
    assert sum(-(-n // 8) for n in lens) > KEPT
    run(paged, random.Random(17), B, 8, width, spare, rounds=2 if parents == "mixed" else 1, parents_of=PARENTS[parents])


@pytest.mark.parametrize("n_pools", [128, 129, 260])
def test_many_pools(paged, n_pools):  # noqa: F811
    """A 4-bit cache has four pools per layer: every pool's part page is copied, and no other page changes."""
    pools = [torch.randint(0, 1 << 15, (8, 8 * (1 + i % 3)), dtype=torch.int16, device="cuda") for i in range(n_pools)]
    before = [p.clone() for p in pools]
    got = paged.paged_fork(i32([20, 9, 0]), i32([[4, 0, 2], [5, 1, 0], [0, 0, 0]]), i32([7, 3, 6, 0, 0, 0, 0, 0]), i32([3]),
                           i32([0, 0, 1]), 8, pools)
    assert got.granted.tolist() == [True] * 3
    for was, p in zip(before, pools):
        was[6], was[3] = was[2], was[1]
        assert torch.equal(p, was)
