"""Arguments of paged_fork that lie over one another (no GPU: every call here is refused before it launches)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def native():
    import build

    build.build()
    from llama import _native

    return _native


B, WIDTH, STRIDE, CAPACITY = 4, 8, 10, 16
MB = 1 << 20


def fork(native, at=(), pools=((64 * MB, 4096, 2048),)):
    """paged_fork at addresses a megabyte apart, changed by `at`; pools are (address, stride, bytes)."""
    names = ("kv_lens", "parents", "block_tables", "free_pages", "n_free", "kv_lens_out", "n_free_out", "granted", "workspace")
    p = {name: (i + 1) * MB for i, name in enumerate(names)}
    p.update(at)
    n = len(pools)
    P, I = ctypes.c_void_p * n, ctypes.c_int64 * n
    rc = native.lib().li4_paged_fork(p["kv_lens"], p["parents"], B, p["block_tables"], STRIDE, WIDTH, p["free_pages"], CAPACITY,
                                     p["n_free"], 16, p["kv_lens_out"], p["n_free_out"], p["granted"], P(*[x[0] for x in pools]),
                                     I(*[x[1] for x in pools]), I(*[x[2] for x in pools]), n, p["workspace"], MB, None)
    return rc, native.last_error()


SIZE = dict(kv_lens=4 * B, parents=4 * B, block_tables=4 * (STRIDE * (B - 1) + WIDTH), free_pages=4 * CAPACITY, n_free=4,
            kv_lens_out=4 * B, n_free_out=4, granted=B)
WRITTEN = ("block_tables", "free_pages", "kv_lens_out", "n_free_out", "granted")
SAME = {("kv_lens_out", "kv_lens"), ("n_free_out", "n_free")}


@pytest.mark.parametrize("a", WRITTEN)
@pytest.mark.parametrize("b", SIZE)
def test_arrays(native, a, b):
    """Whatever is written, over any other array: from its start, its last element, and from below."""
    if a == b:
        return
    base, unit = 20 * MB, 1 if "granted" in (a, b) else 4
    places = [base + SIZE[b] - unit, base - SIZE[a] + unit]
    if (a, b) not in SAME and (b, a) not in SAME:
        places.append(base)
    elif SIZE[a] == 4:
        places = []  # (one element: the same one or none)
    for place in places:
        rc, message = fork(native, {a: place, b: base})
        assert rc == native.LI4_ERR_INVALID_ARG and "overlap" in message and (a in message or b in message), (place - base, message)


@pytest.mark.parametrize("name", SIZE)
def test_an_array_in_a_page(native, name):
    pool = (64 * MB, 4096, 2048)
    for at in (64 * MB, 64 * MB + 5 * 4096 + 2044, 64 * MB + 3 * 4096 - 3 if name == "granted" else 64 * MB + 3 * 4096 + 16):
        rc, message = fork(native, {name: at}, [pool])
        assert rc == native.LI4_ERR_INVALID_ARG and "overlap" in message and name in message, message


def test_pools(native):
    """Pages over other pages: shifted by a page, by part of a page, by a page and part of another pool's, of another stride."""
    first = (64 * MB, 4096, 2048)
    for other in ((64 * MB + 4096, 4096, 2048), (64 * MB + 4096 + 1024, 4096, 1024), (64 * MB + 3 * 4096 - 16, 4096, 32),
                  (64 * MB + 1024, 4096, 4096), (64 * MB - 7 * 4096, 4096, 2048), (64 * MB, 2048, 2048), (64 * MB + 2048, 8192, 4096)):
        for pools in ([first, other], [other, first], [first, (96 * MB, 64, 64), other, (65 * MB, 16, 16)]):
            rc, message = fork(native, pools=pools)
            assert rc == native.LI4_ERR_INVALID_ARG and "overlap" in message, (other, message)
    # three pools between one another: the last one over the first one's next page
    three = [(64 * MB, 4096, 1024), (64 * MB + 1024, 4096, 1024), (64 * MB + 2048, 4096, 2064)]
    rc, message = fork(native, pools=three)
    assert rc == native.LI4_ERR_INVALID_ARG and "overlap" in message


def test_spans_past_64_bits(native):
    assert fork(native, pools=[(64 * MB, 1 << 60, 2048)])[0] == native.LI4_ERR_INVALID_ARG
