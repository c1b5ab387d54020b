"""Arguments that the paged-cache entry points refuse on the host (no kernel is launched, no GPU needed)."""
import pytest


@pytest.fixture(scope="module")
def native():
    import build  # llama-efficient-inference_b200/build.py

    build.build()
    from llama import _native

    return _native


def test_append_refuses_a_negative_limit(native):
    def append(max_len, page=16):
        return native.lib().li4_paged_append_within(16, 16, 4, 16, 8, 8, 16, 16, 16, page, 4, max_len, 16, 16, 16, 16,
                                                    16, 16, None)

    assert append(-1) == native.LI4_ERR_INVALID_ARG and "max_len" in native.last_error()
    assert append(10, page=12) == native.LI4_ERR_UNSUPPORTED
