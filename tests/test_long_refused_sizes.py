"""Workspace sizes of the long-context operators for shapes that the calls refuse: none, as the header says."""

import pytest

from mini_engine_hip.kernels import hip_extension as ext

FAKE = 1 << 20  # an aligned address that nothing reads: arguments are refused before


@pytest.fixture(scope="module")
def lib():
    return ext.load_hip_extension()


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,width", [
    (100, 8192, 8192, 128, 32),              # a token's row of a cache is longer than 1 MB
    ((1 << 21) - 1, 1024, 1024, 16, 32),     # more work-groups than a launch has
])
def test_prompt_weights(lib, tokens, q_heads, kv_heads, dim, width):
    status = lib._lib.mvme_prefill_attention_weights(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16 * width, 2, tokens, q_heads,
                                                     kv_heads, dim, 99, 16, width, 0, FAKE, 1 << 60, None)
    assert status == ext.EINVAL and "too" in lib.last_error()
    assert lib.prefill_weights_workspace_size(2, tokens, q_heads, kv_heads, dim, 16, width) == 0


def test_weighted_steps(lib):
    status = lib._lib.mvme_paged_attention_weights(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16 * 257, (1 << 20) - 1, 16, 8, 128, 99,
                                                   16, 257, 0, FAKE, 1 << 60, None)
    assert status == ext.EINVAL and "too large" in lib.last_error()
    assert lib.weights_workspace_size((1 << 20) - 1, 16, 8, 128, 16, 257) == 0
