"""What the C entries of the causal attention operators refuse beyond tests/test_causal_host.py, without a GPU."""
import ctypes as C

import pytest

from some_amd import _lib
from some_amd.configs import get_config
from some_amd.engine import Engine

P = C.c_void_p(4096)                                  # never dereferenced: every call below fails validation
ROWS = (P, 256, 64)


@pytest.mark.parametrize('scale', [2.4e38, 3.4e38, 1e-46])
def test_scales_past_the_range_of_32_bits(scale):
    lib = _lib.load()
    h = Engine(get_config('two_head_model', lay=0), host_only=True).handle
    calls = [lib.some_op_causal_attention(h, 2, 64, *ROWS, 4, *ROWS, *ROWS, 2, P, P, 1, 10, 10, 1, scale, *ROWS, None, None, None, 0, None),
             lib.some_train_causal_attention_bwd(h, 2, 64, *ROWS, 4, *ROWS, *ROWS, 2, P, P, 1, 10, 10, 1, scale, *ROWS, P, P, *ROWS, *ROWS, *ROWS, *ROWS, P, 1 << 30, None),
             lib.some_op_attention_step(h, 2, 64, *ROWS, 4, P, 128 * 2000, 128, 64, P, 128 * 2000, 128, 64, 2, P, 3, 2000, scale, *ROWS, P, 1 << 30, None)]
    assert calls == [_lib.SOME_EINVAL] * 3 and b'scale' in lib.some_last_error(h)


def test_gain_gradients_that_overlap():
    """One array for both would be written by two blocks at once."""
    lib = _lib.load()
    h = Engine(get_config('two_head_model', lay=0), host_only=True).handle

    def call(dgq, dgk):
        return lib.some_train_qk_norm_rope_bwd(h, 2, 64, *ROWS, 4, *ROWS, 2, 10, P, P, P, 0, 1e4, 1e-6, *ROWS, *ROWS, *ROWS, *ROWS, C.c_void_p(dgq), C.c_void_p(dgk), 1, P,
                                               1 << 30, None)
    for dgk in (4096, 4096 + 252, 4096 - 252):
        assert call(4096, dgk) == _lib.SOME_EINVAL and b'overlap' in lib.some_last_error(h)
