"""Ends of the decoder-layer operators' ranges on the GPU: hints that are too small, windows without an end, values near
the ends of fp32, scores whose step is more than one, probabilities far below the largest one."""
import numpy as np
import pytest

from layer_util import BF16, F16, F32, HALF_STEP, HALF_TINY, Paged, fp8_values, from_bits, to_bits
from oracle import layer as ol
from test_layer_gpu import check_attention, run_attention, run_norm

pytestmark = pytest.mark.gpu


# ---- attention: a bound on the new tokens that is too small -------------------------------------------------------------
@pytest.mark.parametrize("dim,heads,kv_heads,max_new", [(128, 8, 2, 5), (128, 8, 2, 12), (64, 8, 2, 6), (256, 4, 2, 1), (200, 4, 2, 3), (128, 32, 1, 1)])
def test_attention_stores_every_row_whatever_the_bound_on_new_tokens_says(lib, dim, heads, kv_heads, max_new):
    """The context is long enough for every tile of rows to be split over several blocks and joined."""
    rng = np.random.default_rng(dim + max_new)
    p = Paged(rng, [2000], [90], heads, kv_heads, dim, 16, BF16, pad=2)
    check_attention(lib, p, max_new=max_new)
    check_attention(lib, p, max_new=90)


# ---- attention: windows that end nowhere --------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30 + 1, 2 ** 30])
@pytest.mark.parametrize("new,header", [(10, 16), (40, 16), (40, 24)])
def test_attention_window_without_an_end(lib, window, new, header):
    """kv_len below the new tokens, so that the first rows stand in front of key 0: none of the others loses its keys."""
    rng = np.random.default_rng(new)
    p = Paged(rng, [0, 70], [new, new], 4, 4, 64, 16, F16)
    p.kv[0] = new - 5
    a = check_attention(lib, p, window, header=header)
    assert np.array_equal(a, run_attention(lib, p, 0, header=header))
