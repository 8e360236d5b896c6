"""Calls of the decoder-layer operators that lie beyond what their index arithmetic takes: refused on the host, before
anything is launched (no GPU needed)."""
import pytest

from test_layer_cpu import INVALID, P, append, attention, norm, plan


@pytest.mark.parametrize("cols", [(1 << 30) + 1, (1 << 31) - 8192, (1 << 31) - 1])
def test_norm_refuses_rows_that_32_bits_do_not_index(lib, cols):
    """A thread's next column, c + 8192, would pass 2**31 - 1 and come back negative."""
    for kw in (dict(group=0), dict(group=32), dict(type=0), dict(x=P + 4, type=0)):
        assert norm(lib, cols=cols, x_stride=1 << 31, **kw) == INVALID


def test_norm_refuses_a_sum_over_x_at_another_pitch(lib):
    """residual_out's rows are cols apart: over an x whose rows are not, they would land on rows that are still to be read."""
    assert norm(lib, x=P, residual_out=P, x_stride=72) == INVALID
    assert norm(lib, x=P, residual=None, residual_out=P, x_stride=65, type=0) == INVALID


def test_attention_refuses_requests_that_32_bits_do_not_index(lib):
    for requests in ((1 << 30) + 1, (1 << 31) - 1):
        assert attention(lib, requests=requests) == INVALID
        assert lib.tb200_paged_attention_workspace_bytes(3, requests, 4, 2, 64) == 0


def test_factories_refuse_what_the_library_refuses():
    """The arrays are checked behind the sizes, so that none of that size is needed."""
    from tornadovm_b200.arrays import FloatArray, HalfFloatArray, Int8Array, IntArray
    from tornadovm_b200.b200 import B200
    f, h = FloatArray, HalfFloatArray
    with pytest.raises(RuntimeError, match="cols <= 2"):
        B200.rmsnormQuant(1, (1 << 30) + 1, f(4), f(4), 1e-5, "int8", 32, Int8Array(4), f(4))
    k = h(2 * 16 * 64)
    with pytest.raises(RuntimeError, match="requests <= 2"):
        B200.pagedAttention(1, (1 << 30) + 1, 0, 4, 2, 64, h(256), IntArray(2), IntArray(1), IntArray(1), 16, k, k, 0.1, 0, h(256))


def plan_places(**kw):
    """Arrays of a plan for two requests behind one another, 256 bytes each."""
    names = ("cached", "new", "free", "table", "cu", "kv", "positions", "slots", "counts")
    return {n: P + 256 * i for i, n in enumerate(names)} | kw


@pytest.mark.parametrize("out,on,by", [("kv", "cached", 0), ("kv", "new", 0), ("kv", "cached", 4), ("cu", "new", -8), ("cu", "cached", 4), ("positions", "new", 4), ("slots", "cached", 0),
                                       ("counts", "new", -12), ("table", "free", 8), ("table", "cached", 4), ("kv", "cu", 8), ("positions", "slots", 60), ("counts", "positions", 0),
                                       ("kv", "counts", 12), ("slots", "table", 24)])
def test_plan_refuses_outputs_over_other_arrays(lib, out, on, by):
    """Every block reads the lengths for itself while the first one writes kv_lens: updating them in place is a race, and
    so is any other output over an array that the call reads or writes."""
    at = plan_places()
    assert plan(lib, **(at | {out: at[on] + by})) == INVALID


def test_plan_factory_refuses_outputs_over_other_arrays():
    from tornadovm_b200.arrays import IntArray as I, LongArray
    from tornadovm_b200.b200 import B200
    a = dict(requests=2, pageSize=16, maxPages=4, maxTokens=8, cachedLens=I(2), newLens=I(2), freePages=I(3), blockTable=I(8), cuNew=I(3), kvLens=I(2), positions=I(8),
             slots=LongArray(8), counts=I(4))
    B200.pagedPlan(**a)
    B200.pagedPlan(**(a | dict(newLens=a["cachedLens"])))
    a |= dict(counts=I(4), freePages=I(4))
    for kw in (dict(kvLens=a["cachedLens"]), dict(cuNew=a["positions"]), dict(counts=a["freePages"]), dict(blockTable=a["positions"])):
        with pytest.raises(RuntimeError, match="one array"):
            B200.pagedPlan(**(a | kw))


@pytest.mark.parametrize("kw", [dict(in_type=0), dict(in_type=2, q_stride=512), dict(in_type=1, cache_type=2), dict(in_type=2, k_cache=P + 4096, v_cache=P + 4096)])
def test_append_refuses_outputs_over_what_is_still_read_or_written(lib, kw):
    """q_out over a q of another type or row pitch, and one cache for keys and values: threads would overwrite each other."""
    a = dict(q=P, q_out=P, k=P + 1024, v=P + 2048, k_cache=P + 4096, v_cache=P + 8192, cache_type=2) | kw
    assert append(lib, **a) == INVALID


def test_attention_refuses_an_out_over_q_at_another_pitch(lib):
    assert attention(lib, q=P, out=P, q_stride=256, out_stride=264) == INVALID
    assert attention(lib, q=P, out=P, q_stride=300, out_stride=256) == INVALID
