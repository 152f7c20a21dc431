"""K and V pools that share memory are refused (the C ABI, before any CUDA call)."""
import pytest

from test_paged_ops_cpu import POOLS, _call, _err

BYTES = POOLS["num_pages"] * POOLS["inner"] * POOLS["page_tokens"] * POOLS["token_bytes"]


@pytest.mark.parametrize("name,lists", [("copy", ([0], [1], None)), ("fork", ([0], [1], [5], [0])), ("compact", ([5], [0]))])
@pytest.mark.parametrize("apart", [16, BYTES // 2, BYTES - 16, -16, -BYTES + 16])
def test_overlapping_pools_are_refused(name, lists, apart):
    """(The places are no memory: nothing but the refusal may happen.)"""
    assert _call(name, pools=dict(v_pool=POOLS["k_pool"] + apart), lists=lists) != 0
    assert "overlap" in _err()


@pytest.mark.parametrize("apart", [BYTES, -BYTES])
def test_pools_side_by_side_are_taken(apart):
    assert _call("copy", pools=dict(v_pool=POOLS["k_pool"] + apart), lists=([], [], None)) == 0
