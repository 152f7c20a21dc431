"""Numbers that a PrefixPlan refuses (paged.py): they reach the C ABI as 32-bit integers."""
import pytest

import paged


@pytest.mark.parametrize("name", ["num_q_heads", "num_kv_heads", "head_dim", "max_length"])
@pytest.mark.parametrize("value", [(1 << 32) + 64, 1 << 31, -(1 << 31) - 1, 64.0, "64", None])
def test_numbers_that_are_no_32_bit_integers_are_refused(name, value):
    """2^32 + 64 would have become 64, and a plan of other heads or lengths than it says."""
    args = dict(num_q_heads=128, num_kv_heads=64, head_dim=64, max_length=64)
    args[name] = value
    with pytest.raises(ValueError, match=name):
        paged.PrefixPlan([2], [16], **args)


def test_integers_of_other_types_are_taken():
    import numpy as np
    assert [paged._int(v, "x") for v in (np.int64(5), True, 2**31 - 1, -2**31)] == [5, 1, 2**31 - 1, -2**31]
