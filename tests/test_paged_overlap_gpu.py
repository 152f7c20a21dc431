"""Tensors that share memory, as the paged operators take or refuse them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_pools_of_one_tensor():
    from paged import copy_pages
    base = torch.randn(12, 1, 2, 16, 64, device="cuda").half()
    with pytest.raises(ValueError, match="overlap"):
        copy_pages(base[:8], base[4:], [0], [1])
    want = base.clone()
    want[1], want[7] = want[0], want[6]
    copy_pages(base[:6], base[6:], [0], [1])
    assert torch.equal(base, want)
