"""Calls of the 8-bit store that are refused or that write to tensors of the caller's: what they leave behind."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def test_a_refused_write_leaves_the_store_as_it_was(A):
    """more blocks than one launch takes, scattered: refused before any row claims its slot, so later writes hold their rows"""
    cap, n = 5000, (1 << 30) + 64
    bank = A.Points8(cap, 1)
    slots = torch.arange(n, dtype=torch.int32, device="cuda") % cap
    with pytest.raises(A.AnnembedError, match="more than one call"):
        bank.write(torch.zeros(n, 1, dtype=torch.bfloat16, device="cuda"), slots=slots)
    x = torch.arange(1, cap + 1, device="cuda").view(cap, 1) % 16 + 1.0
    bank.write(x, slots=torch.randperm(cap, device="cuda").to(torch.int32))
    assert torch.equal(bank.read().sort(0)[0], x.sort(0)[0])
