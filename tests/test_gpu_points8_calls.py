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


def test_autograd_sees_what_is_written(A):
    """a tensor that a call writes to has another version after it, so a backward pass that needs what it held before says so"""
    bank = A.Points8(20, 16)
    idx, p = torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.full((6, 2), 0.5, device="cuda")
    w = torch.randn(6, 20, device="cuda", requires_grad=True)
    stats = A.teacher_loss(w, idx, p)[1]
    calls = [lambda t: bank.product(torch.ones(6, 16, device="cuda"), out=t), lambda t: A.teacher_loss(w, idx, p, grad=t), lambda t: A.teacher_loss(t, idx, p, grad=t),
             lambda t: A.teacher_grad(w, stats, idx, p, out=t), lambda t: A.teacher_grad(t, stats, idx, p, out=t), lambda t: bank.product(bank, n=20, m=6, out=t)]
    for call in calls:
        kept = w.exp()   # (its backward multiplies by what it gave)
        before = kept._version
        call(kept.detach())
        assert kept._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.sum().backward()
    for shape, call in (((6, 16), lambda t: bank.read(n=6, out=t)), ((3, 16), lambda t: bank.product_grad(torch.ones(3, 20, device="cuda"), out=t))):
        t = torch.zeros(shape, device="cuda")
        before = t._version
        call(t)
        assert t._version > before
    v = torch.ones(20, 1, device="cuda", requires_grad=True)
    kept = (v * bank.scales()).sum()   # (its backward multiplies by the scale bytes)
    codes = bank.codes()._version
    bank.write(torch.ones(1, 16, device="cuda"))
    assert bank.codes()._version > codes
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    with torch.inference_mode():   # (its tensors have no version)
        t = torch.zeros(6, 20, device="cuda")
        A.teacher_loss(w, idx, p, grad=t)
        assert t.any()


def test_rows_of_a_tensor_are_all_taken(A):
    """m and x_first choose points of another store: with a tensor they would be passed over, so they are refused"""
    bank = A.Points8(40, 30)
    x = torch.ones(5, 30, device="cuda")
    for more in (dict(m=3), dict(m=6), dict(x_first=1), dict(x_first=1, m=4)):
        with pytest.raises(A.AnnembedError):
            bank.product(x, **more)
    assert bank.product(x, m=5, x_first=0).shape == (5, 40)
