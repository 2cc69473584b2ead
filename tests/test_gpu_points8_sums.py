"""Sums of the 8-bit product are held in 32 bits whatever the result's type and whichever kernel computes them: small integers, whose sums are
exact in 32 bits in any order, so results are the exact sums rounded once, bit for bit."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one launch for few rows, of whole and of shared groups; 64 x 64, 128 x 128 and 256 x 256 tiles, each with rests
SHAPES = [(1, 33000, 28), (3, 150, 784), (17, 2000, 300), (20, 1500, 500), (40, 1000, 200), (70, 200, 300), (130, 257, 1030), (300, 700, 2000), (1300, 1400, 300), (700, 4100, 130), (3830, 4090, 1030)]


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def exact(x, p):
    return torch.from_numpy(x).cuda().double() @ torch.from_numpy(p).cuda().double().T


def cancelling(rows, dim, rng, signs):
    """integers of at most 3 bits, and in every group of eight coordinates two of 448 (times `signs` for the second), the largest code"""
    x = rng.integers(-7, 8, (rows, dim)).astype(np.float32)
    first = np.arange(0, dim - 1, 8)
    x[:, first] = 448.0
    x[:, first + 1] = 448.0 * signs
    return x


@pytest.mark.parametrize("m,n,dim", SHAPES)
def test_what_cancels_leaves_the_small_products(A, m, n, dim):
    """448 * 448 and -448 * 448 beside products of 49 and less: sums cut 13 bits below the largest of eight products would lose the latter"""
    rng = np.random.default_rng(dim)
    p, x = cancelling(n, dim, rng, 1), cancelling(m, dim, rng, -1)
    want = exact(x, p)
    assert want.abs().max() < 2.0 ** 24
    bank, held = A.Points8(n, dim), A.Points8(m, dim)
    bank.write(torch.from_numpy(p).cuda())
    held.write(torch.from_numpy(x).cuda())
    for dtype in TYPES:
        assert torch.equal(bank.product(torch.from_numpy(x).cuda(), dtype=dtype), want.to(dtype))
        assert torch.equal(bank.product(held, dtype=dtype), want.to(dtype))


@pytest.mark.parametrize("m,n,dim", SHAPES)
def test_every_place_to_every_type(A, m, n, dim):
    """every place of every tile is its own, behind an odd stride and off 16 bytes"""
    rng = np.random.default_rng(m + n)
    p, x = rng.integers(-7, 8, (n, dim)).astype(np.float32), rng.integers(-7, 8, (m, dim)).astype(np.float32)
    want = exact(x, p)
    bank, held = A.Points8(n, dim), A.Points8(m + 2, dim)
    bank.write(torch.from_numpy(p).cuda())
    held.write(torch.from_numpy(x).cuda(), first=1)
    for dtype in TYPES:
        c = torch.full((m, n + 9), 7.0, dtype=dtype, device="cuda")
        bank.product(torch.from_numpy(x).to(dtype).cuda(), out=c[:, 3:3 + n])
        assert torch.equal(c[:, 3:3 + n], want.to(dtype)) and (c[:, :3] == 7).all() and (c[:, 3 + n:] == 7).all()
        c.fill_(7.0)
        bank.product(held, x_first=1, m=m, out=c[:, 3:3 + n])
        assert torch.equal(c[:, 3:3 + n], want.to(dtype)) and (c[:, :3] == 7).all() and (c[:, 3 + n:] == 7).all()


def test_equal_calls_give_equal_bits(A):
    """one order of summation: a product of ordinary numbers, again and again, into other memory"""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    for m, n, dim in SHAPES:
        bank = A.Points8(n, dim)
        bank.write(torch.randn(n, dim, generator=g, device="cuda"))
        x = torch.randn(m, dim, generator=g, device="cuda")
        for dtype in TYPES:
            first = bank.product(x, dtype=dtype)
            for _ in range(4):
                assert torch.equal(first, bank.product(x, dtype=dtype))
