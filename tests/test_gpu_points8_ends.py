"""The ends of things in the 8-bit store: of f32's range, where what is finite stays finite and multiplies as such, and of a tensor's memory."""
import numpy as np
import pytest
import torch

from tests import points8_util as U

pytestmark = pytest.mark.gpu

TOP = 240.0 * 2.0 ** 120   # the largest code under the largest scale whose value f32 has: the next one stands for 2^128


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def held(x):
    """the format's value, or the largest that f32 has"""
    return np.clip(U.values(x), -TOP, TOP)


@pytest.mark.parametrize("m", [1, 70, 700])
def test_the_largest_coordinates_stay_finite(A, m):
    f32max = np.finfo(np.float32).max
    n, dim = 600, 200
    p = np.zeros((n, dim), np.float32)
    p[0, 3], p[1, 3], p[2, 150], p[3, 3] = f32max, -f32max, 3.3e38, 3.29e38
    p[4, :4] = f32max, 1.0, -3.1e38, 2.0 ** 112
    p[5, 7] = 1.5
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    want = held(p)
    got = bank.read().cpu().double().numpy()
    np.testing.assert_array_equal(got, want)
    assert np.isfinite(got).all() and abs(got[0, 3] / f32max - 1) <= 2.0 ** -4 and (bank.scales()[:5].amax(1) == 247).all()
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.zeros(m, dim)
        x[:, 7] = 2.0
        c = bank.product(x.cuda(), dtype=dtype).cpu()   # zeros meet the largest values
        assert torch.equal(c, torch.from_numpy(held(x.numpy()) @ want.T).to(dtype))
        x = torch.zeros(m, dim)
        x[:, 3], x[:, 150] = 2.0 ** -100, 2.0 ** -101
        c = bank.product(x.cuda(), dtype=dtype).cpu()
        assert torch.equal(c, torch.from_numpy(held(x.numpy()) @ want.T).to(dtype))
        big = torch.full((m, dim), float(f32max))
        big[:, 8:] = 0
        c = bank.product(big.cuda(), dtype=dtype).cpu()[:, 5]   # a large row too: 1.5 * TOP is beyond f32
        assert torch.isinf(c).all()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        dc = torch.zeros(m, n, dtype=dtype)
        dc[:, 5] = 3.0
        assert torch.equal(bank.product_grad(dc.cuda()).cpu(), torch.from_numpy(dc.double().numpy() @ want).float())
        dc[:, 0] = 2.0 ** -10
        assert torch.equal(bank.product_grad(dc.cuda()).cpu(), torch.from_numpy(dc.double().numpy() @ want).float())


@pytest.mark.parametrize("m", [1, 70, 700])
def test_the_smallest_values(A, m):
    """values held below 2^-126: read back exactly, multiplied as the nearest multiple of 2^-133"""
    n, dim = 600, 130
    p = np.zeros((n, dim), np.float32)
    p[np.arange(300), 5] = np.arange(1, 301, dtype=np.float64) * 2.0 ** -135
    p[np.arange(300), 129] = np.float32(-(2.0 ** -126))
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    want = U.values(p)
    np.testing.assert_array_equal(bank.read().cpu().double().numpy(), want)
    scale = 2.0 ** 100
    x = torch.zeros(m, dim)
    x[:, 5] = scale
    got = bank.product(x.cuda()).cpu().double().numpy()
    assert (np.abs(got - scale * want[:, 5]) <= scale * 2.0 ** -134).all()
    grid = 2.0 ** -133
    exact = np.abs(want[:, 5]) % grid == 0
    assert exact.sum() > 300 and np.array_equal(got[:, exact], np.broadcast_to(scale * want[:, 5], got.shape)[:, exact])
    dc = torch.zeros(m, n)
    dc[:, :300] = scale
    grad = bank.product_grad(dc.cuda()).cpu().double().numpy()
    assert (np.abs(grad[:, 5] - scale * want[:, 5].sum()) <= scale * (300 * 2.0 ** -134 + 300 * 2.0 ** -24 * want[:, 5].sum())).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,dim", [(1, 1, 1), (1, 65, 130), (5, 129, 40), (64, 4097, 28), (65, 63, 200), (300, 5001, 784), (130, 70001, 131), (2100, 3001, 130)])
def test_the_last_value_of_dc_counts(A, m, n, dim, dtype):
    """an odd number of values, the last ones of their memory and of a page, and beside NaN: sums of small integers are exact"""
    rng = np.random.default_rng(n)
    p, dc = rng.integers(-7, 8, (n, dim)).astype(np.float32), rng.integers(-7, 8, (m, n)).astype(np.float32)
    p[-1], dc[:, -1] = 7, 5
    want = torch.from_numpy(dc @ p)
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    src = torch.from_numpy(dc).to(dtype).cuda()
    size = src.element_size()
    room = torch.full((m * n + 3 * 4096 // size,), float("nan"), dtype=dtype, device="cuda")
    end = (-(room.data_ptr() + m * n * size) % 4096 + 4096) // size + m * n   # elements to an end of a page behind m * n
    for last in (end, end - 1, end + 1):
        view = room[last - m * n:last].view(m, n)
        view.copy_(src)
        assert (view.data_ptr() + m * n * size) % 4096 == (last - end) * size % 4096
        assert torch.equal(bank.product_grad(view).cpu(), want)
        room.fill_(float("nan"))
