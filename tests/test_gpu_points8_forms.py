"""Every form of the 8-bit store's writes and reads and of the gradient's kernels, against what is exact: integers whose sums are exact in 32
bits, bit for bit, and one call against the same work in parts.  tests/test_points8_plan.py says which form a size takes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def integers(rng, most, rows, cols):
    return rng.integers(-most, most + 1, (rows, cols)).astype(np.float32)


# several slices of the points; tiles of 64 and of 128 rows; joins of 1, 4, 16 and 64 groups; odd m, n and dim
GRADIENTS = [(16, 40000, 64), (64, 10007, 128), (300, 5001, 784), (16, 100000, 128), (300, 60000, 784), (1, 30001, 5), (129, 70001, 131), (2100, 3001, 1000), (4111, 2003, 515), (257, 33333, 200), (200, 65, 130), (3000, 129, 1500)]


@pytest.mark.parametrize("m,n,dim", GRADIENTS)
def test_gradient_of_integers(A, m, n, dim):
    """|dc p| <= 49: sums of up to 10^5 of them stay below 2^24"""
    rng = np.random.default_rng(n)
    p, dc = integers(rng, 7, n, dim), integers(rng, 7, m, n)
    want = torch.from_numpy(dc @ p)
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    for dtype in TYPES:
        dev = torch.from_numpy(dc).to(dtype).cuda()
        assert torch.equal(bank.product_grad(dev).cpu(), want)
        if m * n < 2 * 10 ** 7:   # rows 3 elements apart of what they hold, off 16 bytes; results of 16 bits, rounded once
            wide = torch.full((m, n + 3), float("nan"), dtype=dtype, device="cuda")
            wide[:, 2:2 + n] = dev
            assert torch.equal(bank.product_grad(wide[:, 2:2 + n]).cpu(), want)
            for out in TYPES[1:]:
                assert torch.equal(bank.product_grad(dev, dtype=out).cpu(), want.to(out))


@pytest.mark.parametrize("m,n,dim", GRADIENTS)
def test_gradient_of_wide_integers(A, m, n, dim):
    """dc of f32 with 19 significant bits (three partial products), of f16 with 11 (two): 24 entries a row, the first and the last point and
    others, p of -1, 0 and 1: every sum is below 24 * 2^19 < 2^24"""
    rng = np.random.default_rng(m)
    p = integers(rng, 1, n, dim)
    p[[0, n - 1]] = 1
    at = rng.integers(0, n, (m, 24))
    at[:, 0], at[:, 1] = 0, n - 1
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    for dtype, most in ((torch.float32, (1 << 19) - 1), (torch.float16, 2047)):
        dc = np.zeros((m, n), np.float32)
        np.put_along_axis(dc, at, (rng.integers(most // 2, most + 1, (m, 24)) * rng.choice([-1, 1], (m, 24)) | 1).astype(np.float32), 1)
        want = torch.from_numpy(dc @ p)
        assert torch.equal(bank.product_grad(torch.from_numpy(dc).to(dtype).cuda()).cpu(), want)


def noise(n, dim, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    return torch.randn(n, dim, generator=g, device="cuda").to(dtype)


# blocks on both sides of 2^20, from where a group of lanes takes four of them; one block a row and two
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [((1 << 20) - 5, 16), ((1 << 20) + 77, 16), ((1 << 19) + 5, 130), (150001, 1000)])
def test_large_writes_and_reads_are_their_parts(A, n, dim, dtype):
    x = noise(n, dim, dtype)
    whole, parts = A.Points8(n + 9, dim), A.Points8(n + 9, dim)
    step = 100003
    whole.write(x, first=7)
    for lo in range(0, n, step):
        parts.write(x[lo:lo + step], first=7 + lo)
    assert torch.equal(whole.codes().view(torch.uint8), parts.codes().view(torch.uint8)) and torch.equal(whole.scales(), parts.scales())
    got = whole.read(n=n, first=7, dtype=dtype)
    ids = torch.randperm(n + 9, device="cuda")[:n].to(torch.int32)
    by_ids = whole.read(slots=ids, dtype=dtype)
    for lo in range(0, n, step):
        assert torch.equal(got[lo:lo + step], parts.read(n=min(step, n - lo), first=7 + lo, dtype=dtype))
        assert torch.equal(by_ids[lo:lo + step], parts.read(slots=ids[lo:lo + step], dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [((1 << 20) - 5, 16), ((1 << 20) + 77, 16), ((1 << 19) + 5, 130), (150001, 1000)])
def test_large_scattered_writes_are_their_parts(A, n, dim, dtype):
    """with repeated and skipped slots: parts written one after the other hold the last of equal slots; twice, so nothing is left claimed"""
    cap = n // 2
    whole, parts = A.Points8(cap, dim), A.Points8(cap, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    step = 4001   # (a part of it is one launch that looks for repeated slots itself)
    for turn in range(2):
        x = noise(n + turn, dim, dtype)[:n]
        slots = torch.randint(-1, cap + 1, (n,), generator=g, device="cuda").to(torch.int32)
        whole.write(x, slots=slots)
        for lo in range(0, n, step):
            parts.write(x[lo:lo + step], slots=slots[lo:lo + step])
        assert torch.equal(whole.codes().view(torch.uint8), parts.codes().view(torch.uint8)) and torch.equal(whole.scales(), parts.scales())


@pytest.mark.parametrize("m,n,dim", [(130, 129, 30000), (70, 300, 130)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_rows_far_apart(A, m, n, dim, dtype):
    """rows of dc 4.2 million elements apart, more than the copies' 32-bit offsets reach in a tile of 128 rows (of 64 for f32)"""
    rng = np.random.default_rng(dim)
    p, dc = integers(rng, 7, n, dim), integers(rng, 7, m, n)
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    step = 8_400_001 if dtype != torch.float32 and m < 128 else 4_200_001
    room = torch.full(((m - 1) * step + n,), float("nan"), dtype=dtype, device="cuda")
    far = room.as_strided((m, n), (step, 1))
    far.copy_(torch.from_numpy(dc).to(dtype))
    assert torch.equal(bank.product_grad(far).cpu(), torch.from_numpy(dc @ p))


@pytest.mark.parametrize("n,dim", [(1500, 200), (5000, 28), (7000, 200)])
def test_captured_scattered_writes(A, n, dim):
    """slots looked at by every workgroup, claimed and given back by the rows themselves, claimed and given back in a launch: replayed with other slots,
    with writes of the same store between"""
    cap = 3000
    bank, plain = A.Points8(cap, dim), A.Points8(cap, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    x, slots = torch.zeros(n, dim, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bank.write(x, slots=slots)
    for turn in range(3):
        x.normal_(generator=g)
        slots.copy_(torch.randint(-1, cap + 1, (n,), generator=g, device="cuda"))
        graph.replay()
        plain.write(x, slots=slots)
        assert torch.equal(bank.codes().view(torch.uint8), plain.codes().view(torch.uint8)) and torch.equal(bank.scales(), plain.scales())
        for store in (bank, plain):
            store.write(x[:100] * 2, first=turn)
            store.write(x.flip(0), slots=slots)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_product_of_rows_far_apart(A, dtype):
    """rows of the result farther apart than the 32-bit offsets of a 128 x 128 tile's stores reach, with a rest of both; nothing between them is written"""
    m, n, dim = 130, 8333, 200
    rng = np.random.default_rng(m)
    p, x = integers(rng, 7, n, dim), integers(rng, 7, m, dim)
    bank = A.Points8(n, dim)
    bank.write(torch.from_numpy(p).cuda())
    step = 8_400_001 if dtype != torch.float32 else 4_200_001
    room = torch.full(((m - 1) * step + n,), 7.0, dtype=dtype, device="cuda")
    far = room.as_strided((m, n), (step, 1))
    for turn in range(2):   # (tiles follow one another in a workgroup: the second call's find the first's results)
        bank.product(torch.from_numpy(x).cuda(), out=far)
        assert torch.equal(far.cpu(), torch.from_numpy(x @ p.T).to(dtype))
    assert (room.as_strided((m - 1, step - n), (step, 1), n) == 7).all()
