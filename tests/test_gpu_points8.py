"""GPU tests of the 8-bit store, the product with it and the product's gradient, against 64-bit oracles (tests/points8_util.py).

Tolerances.  Codes, scale bytes and values read back are equal to the oracle's bit for bit (scales are powers of two, one rounding a code).
product: products of codes and scales are exact, a sum of K terms in f32 is off by at most K 2^-23 sum |x_k p_k| whatever its order and whether
the adder rounds or cuts, the result's rounding by eps / 2 of it (of the smallest normal number at least).  Results of 16 bits come from the
8-bit matrix cores: they add eight products at a time and keep 13 bits below the largest, so the seven others lose less than 2^-13 of it each:
7 * 2^-13 sum |x_k p_k| more.  product_grad: n terms, three partial products for f32."""
import numpy as np
import pytest
import torch

from tests import points8_util as U

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def vectors(n, dim, seed, dtype=torch.float32):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(n, dim)) * np.exp(rng.normal(size=dim)) * np.exp(2 * rng.normal(size=(n, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


def n64(t):
    return t.detach().cpu().float().numpy().astype(np.float64) if t.dtype != torch.float64 else t.cpu().numpy()


def assert_held(bank, rows, x):
    codes, bytes_ = U.quantise(n64(x))
    got_c, got_s = n64(bank.codes()[rows]), bank.scales()[rows].cpu().numpy()
    np.testing.assert_array_equal(got_s, bytes_)
    np.testing.assert_array_equal(got_c, codes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 15), (5, 16), (2, 17), (7, 127), (64, 128), (9, 129), (33, 784), (1025, 28), (300, 1024), (2, 5000)])
def test_write_and_read(A, n, dim, dtype):
    bank = A.Points8(n + 3, dim)
    x = vectors(n, dim, 1, dtype)
    bank.write(x.cuda(), first=2)
    assert_held(bank, slice(2, 2 + n), x)
    assert not bank.codes().view(torch.uint8)[:2].any() and not bank.codes().view(torch.uint8)[2 + n:].any()   # other rows as they were
    want = U.values(n64(x))
    for out in TYPES:
        got = bank.read(n=n, first=2, dtype=out)
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(out))
    assert not bank.read(n=2).any()


def test_special_values(A):
    """zeros, the borders of a scale, subnormals, the largest numbers, NaN and infinities beside ordinary values"""
    x = np.zeros((12, 130), np.float32)
    x[1, :3] = 448.0, -448.0, 1.0
    x[2, :3] = np.nextafter(np.float32(448.0), np.float32(1e9)), 1.0, -0.0078125
    x[3, :4] = 1e-45, -3e-45, 1e-40, 1e-39
    x[4, :2] = 3.0e38, -1e38
    x[5, :4] = np.nan, 1.0, -2.0, 3.0
    x[6, :4] = np.inf, 1.0, -np.inf, 3.0
    x[7, :] = np.inf
    x[8, :16] = 448.0 * 2.0 ** -np.arange(16)
    x[9, :17] = 256.0 + 16.0 * np.arange(17) * 0.75          # ties and others between codes
    x[10, 128] = 5.0                                          # the short last block alone
    x[11, :6] = 448.0, 2.0 ** -10, 1.5 * 2.0 ** -10, 2.0 ** -9, 3.0 * 2.0 ** -10, 2.0 ** -11   # around the smallest code: ties to even
    bank = A.Points8(12, 130)
    bank.write(torch.from_numpy(x).cuda())
    assert_held(bank, slice(None), torch.from_numpy(x))
    np.testing.assert_array_equal(n64(bank.read()), U.values(x))


@pytest.mark.parametrize("n,dim", [(5, 200), (1024, 200), (1025, 200), (5000, 200), (1025, 128), (5000, 28)])
def test_slots(A, n, dim):
    """scattered, padded, repeated and invalid slots, on both sides of the size where the rows claim their slots, of one block and more; twice"""
    rng = np.random.default_rng(n)
    cap = 3000
    bank = A.Points8(cap, dim)
    held = np.zeros((cap, dim))
    for turn in range(2):
        x = vectors(n, dim, 10 * n + turn)
        slots = rng.integers(0, cap, n).astype(np.int64)
        slots[rng.integers(0, n, max(1, n // 10))] = -1
        slots[0] = cap                    # outside: skipped
        slots[n - 1] = slots[n // 2] if slots[n // 2] >= 0 else 7
        bank.write(x.cuda(), slots=torch.from_numpy(slots).to(torch.int32).cuda())
        v = U.values(n64(x))
        for i, s in enumerate(slots):     # in order: the last of equal slots stays
            if 0 <= s < cap:
                held[s] = v[i]
        np.testing.assert_array_equal(n64(bank.read()), held)
    want = torch.from_numpy(np.where((slots >= 0)[:, None], np.where((slots < cap)[:, None], held[np.clip(slots, 0, cap - 1)], np.nan), 0.0)).float()
    got = bank.read(slots=torch.from_numpy(slots).to(torch.int32).cuda()).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=1e30), torch.nan_to_num(want, nan=1e30))
    assert bank.read(slots=torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, dim)
    bank.write(torch.zeros(0, dim, device="cuda"))
    np.testing.assert_array_equal(n64(bank.read()), held)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(A, dtype):
    n, dim = 37, 300
    x = vectors(n, dim, 5, dtype)
    base = torch.zeros(n * 2, dim + 13, dtype=dtype, device="cuda")
    view = base[::2, 5:5 + dim]           # rows two strides apart, starting off 16 bytes
    view.copy_(x)
    bank = A.Points8(n, dim)
    bank.write(view)
    assert_held(bank, slice(None), x)
    out = torch.full((n, dim + 7), 9.0, dtype=dtype, device="cuda")
    bank.read(dtype=dtype, out=out[:, 3:3 + dim])
    assert torch.equal(out[:, 3:3 + dim].cpu(), torch.from_numpy(U.values(n64(x))).to(dtype))
    assert (out[:, :3] == 9).all() and (out[:, 3 + dim:] == 9).all()


def product_bound(x, p, terms, want, dtype, eights=False):
    f = torch.finfo(dtype)
    return (terms * 2.0 ** -23 + eights * 7 * 2.0 ** -13) * (np.abs(x) @ np.abs(p)) + f.eps / 2 * np.maximum(np.abs(want), f.smallest_normal)


@pytest.mark.parametrize("m,n,dim", [(1, 1, 1), (1, 3, 28), (1, 1000, 784), (17, 32768, 28), (20, 1500, 500), (31, 700, 600), (9, 3000, 1500), (50, 3000, 200), (64, 16384, 10), (700, 4100, 130), (129, 33000, 100), (4100, 4200, 140), (2500, 2600, 28), (65, 16300, 520), (2, 129, 128), (5, 64, 130), (16, 500, 784), (17, 257, 100), (33, 31, 1000), (64, 2000, 16), (127, 128, 129),
                                     (128, 128, 256), (129, 385, 640), (200, 1111, 784), (300, 700, 2000), (513, 1025, 64), (1, 40, 9000)])
def test_product(A, m, n, dim):
    bank = A.Points8(n + 5, dim)
    p = vectors(n + 5, dim, 3)
    bank.write(p.cuda())
    pv = U.values(n64(p))[3:3 + n]
    for dtype, out in [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32)]:
        x = vectors(m, dim, 4, dtype)
        if dtype == torch.float16:
            x = x / 64
        xv = U.values(n64(x))
        want = xv @ pv.T
        c = torch.full((m, n + 9), 7.0, dtype=out, device="cuda")
        bank.product(x.cuda(), n=n, first=3, out=c[:, 2:2 + n])
        if out == torch.float16:
            fits = np.abs(want) < 65000
        else:
            fits = np.ones_like(want, bool)
        got = n64(c[:, 2:2 + n])
        assert (np.abs(got - want) <= product_bound(xv, pv.T, dim, want, out, out != torch.float32))[fits].all()
        assert (c[:, :2] == 7).all() and (c[:, 2 + n:] == 7).all()
    q = A.Points8(m + 2, dim)
    q.write(x.cuda(), first=1)
    a = bank.product(q, n=n, first=3, x_first=1, m=m, dtype=torch.float32)
    # the same terms, in an order of their own: each sum is off by the bound at most
    assert (np.abs(n64(a) - want) <= product_bound(xv, pv.T, dim, want, torch.float32)).all()


def test_product_small_integers(A):
    """sums of small integers are exact in any order: equal bit for bit, and every place of every tile is its own"""
    rng = np.random.default_rng(0)
    for m, n, dim in [(130, 200, 300), (3, 150, 784), (257, 300, 1030), (40, 40, 128), (16, 333, 4097)]:
        p, x = rng.integers(-7, 8, (n, dim)).astype(np.float32), rng.integers(-7, 8, (m, dim)).astype(np.float32)
        bank = A.Points8(n, dim)
        bank.write(torch.from_numpy(p).cuda())
        got = bank.product(torch.from_numpy(x).cuda()).cpu().numpy()
        np.testing.assert_array_equal(got, x @ p.T)
        dc = rng.integers(-7, 8, (m, n)).astype(np.float32)
        for dtype in TYPES:
            np.testing.assert_array_equal(bank.product_grad(torch.from_numpy(dc).to(dtype).cuda()).cpu().numpy(), dc @ p)


def test_product_nan_stays_in_its_row_and_column(A):
    p, x = vectors(200, 300, 1), vectors(150, 300, 2)
    p[17, 250] = float("inf")
    x[41, 3] = float("nan")
    bank = A.Points8(200, 300)
    bank.write(p.cuda())
    c = bank.product(x.cuda()).cpu()
    nan = torch.isnan(c)
    want = torch.zeros_like(nan)
    want[41, :] = True
    want[:, 17] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("m,n,dim", [(1, 1, 1), (1, 1000, 784), (3, 65, 28), (64, 63, 128), (129, 200, 130), (300, 5000, 784), (16, 40000, 64), (257, 100, 1000)])
def test_product_grad(A, m, n, dim):
    bank = A.Points8(n + 5, dim)
    p = vectors(n + 5, dim, 3)
    bank.write(p.cuda())
    pv = U.values(n64(p))[3:3 + n]
    rng = np.random.default_rng(7)
    for dtype, out in [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.bfloat16, torch.float32)]:
        dc = torch.from_numpy((rng.normal(size=(m, n)) * 0.01).astype(np.float32)).to(dtype)
        wide = torch.zeros(m, n + 11, dtype=dtype, device="cuda")
        wide[:, 3:3 + n] = dc.cuda()
        dv = n64(dc)
        want = dv @ pv
        dx = torch.full((m, dim + 5), 7.0, dtype=out, device="cuda")
        bank.product_grad(wide[:, 3:3 + n], n=n, first=3, out=dx[:, 2:2 + dim])
        got = n64(dx[:, 2:2 + dim])
        assert (np.abs(got - want) <= product_bound(dv, pv, 3 * n + 64, want, out)).all()
        assert (dx[:, :2] == 7).all() and (dx[:, 2 + dim:] == 7).all()
    again = bank.product_grad(wide[:, 3:3 + n], n=n, first=3)
    assert torch.equal(again, bank.product_grad(wide[:, 3:3 + n], n=n, first=3))   # one order of summation
    # against differences: the product is linear, so a difference of two products is its derivative
    if m * n < 10 ** 5 and dim > 1:
        assert np.abs(dv @ pv[:, 1] - n64(again)[:, 1]).max() <= (product_bound(dv, pv, 3 * n + 64, want, torch.float32))[:, 1].max()


def test_product_grad_extremes(A):
    """the largest f32 gradients are cut, not rounded past the largest bf16; no points sum to zero; NaN and inf stay in their rows"""
    bank = A.Points8(64, 32)
    bank.write((torch.eye(64, 32) * 0.5).cuda())
    dc = torch.zeros(4, 64)
    dc[0, 3], dc[1, 4], dc[2, 5] = 3.4e38, float("nan"), -3.0e38
    got = bank.product_grad(dc.cuda()).cpu()
    assert abs(got[0, 3].item() / 1.7e38 - 1) < 1e-6 and abs(got[2, 5].item() / -1.5e38 - 1) < 1e-6
    assert torch.isnan(got[1]).all() and not torch.isnan(got[[0, 2, 3]]).any() and not got[3].any()
    assert not bank.product_grad(torch.zeros(3, 0, device="cuda"), n=0).any()
    assert bank.product(torch.zeros(0, 32, device="cuda")).shape == (0, 64)
    assert bank.product(torch.ones(2, 32, device="cuda"), n=0).shape == (2, 0)


def test_offsets_past_32_bits(A):
    """rows whose codes lie beyond 4 GiB"""
    cap, dim = 4_300_000, 1024
    bank = A.Points8(cap, dim)
    x = vectors(300, dim, 8)
    bank.write(x.cuda(), first=cap - 300)
    slots = torch.arange(cap - 300, cap, dtype=torch.int32, device="cuda")
    v = U.values(n64(x))
    np.testing.assert_array_equal(n64(bank.read(slots=slots)), v)
    q = vectors(70, dim, 9)
    qv = U.values(n64(q))
    got = n64(bank.product(q.cuda(), n=300, first=cap - 300))
    assert (np.abs(got - qv @ v.T) <= product_bound(qv, v.T, dim, qv @ v.T, torch.float32)).all()
    dc = vectors(20, 300, 10)
    got = n64(bank.product_grad(dc.cuda(), n=300, first=cap - 300))
    assert (np.abs(got - n64(dc) @ v) <= product_bound(n64(dc), v, 964, n64(dc) @ v, torch.float32)).all()


def test_graph_of_the_points_held(A):
    x = vectors(700, 40, 6) / 8
    bank = A.Points8(800, 40)
    bank.write(x.cuda(), first=50)
    a = A.KGraph.bruteforce_l2_points8(bank, 7, n=700, first=50)
    b = A.KGraph.bruteforce_l2(U.values(n64(x)).astype(np.float32), 7)
    for p, q in zip(a.get_neighbours(), b.get_neighbours()):
        np.testing.assert_array_equal(p, q)


def test_streams_and_graphs(A):
    """on a stream that is not the current one's default, two captured calls side by side, replayed with other inputs and eager work between"""
    dim, n, m = 200, 900, 70
    bank = A.Points8(n, dim)
    p = vectors(n, dim, 1).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bank.write(p)
        x = vectors(m, dim, 2).cuda()
        want = bank.product(x)
    side.synchronize()
    assert torch.equal(want, bank.product(x))
    dc = vectors(m, n, 3).cuda().bfloat16()
    slots = torch.arange(m, dtype=torch.int32, device="cuda")
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c = bank.product(x)
            d = bank.product_grad(dc)
            r = bank.read(slots=slots)
        graphs.append(g)
        outs.append((c, d, r))
    for turn in range(3):
        x.copy_(vectors(m, dim, 20 + turn).cuda())
        dc.copy_(vectors(m, n, 30 + turn).cuda())
        slots.copy_(torch.randperm(n, device="cuda")[:m].to(torch.int32))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = bank.product(x), bank.product_grad(dc), bank.read(slots=slots)
        for o in outs:
            for a, b in zip(o, eager):
                assert torch.equal(a, b)
    w = torch.cuda.CUDAGraph()
    big = vectors(1500, dim, 4).cuda()
    where = torch.randint(0, n, (1500,), device="cuda").to(torch.int32)
    with torch.cuda.graph(w):
        bank.write(big, slots=where)
    for turn in range(3):
        big.copy_(vectors(1500, dim, 40 + turn).cuda())
        where.copy_(torch.randint(0, n, (1500,), device="cuda").to(torch.int32))
        w.replay()
        torch.cuda.synchronize()
        v, held = U.values(n64(big)), {}
        for i, s in enumerate(where.cpu().tolist()):
            held[s] = v[i]
        got = n64(bank.read())
        for s, row in held.items():
            np.testing.assert_array_equal(got[s], row)


def test_refusals(A):
    bank = A.Points8(100, 64)
    x = torch.zeros(10, 64, device="cuda")
    bad = [
        lambda: A.Points8(0, 64), lambda: A.Points8(10, 0), lambda: A.Points8(1 << 33, 4), lambda: A.Points8(10, (1 << 20) + 1),
        lambda: bank.write(x.cpu()), lambda: bank.write(x.double()), lambda: bank.write(x[:, :63]), lambda: bank.write(x.t().contiguous().t()),
        lambda: bank.write(x, first=91), lambda: bank.write(x, first=-1), lambda: bank.write(x[0]), lambda: bank.write(x[:1].expand(10, 64)),
        lambda: bank.write(x, slots=torch.zeros(9, dtype=torch.int32, device="cuda")), lambda: bank.write(x, slots=torch.zeros(10, dtype=torch.int64, device="cuda")),
        lambda: bank.write(x, slots=torch.zeros(10, dtype=torch.int32)), lambda: bank.read(n=101), lambda: bank.read(n=3, first=98),
        lambda: bank.read(dtype=torch.float64), lambda: bank.read(n=4, out=torch.zeros(5, 64, device="cuda")),
        lambda: bank.product(x[:, :60]), lambda: bank.product(x, n=101), lambda: bank.product(x.repeat(7, 1), work=torch.zeros(3, device="cuda")),
        lambda: bank.product(x, out=torch.zeros(10, 99, device="cuda")), lambda: bank.product(A.Points8(5, 32)), lambda: bank.product(A.Points8(5, 64), m=6),
        lambda: bank.product_grad(x), lambda: bank.product_grad(torch.zeros(4, 100, device="cuda", dtype=torch.int32)),
        lambda: A.Points8(5000, 64).product_grad(torch.zeros(4, 5000, device="cuda"), work=torch.zeros(1, device="cuda")),
        lambda: A.KGraph.bruteforce_l2_points8(bank, 0), lambda: A.KGraph.bruteforce_l2_points8(bank, 10, n=10), lambda: A.KGraph.bruteforce_l2_points8(bank, 3, n=200),
    ]
    for f in bad:
        with pytest.raises(A.AnnembedError):
            f()
    from annembed_amd import _lib as L
    lib = L.load()
    assert lib.ae_points8_write(bank.handle, x.data_ptr(), 9, 10, 64, 0, None, None) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_write(bank.handle, x.data_ptr() + 2, 0, 9, 64, 0, None, None) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_write(bank.handle, None, 0, 10, 64, 0, None, None) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_write(None, x.data_ptr(), 0, 10, 64, 0, None, None) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_write(bank.handle, x.data_ptr(), 0, 10, 63, 0, None, None) == L.AE_ERR_INVALID_ARG
    assert b"stride" in lib.ae_last_error_message()
    many, c = x.repeat(7, 1), torch.zeros(70, 100, device="cuda")
    assert lib.ae_points8_product(bank.handle, 0, 100, many.data_ptr(), 0, 70, 64, c.data_ptr(), 0, 100, None, 0, None) == L.AE_ERR_INVALID_ARG
    assert b"scratch" in lib.ae_last_error_message()
    assert lib.ae_points8_read(bank.handle, 0, None, 0, None, 0, 0, None) == L.AE_OK


def test_strides_of_gigabytes(A):
    """rows of dc, of dx and of the product so far apart that a tile of them spans more than 32-bit offsets reach; few and more rows"""
    n, dim = 300, 130
    bank = A.Points8(n, dim)
    p = vectors(n, dim, 1)
    bank.write(p.cuda())
    pv = U.values(n64(p))
    step = 9_000_000
    for m in (3, 20, 70):
        room = torch.zeros((m - 1) * step + n, dtype=torch.bfloat16, device="cuda")
        dc = vectors(m, n, 2).bfloat16()
        far = room.as_strided((m, n), (step, 1))
        far.copy_(dc)
        got, want = n64(bank.product_grad(far)), n64(dc) @ pv
        assert (np.abs(got - want) <= product_bound(n64(dc), pv, 3 * n + 64, want, torch.float32)).all()
        x = vectors(m, dim, 3)
        xv = U.values(n64(x))
        bank.product(x.cuda(), out=far)
        assert (np.abs(n64(far) - xv @ pv.T) <= product_bound(xv, pv.T, dim, xv @ pv.T, torch.bfloat16, eights=True)).all()
        assert not room.as_strided((m - 1, step - n), (step, 1), n).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_that_ends_with_a_page(A, dtype):
    """an odd number of 16-bit values whose last one is the last of a page: the copies may not take the dword that it starts"""
    n, dim, m = 129, 40, 5
    bank = A.Points8(n, dim)
    p = vectors(n, dim, 1)
    bank.write(p.cuda())
    pv = U.values(n64(p))
    room = torch.full((8192,), float("nan"), dtype=dtype, device="cuda")
    end = 2048 * 3 - room.data_ptr() % 4096 // 2   # elements to a page's end
    dc = vectors(m, n, 2).to(dtype)
    for last in (end, end - 1):   # (the other one may, and what it takes there is NaN)
        view = room[last - m * n:last].view(m, n)
        view.copy_(dc)
        assert (view.data_ptr() + 2 * m * n) % 4096 == (0 if last == end else 4094)
        got, want = n64(bank.product_grad(view)), n64(dc) @ pv
        assert (np.abs(got - want) <= product_bound(n64(dc), pv, 3 * n + 64, want, torch.float32)).all()
        room.fill_(float("nan"))


def test_the_same_store_on_both_sides_and_views_of_it(A):
    """products of a store with itself, a part with another; the store's memory outlives the object that views of it came from"""
    x = vectors(200, 96, 1)
    bank = A.Points8(200, 96)
    bank.write(x.cuda())
    v = U.values(n64(x))
    got = n64(bank.product(bank, n=50, first=150, x_first=7, m=120))
    want = v[7:127] @ v[150:].T
    assert (np.abs(got - want) <= product_bound(v[7:127], v[150:].T, 96, want, torch.float32)).all()
    codes, scales = bank.codes(), bank.scales()
    keep = codes.float() * torch.exp2(scales.float() - 127)
    del bank
    other = A.Points8(200, 96)
    other.write(torch.ones(200, 96, device="cuda"))
    assert torch.equal(codes.float() * torch.exp2(scales.float() - 127), keep)


def test_rows_behind_the_last_point_do_not_count(A):
    """points behind the range that is asked for hold NaN, so do the rows' neighbours in memory"""
    bank = A.Points8(64, 100)
    bank.write(torch.full((64, 100), float("nan"), device="cuda"))
    p = vectors(20, 100, 1)
    bank.write(p.cuda(), first=16)
    pv = U.values(n64(p))
    for m in (2, 30, 70):
        room = torch.full((m + 2, 120), float("nan"), device="cuda")
        x = vectors(m, 100, 2)
        room[1:-1, 8:108] = x.cuda()
        xv = U.values(n64(x))
        for dtype in TYPES:
            got = n64(bank.product(room[1:-1, 8:108], n=20, first=16, dtype=dtype))
            fits = np.abs(xv @ pv.T) < (65000 if dtype == torch.float16 else np.inf)   # (beyond, f16 has its infinities)
            assert (np.abs(got - xv @ pv.T) <= product_bound(xv, pv.T, 100, xv @ pv.T, dtype, eights=dtype != torch.float32))[fits].all()
            wide = torch.full((m + 2, 33), float("nan"), dtype=dtype, device="cuda")
            dc = vectors(m, 20, 3).to(dtype)
            wide[1:-1, 5:25] = dc.cuda()
            got, want = n64(bank.product_grad(wide[1:-1, 5:25], n=20, first=16)), n64(dc) @ pv
            assert (np.abs(got - want) <= product_bound(n64(dc), pv, 3 * 20 + 64, want, torch.float32)).all()


@pytest.mark.parametrize("n,dim", [(4097, 40), (6000, 100), (6001, 100), (6000, 1500), (6001, 784)])
def test_slots_that_come_again_far_behind(A, n, dim):
    """repeated slots at every distance, on both sides of the number of rows up to which a workgroup looks for them itself"""
    cap = n // 3
    bank = A.Points8(cap, dim)
    x = vectors(n, dim, 5)
    rng = np.random.default_rng(n)
    slots = rng.integers(0, cap, n)
    slots[rng.random(n) < 0.1] = -1
    slots[0] = slots[n - 1] = 7
    bank.write(x.cuda(), slots=torch.from_numpy(slots).to(torch.int32).cuda())
    last = {s: i for i, s in enumerate(slots.tolist()) if s >= 0}
    at = sorted(last)
    v = U.values(n64(x[[last[s] for s in at]]))
    np.testing.assert_array_equal(n64(bank.read(slots=torch.tensor(at, dtype=torch.int32, device="cuda"))), v)
    rest = sorted(set(range(cap)) - set(at))
    assert not bank.read(slots=torch.tensor(rest, dtype=torch.int32, device="cuda")).any()
