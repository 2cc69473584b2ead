"""What the 8-bit store and the teacher's loss decide without a GPU: the refusals of the C entry points, the checks of the torch wrappers,
scratch sizes, and the oracles that the GPU tests compare with."""
import ctypes as C
import subprocess
import sys

import numpy as np
import pytest
import torch

import annembed_amd as A
from annembed_amd import _lib as L
from annembed_amd import points8 as P
from tests import points8_util as U


def test_the_package_does_without_torch():
    code = "import sys, annembed_amd; assert 'torch' not in sys.modules; annembed_amd.Points8; assert 'torch' in sys.modules"
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(__import__("pathlib").Path(__file__).parent.parent))
    with pytest.raises(AttributeError):
        A.points16
    assert {"Points8", "teacher_loss", "teacher_grad"} <= set(A.__all__)


# arguments of ae_teacher_loss that are in order; the addresses are looked at, never followed: each call below is refused before it launches
GOOD = dict(logits=4096, type=0, rows=4, cols=50, ld=50, idx=4096, list=4096, k=3, ldk=3, kind=0, temperature=1.0, weight=None, loss=4096, stats=4096, grad=8192, ldg=50,
            work=None, work_bytes=0, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(type=3), "type"), (dict(logits=None), "NULL"), (dict(logits=4098), "aligned"), (dict(logits=4097, type=1), "aligned"), (dict(ld=49), "stride"),
    (dict(idx=None), "list"), (dict(list=None), "list"), (dict(idx=4098), "aligned"), (dict(list=4097), "aligned"), (dict(k=0), "entries"), (dict(k=1025, ldk=1025), "entries"),
    (dict(ldk=2), "stride"), (dict(ldk=1 << 39), "out of range"), (dict(kind=2), "kind"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=1e-40), "temperature"),
    (dict(cols=0, ld=50), "columns"), (dict(cols=(1 << 32) - 1, ld=1 << 32), "columns"), (dict(rows=1 << 24), "more than one call"), (dict(rows=1 << 14, cols=1 << 30, ld=1 << 30), "more than one call"),
    (dict(ld=1 << 39), "out of range"), (dict(grad=4097), "aligned"), (dict(ldg=49), "stride"), (dict(grad=4096, ldg=51), "in place"), (dict(loss=None), "NULL"),
    (dict(stats=None), "NULL"), (dict(loss=4097), "aligned"), (dict(stats=4098), "aligned"),
])
def test_teacher_loss_refuses(change, word):
    lib = L.load()
    assert lib.ae_teacher_loss(*{**GOOD, **change}.values()) == L.AE_ERR_INVALID_ARG
    assert word in lib.ae_last_error_message().decode()


@pytest.mark.parametrize("change,word", [
    (dict(type=3), "type"), (dict(logits=None), "NULL"), (dict(stats=None), "NULL"), (dict(stats=4097), "aligned"), (dict(grad=None), "NULL"), (dict(grad=4096, ldg=60), "in place"),
    (dict(k=2000, ldk=2000), "entries"), (dict(temperature=0.0), "temperature"), (dict(cols=60), "stride"),
])
def test_teacher_grad_refuses(change, word):
    lib = L.load()
    a = {**GOOD, **change}
    args = [a[n] for n in ("logits", "type", "rows", "cols", "ld", "stats", "idx", "list", "k", "ldk", "kind", "temperature", "weight", "grad", "ldg", "stream")]
    assert lib.ae_teacher_grad(*args) == L.AE_ERR_INVALID_ARG
    assert word in lib.ae_last_error_message().decode()


def test_no_rows_is_a_call_that_does_nothing():
    lib = L.load()
    assert lib.ae_teacher_loss(*{**GOOD, "rows": 0, "logits": None, "idx": None, "loss": None}.values()) == L.AE_OK
    assert lib.ae_teacher_grad(None, 1, 0, 50, 50, None, None, None, 3, 3, 0, 1.0, None, None, 50, None) == L.AE_OK


def test_scratch_of_the_loss():
    lib, need = L.load(), C.c_uint64()
    for rows, cols in [(0, 5), (1, 1), (300, 784), (4096, 16383)]:
        assert lib.ae_teacher_loss_work(rows, cols, C.byref(need)) == L.AE_OK and need.value == 0
    for rows, cols in [(1, 16384), (1, 10 ** 6), (300, 60000), (4096, 32768), (1, (1 << 32) - 2)]:
        assert lib.ae_teacher_loss_work(rows, cols, C.byref(need)) == L.AE_OK
        assert need.value % (8 * rows) == 0 and 1 <= need.value // (8 * rows) <= 1024
    assert lib.ae_teacher_loss_work(5, 0, C.byref(need)) == L.AE_ERR_INVALID_ARG
    assert lib.ae_teacher_loss_work(5, 10, None) == L.AE_ERR_INVALID_ARG


def test_store_refuses_without_a_store():
    lib, n, p = L.load(), C.c_uint64(), C.c_void_p()
    assert lib.ae_points8_info(None, None, None, None, None) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_device(None, C.byref(p), C.byref(p)) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_product_work(None, 1, 1, C.byref(n)) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_product_grad_work(None, 1, 1, 0, C.byref(n)) == L.AE_ERR_INVALID_ARG
    assert lib.ae_points8_destroy(None) == L.AE_OK
    for bad in [(0, 4), (4, 0), (1 << 32, 4), (4, (1 << 20) + 1), (-1, 4)]:
        with pytest.raises(A.AnnembedError) as e:
            A.Points8(*bad)
        assert e.value.code == L.AE_ERR_INVALID_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="what is said where there is no GPU")
def test_without_a_gpu_the_calls_say_so():
    lib, h = L.load(), C.c_void_p()
    assert lib.ae_points8_create(4, 4, C.byref(h)) == L.AE_ERR_NO_DEVICE
    assert lib.ae_points8_write(None, None, 0, 0, 0, 0, None, None) == L.AE_ERR_NO_DEVICE
    assert lib.ae_teacher_loss(*GOOD.values()) == L.AE_ERR_NO_DEVICE
    with pytest.raises(A.AnnembedError) as e:
        A.Points8(4, 4)
    assert e.value.code == L.AE_ERR_NO_DEVICE
    s, i, t = torch.zeros(2, 5), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    for f in (lambda: A.teacher_loss(s, i, t), lambda: A.teacher_grad(s, torch.zeros(2, 2), i, t)):
        with pytest.raises(A.AnnembedError, match="GPU"):
            f()


CPU = torch.device("cpu")


def test_rows_of_the_wrappers():
    t = torch.zeros(6, 10)
    assert P._rows(t, "t", CPU) == (t.data_ptr(), L.AE_TYPE_F32, 10)
    assert P._rows(t[:, 3:7], "t", CPU)[1:] == (L.AE_TYPE_F32, 10) and P._rows(t[:, 3:7], "t", CPU)[0] == t.data_ptr() + 12
    assert P._rows(t[::2].bfloat16()[::3], "t", CPU)[1] == L.AE_TYPE_BF16
    assert P._rows(t[::2], "t", CPU)[2] == 20
    assert P._rows(t[:1].expand(1, 10), "t", CPU)[2] == 10
    assert P._rows(t[:1, :1].t(), "t", CPU)[2] >= 1
    assert P._rows(t[:, :1], "t", CPU)[2] == 10   # one element a row: its inner stride does not matter
    assert P._rows(t[:0], "t", CPU)[2] == 10
    for bad in (t[0], t.double(), t.t(), t[:1].expand(6, 10), t[:, ::2], t.numpy(), None, t.to(torch.int32)):
        with pytest.raises(A.AnnembedError):
            P._rows(bad, "t", CPU)
    with pytest.raises(A.AnnembedError):
        P._rows(t, "t", torch.device("cuda", 0))
    with pytest.raises(A.AnnembedError):
        P._rows(t, "t", CPU, (6, 9))


def test_lists_and_vectors_of_the_wrappers():
    i, v = torch.zeros(6, 4, dtype=torch.int32), torch.zeros(6, 4)
    assert P._list(i, v, 6, CPU)[2:] == (4, 4)
    assert P._list(i[::2], v[::2], 3, CPU)[2:] == (4, 8)
    assert P._list(i[:, 1:3], v[:, 1:3], 6, CPU)[2:] == (2, 4)
    assert P._list(i[:1], v[:1].clone(), 1, CPU)[2:] == (4, 4)
    for bi, bv, rows in [(i.long(), v, 6), (i, v.double(), 6), (i, v[:, :3], 6), (i, v, 5), (i, v.t().contiguous().t(), 6), (i[:, ::2], v[:, ::2], 6), (i[0], v[0], 4), (i, None, 6),
                         (None, v, 6), (i[:1].expand(6, 4), v[:1].expand(6, 4), 6), (i[:1, ::2], v[:1, ::2], 1)]:
        with pytest.raises(A.AnnembedError):
            P._list(bi, bv, rows, CPU)
    w = torch.zeros(6)
    assert P._vector(None, "w", CPU, 6, P._F32) is None
    assert P._vector(w, "w", CPU, 6, P._F32) == w.data_ptr()
    for bad in (w[:5], w.double(), w.view(2, 3), torch.zeros(12)[::2], [0.0] * 6):
        with pytest.raises(A.AnnembedError):
            P._vector(bad, "w", CPU, 6, P._F32)
    for bad in ("top", None, 0):
        with pytest.raises(A.AnnembedError):
            P._kind(bad)


def test_the_oracles_format_is_e4m3():
    """the oracle's codes are those of torch's own 8-bit type under the oracle's scales, for magnitudes over the whole range of f32"""
    rng = np.random.default_rng(3)
    x = (rng.normal(size=(64, 300)) * np.exp2(rng.integers(-12, 13, (64, 300)))).astype(np.float32)
    x *= np.exp2(rng.integers(-100, 100, (64, 1))).astype(np.float32)
    x[3] = 0
    x[4, :128] = 448.0
    x[5, :128] = np.nextafter(np.float32(448.0), np.float32(1000.0))
    codes, bytes_ = U.quantise(x)
    z = torch.from_numpy(x).double() * torch.exp2(127 - torch.from_numpy(bytes_).double()).repeat_interleave(U.BLOCK, 1)[:, :300]
    assert (z.abs() <= 448).all() and torch.equal(z, z.float().double())
    assert torch.equal(z.float().to(torch.float8_e4m3fn).double(), torch.from_numpy(codes))
    assert bytes_[4, 0] == 127 and bytes_[5, 0] == 128 and (bytes_[3] == 1).all()
    assert (np.abs(U.values(x) - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -10 * np.ldexp(1.0, bytes_ - 127).repeat(U.BLOCK, 1)[:, :300]).all()


def test_the_oracles_gradient_is_its_losses():
    """central differences in 64 bits, h = 2^-13: off by h^2 / 6 of a third derivative (at most 2 w P / T^3) and by the loss's rounding over h"""
    rng = np.random.default_rng(4)
    s = 2 * rng.normal(size=(3, 20))
    idx = np.array([[1, 5, 5], [-1, 0, 19], [7, -1, -1]])
    h = 2.0 ** -13
    for kind, vals in (("proba", rng.uniform(0.1, 0.5, (3, 3))), ("logits", rng.normal(size=(3, 3)))):
        for temp in (0.7, 2.0):
            w = np.array([1.0, 0.25, -2.0])
            _, _, g = U.teacher(s, idx, vals, kind, temp, w)
            for v in range(20):
                up, down = s.copy(), s.copy()
                up[:, v] += h
                down[:, v] -= h
                d = (U.teacher(up, idx, vals, kind, temp, w)[0] - U.teacher(down, idx, vals, kind, temp, w)[0]) / (2 * h)
                assert (np.abs(d - g[:, v]) <= h * h / 3 * 2 * 1.5 / temp ** 3 + 1e-11).all()
