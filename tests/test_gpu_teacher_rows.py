"""Every logit of a row counts, in every form of the teacher's loss: rows held in registers of each size, and rows in slices.

A row of equal logits sums to its length exactly (an exponential of 0 is 1, sums of integers below 2^24 are exact in any order), so ln sum is the
logarithm of the length, rounded once or twice: off by 2^-23 of itself at most, while a lost piece of 4 logits is 4 / length."""
import numpy as np
import pytest
import torch

from tests import points8_util as U

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
u = 2.0 ** -23
# a wave; 256 threads with 1, 2, 4 and 8 pieces; 512 and 1024 threads; slices, whose borders lie at multiples of 8 near 8192
COLS = [1, 3, 63, 64, 65, 255, 256, 257, 1000, 2049, 4097, 8191, 8200, 16383, 16385, 16391, 24577, 32767, 32769, 60000, 65535, 65537, 70001, 140001, 600007]


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def forms(A, s, idx, p, **more):
    """the statistics from the loss alone and with its gradient, and the three ways to the gradient"""
    loss, stats = A.teacher_loss(s, idx, p, **more)
    loss2, stats2, grad = A.teacher_loss(s, idx, p, grad=True, **more)
    return loss, stats, loss2, stats2, grad, A.teacher_grad(s, stats, idx, p, **more)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_no_logit_is_lost(A, cols, dtype):
    s = torch.zeros(3, cols, dtype=dtype, device="cuda")
    idx = torch.tensor([[0], [cols - 1], [cols // 2]], dtype=torch.int32, device="cuda")
    p = torch.ones(3, 1, device="cuda")
    loss, stats, loss2, stats2, grad, again = forms(A, s, idx, p)
    want = np.log(cols)
    for st in (stats, stats2):
        assert not st[:, 0].any() and (np.abs(st[:, 1].cpu().numpy() - want) <= u * want).all()
    for one in (loss, loss2):   # p = 1: the loss is ln sum
        assert (np.abs(one.cpu().numpy() - want) <= 2 * u * want).all()
    q = 1.0 / cols   # (the exponent's rounding, then the type's)
    for g in (grad, again):
        g = g.float().cpu().numpy()
        size = np.full((3, cols), q)
        size[np.arange(3), idx[:, 0].cpu().numpy()] -= 1.0
        off = np.abs(g - size)
        assert (off <= q * (want + 4) * 2 * u + np.abs(size) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [c for c in COLS if c >= 1000])
def test_what_a_row_has_left_stands_anywhere(A, cols, dtype):
    """-inf everywhere but in a few columns: the last 1 to 9, the first, and some around the borders of slices and pieces"""
    rng = np.random.default_rng(cols)
    per = -(-cols // max(1, min(-(-1024 // 24), -(-cols // 8192))))   # near a slice's length of 24 rows
    windows = [np.arange(cols - w, cols) for w in range(1, 10)] + [np.arange(0, 5)]
    for border in (per // 8 * 8, -(-per // 8) * 8, 8192, 2048, cols // 2, cols - 8, cols - 16):
        for lo in (border - 4, border):
            lo = min(max(lo, 0), cols - 4)
            windows.append(np.arange(lo, lo + 4))
    rows = len(windows)
    assert rows == 24
    s = np.full((rows, cols), -np.inf, np.float32)
    idx = np.zeros((rows, 2), np.int64)
    for r, w in enumerate(windows):
        s[r, w] = np.round(rng.normal(size=len(w)) * 8) / 4   # (numbers that every type has)
        idx[r] = w[0], w[-1]
    p = np.tile(np.float32([0.25, 0.5]), (rows, 1))
    loss, stats, grad = U.teacher(s, idx, p)
    got = forms(A, torch.from_numpy(s).to(dtype).cuda(), torch.from_numpy(idx).to(torch.int32).cuda(), torch.from_numpy(p).cuda())
    # at most 9 terms of 1 or less, each off by its argument (below 16) times u and 2 u more, the sum by 8 u: ln sum by 32 u; the loss by 0.75 of
    # that and its own terms
    for st in (got[1], got[3]):
        st = st.cpu().numpy()
        assert np.array_equal(st[:, 0], stats[:, 0]) and (np.abs(st[:, 1] - stats[:, 1]) <= 32 * u).all()
    for one in (got[0], got[2]):
        assert (np.abs(one.cpu().numpy() - loss) <= 64 * u).all()
    for g in (got[4], got[5]):
        g = g.float().cpu().numpy().astype(np.float64)
        assert (np.abs(g - grad) <= 96 * u + np.abs(grad) * torch.finfo(dtype).eps / 2).all()
        assert not g[np.isneginf(s)].any()


def test_a_row_of_more_than_2_to_the_31_columns(A):
    """columns beyond int32 are named by their 32 bits.  1024 slices of 2 million equal logits sum exactly, their join is off by 2^-24 a step: ln sum by 16 u"""
    cols = (1 << 31) + 100003
    s = torch.zeros(1, cols, dtype=torch.bfloat16, device="cuda")
    at = cols - 2
    idx = torch.tensor([[at - (1 << 32), 5]], dtype=torch.int32, device="cuda")
    p = torch.tensor([[0.75, 0.25]], device="cuda")
    loss, stats = A.teacher_loss(s, idx, p)
    want = np.log(cols)
    assert stats[0, 0] == 0 and abs(stats[0, 1].item() - want) <= (want + 16) * u
    entropy = 0.75 * np.log(0.75) + 0.25 * np.log(0.25)
    assert abs(loss.item() - (entropy + want)) <= 2 * (want + 16) * u
    loss2, stats2, grad = A.teacher_loss(s, idx, p, grad=True)
    assert torch.equal(loss, loss2) and torch.equal(stats, stats2)
    q = grad[0, 7].item()
    assert abs(q * cols - 1) <= 2.0 ** -8 and grad[0, at] == -0.75 and grad[0, 5] == -0.25 and (grad[0] == q).sum().item() == cols - 2
    A.teacher_grad(s, stats, idx, p, out=grad)
    assert grad[0, 7].item() == q and grad[0, at] == -0.75 and grad[0, 5] == -0.25 and (grad[0] == q).sum().item() == cols - 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [16, 64, 1024, 4096, 8192, 16384, 32768, 131072])
@pytest.mark.parametrize("k", [1, 63, 64, 65, 130, 1023, 1024])
def test_equal_columns_of_long_lists_add_up(A, cols, k, dtype):
    """entries of 2^-12 on few columns of a row of equal logits: a listed column's gradient is q k 2^-12 less its count of them, off by some u of either;
    a lost entry is 2^-12"""
    rng = np.random.default_rng(k)
    rows = 5
    few = rng.integers(0, cols, (rows, max(1, k // 5)))
    idx = np.take_along_axis(few, rng.integers(0, few.shape[1], (rows, k)), 1)
    idx[rng.random((rows, k)) < 0.1] = -1
    idx[4] = cols - 1
    used = (idx >= 0)
    p = np.where(used, np.float32(2.0 ** -12), np.float32(np.nan)).astype(np.float32)   # (what stands in an empty place is not looked at)
    s = torch.zeros(rows, cols, dtype=dtype, device="cuda")
    di, dp = torch.from_numpy(idx).to(torch.int32).cuda(), torch.from_numpy(p).cuda()
    got = forms(A, s, di, dp)
    P, q = used.sum(1) * 2.0 ** -12, 1.0 / cols
    want = np.repeat((P * q)[:, None], cols, 1)
    for r in range(rows):
        np.subtract.at(want[r], idx[r][used[r]], 2.0 ** -12)
    ln = np.log(cols)
    for g in got[4:]:
        off = np.abs(g.float().cpu().numpy() - want)
        assert (off <= 64 * u * (P * q)[:, None] + (u + torch.finfo(dtype).eps / 2) * np.abs(want) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()
    loss = P * (np.log(2.0 ** -12) + ln)
    for one in (got[0], got[2]):
        assert (np.abs(one.cpu().numpy() - loss) <= 4 * u * P * (ln + 9)).all()
    e = s.clone()   # in place
    assert torch.equal(A.teacher_loss(e, di, dp, grad=e)[2], got[4])
    e = s.clone()
    assert torch.equal(A.teacher_grad(e, got[1], di, dp, out=e), got[5])
