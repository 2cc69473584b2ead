"""GPU tests of the teacher's loss and its gradient against the definition in 64 bits (tests/points8_util.py).

Tolerances, u = 2^-23.  The sum of exponentials runs over at most cols / 64 terms a lane and 16 joins, each off by u, an exponential by
2 u + |argument| u (the argument's rounding), so ln sum is off by (cols / 64 + 32 + a) u, a the mean |argument| under the softmax, taken as 8
/ T or the row's largest where the row is flat; a loss by w P times that plus 4 u of itself.  A gradient: q is off by that plus
2 |argument| u relative, then eps / 2 of the type."""
import numpy as np
import pytest
import torch

from tests import points8_util as U

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
u = 2.0 ** -23


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def n64(t):
    return t.detach().cpu().float().numpy().astype(np.float64)


def make(rows, cols, k, seed, dtype, kind):
    rng = np.random.default_rng(seed)
    s = torch.from_numpy((3 * rng.normal(size=(rows, cols))).astype(np.float32)).to(dtype)
    idx = rng.integers(0, cols, (rows, k))
    t = rng.normal(size=(rows, k)).astype(np.float32)
    if kind == "proba":
        e = np.exp(t)
        t = (e / e.sum(1, keepdims=True)).astype(np.float32)
    return s, idx, t


def dev(idx, t):
    return torch.from_numpy(idx).to(torch.int32).cuda(), torch.from_numpy(t).cuda()


def assert_close(s, idx, t, kind, temp, weight, got, dtype):
    loss, stats, grad = U.teacher(n64(s), idx, t, kind, temp, weight)
    sv = n64(s)
    w = np.ones(len(loss)) if weight is None else np.abs(weight)
    P = np.where(idx >= 0, t if kind == "proba" else 1.0 / max(1, idx.shape[1]), 0).sum(1) if kind == "proba" else np.ones(len(loss))
    arg = np.nan_to_num(sv.max(1, keepdims=True, initial=-np.inf, where=np.isfinite(sv)) - sv, nan=0, posinf=0, neginf=0) / temp
    base = (sv.shape[1] / 64 + 40 + np.minimum(arg.max(1), 60)) * u
    if "loss" in got:
        g = n64(got["loss"])
        fine = np.isfinite(loss)
        np.testing.assert_array_equal(np.isnan(g), np.isnan(loss))
        np.testing.assert_array_equal(g[~fine & ~np.isnan(loss)], loss[~fine & ~np.isnan(loss)])
        # p ln p and p s terms of either sign: |p ln p| + |p arg| bounds what cancels
        size = w * (np.abs(P) * (base + 8 * u * (2 + arg.max(1)))) + 4 * u * np.abs(loss)
        assert (np.abs(g - loss)[fine] <= size[fine]).all(), (np.abs(g - loss) / size).max()
    if "grad" in got:
        g = n64(got["grad"])
        nan = np.isnan(grad)
        np.testing.assert_array_equal(np.isnan(g), nan)
        q = np.abs(grad) + 2 * (w / temp)[:, None] * np.abs(P)[:, None] * np.exp(-np.minimum(arg - 0 * arg, 700)) / 1.0
        tol = q * (base[:, None] + 4 * (arg + 2) * u) + torch.finfo(dtype).eps / 2 * np.abs(grad) + float(torch.finfo(dtype).smallest_normal)
        assert (np.abs(g - grad)[~nan] <= tol[~nan]).all(), np.nanmax(np.abs(g - grad) / tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["proba", "logits"])
@pytest.mark.parametrize("rows,cols,k,temp", [(1, 1, 1, 1.0), (3, 7, 2, 0.5), (5, 64, 12, 1.0), (2, 257, 64, 2.0), (70, 1000, 12, 1.0), (4, 2048, 1, 4.0), (3, 8200, 33, 1.0), (300, 777, 5, 0.7),
                                              (2, 33000, 12, 1.0), (1, 60000, 12, 1.0), (2, 140001, 1024, 2.0), (1, 600000, 12, 1.0)])
def test_loss_and_gradient(A, rows, cols, k, temp, kind, dtype):
    s, idx, t = make(rows, cols, k, 1, dtype, kind)
    d = s.cuda()
    di, dt = dev(idx, t)
    loss, stats, grad = A.teacher_loss(d, di, dt, teacher=kind, temperature=temp, grad=True)
    assert_close(s, idx, t, kind, temp, None, {"loss": loss, "grad": grad}, dtype)
    loss2, stats2 = A.teacher_loss(d, di, dt, teacher=kind, temperature=temp)
    assert torch.equal(loss, loss2) and torch.equal(stats, stats2)
    up = np.random.default_rng(5).normal(size=rows).astype(np.float32)
    g = A.teacher_grad(d, stats, di, dt, torch.from_numpy(up).cuda(), teacher=kind, temperature=temp)
    assert_close(s, idx, t, kind, temp, up.astype(np.float64), {"grad": g}, dtype)
    own = A.teacher_grad(d, stats, di, dt, teacher=kind, temperature=temp)
    assert_close(s, idx, t, kind, temp, None, {"grad": own}, dtype)
    # in place, both ways
    e = d.clone()
    assert torch.equal(A.teacher_loss(e, di, dt, teacher=kind, temperature=temp, grad=e)[2], grad) and torch.equal(e, grad)
    e = d.clone()
    assert torch.equal(A.teacher_grad(e, stats, di, dt, teacher=kind, temperature=temp, out=e), own)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 5000, 70001])
def test_masks_and_empty_rows(A, dtype, cols):
    """-inf and lowest logits, rows of them, lists that are empty, repeated, outside, of zero probability; weight 0 over NaN"""
    s, idx, t = make(16, cols, 6, 2, dtype, "proba")
    low = torch.finfo(dtype).min
    weight = np.ones(16, np.float32)
    s[0, :] = float("-inf")                         # nothing left
    s[1, 5:] = float("-inf"); idx[1] = 0, 1, 2, 3, 4, 4
    s[2, :] = low                                   # all masked by the lowest value: uniform
    s[3, 10:] = low; idx[3] = 0, 1, 2, 3, 3, 3
    idx[4] = -1                                     # an empty list
    idx[5, 1:] = -1; t[5, 1:] = np.nan              # what stands in an empty place is not looked at
    idx[6] = 7                                      # one column six times
    idx[7, 2] = cols                                # outside the row
    s[8, 3] = float("nan")
    s[9, 3] = float("inf")
    s[10, :] = float("nan"); weight[10] = 0; idx[10] = cols + 5   # padding
    s[11, 4] = float("-inf"); idx[11, 0] = 4        # the teacher wants what the student rules out
    t[12] = 0                                       # a list of nothing
    s[13, 4] = float("-inf"); idx[13, 0] = 4; t[13, 0] = 0
    t[14] *= 0.25                                   # a truncated list
    weight[15] = -2.5
    di, dt = dev(idx, t)
    loss, stats, grad = A.teacher_loss(s.cuda(), di, dt, row_weight=torch.from_numpy(weight).cuda(), grad=True)
    assert_close(s, idx, t, "proba", 1.0, weight, {"loss": loss, "grad": grad}, dtype)
    assert loss[11].item() == float("inf") and not loss[[0, 4, 10, 12]].any() and not grad[[0, 10]].any()
    up = weight.copy()
    g = A.teacher_grad(s.cuda(), stats, di, dt, torch.from_numpy(up).cuda())
    assert torch.equal(torch.nan_to_num(g, nan=5.0), torch.nan_to_num(grad, nan=5.0))
    tl = np.where(idx >= 0, 3 * t, 0).astype(np.float32)
    tl[14] = -np.inf                                # no entry of the teacher's either
    tl[15, 1:] = -np.inf
    loss, _, grad = A.teacher_loss(s.cuda(), di, torch.from_numpy(tl).cuda(), teacher="logits", row_weight=torch.from_numpy(weight).cuda(), grad=True)
    assert_close(s, idx, tl, "logits", 1.0, weight, {"loss": loss, "grad": grad}, dtype)


def test_strides(A):
    s, idx, t = make(9, 501, 5, 3, torch.bfloat16, "proba")
    wide = torch.zeros(9, 600, dtype=torch.bfloat16, device="cuda")
    view = wide[:, 7:508]
    view.copy_(s)
    iw, tw = torch.full((9, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(9, 8, device="cuda")
    iw[:, :5], tw[:, :5] = dev(idx, t)
    out = torch.full((9, 640), 3.0, dtype=torch.bfloat16, device="cuda")
    loss, _, _ = A.teacher_loss(view, iw[:, :5], tw[:, :5], grad=out[:, 9:510])
    want = A.teacher_loss(s.cuda(), *dev(idx, t), grad=True)
    assert torch.equal(loss, want[0]) and torch.equal(out[:, 9:510], want[2])
    assert (out[:, :9] == 3).all() and (out[:, 510:] == 3).all()
    A.teacher_loss(view, iw[:, :5], tw[:, :5], grad=view)
    assert torch.equal(view, want[2]) and not wide[:, :7].any() and not wide[:, 508:].any()
    loss0, _, g0 = A.teacher_loss(torch.zeros(0, 5, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, 2, device="cuda"), grad=True)
    assert loss0.shape == (0,) and g0.shape == (0, 5)


def test_offsets_past_32_bits(A):
    s, idx, t = make(3, 1000, 5, 4, torch.bfloat16, "proba")
    wide = torch.zeros(2 * (1 << 31) + 1000, dtype=torch.bfloat16, device="cuda")
    view = wide.as_strided((3, 1000), (1 << 31, 1))
    view.copy_(s)
    want = A.teacher_loss(s.cuda(), *dev(idx, t), grad=True)
    got = A.teacher_loss(view, *dev(idx, t), grad=view)
    assert torch.equal(got[0], want[0]) and torch.equal(view, want[2])


def test_gradient_against_differences(A):
    """central differences of the loss itself, step h = 2^-6: off by h^2 / 6 times a third derivative of at most 1 (P = 1, T = 1), and by the loss's
    own rounding, 64 u (1 + loss), over h"""
    s, idx, t = make(4, 50, 6, 6, torch.float32, "logits")
    di, dt = dev(idx, t)
    d = s.cuda()
    loss, _, g = A.teacher_loss(d, di, dt, teacher="logits", grad=True)
    h = 2.0 ** -6
    for v in list(range(0, 50, 7)) + idx[0].tolist():
        a, b = d.clone(), d.clone()
        a[:, v] += h
        b[:, v] -= h
        la, lb = A.teacher_loss(a, di, dt, teacher="logits")[0], A.teacher_loss(b, di, dt, teacher="logits")[0]
        diff = (la - lb) / (n64(a[:, v]) - n64(b[:, v]) if False else 2 * h)
        assert (diff - g[:, v]).abs().max().item() <= h * h / 6 + 64 * u * (1 + loss.max().item()) / h


def test_graph_capture(A):
    s, idx, t = make(20, 3000, 12, 7, torch.float32, "proba")
    d = s.cuda()
    di, dt = dev(idx, t)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, stats, grad = A.teacher_loss(d, di, dt, grad=True)
            again = A.teacher_grad(d, stats, di, dt)
        graphs.append(g)
        outs.append((loss, stats, grad, again))
    for turn in range(3):
        d.copy_(make(20, 3000, 12, 70 + turn, torch.float32, "proba")[0])
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        loss, stats, grad = A.teacher_loss(d, di, dt, grad=True)
        eager = loss, stats, grad, A.teacher_grad(d, stats, di, dt)
        for o in outs:
            for a, b in zip(o, eager):
                assert torch.equal(a, b)


def test_refusals(A):
    s, i, t = torch.zeros(4, 50, device="cuda"), torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.ones(4, 3, device="cuda")
    stats = A.teacher_loss(s, i, t)[1]
    bad = [
        lambda: A.teacher_loss(s.cpu(), i, t), lambda: A.teacher_loss(s, i.cpu(), t), lambda: A.teacher_loss(s.double(), i, t), lambda: A.teacher_loss(s, i.long(), t),
        lambda: A.teacher_loss(s, i, t.bfloat16()), lambda: A.teacher_loss(s, i[:3], t), lambda: A.teacher_loss(s, i, t[:, :2]), lambda: A.teacher_loss(s, i, t, teacher="top"),
        lambda: A.teacher_loss(s, i, t, temperature=0.0), lambda: A.teacher_loss(s, i, t, temperature=float("nan")), lambda: A.teacher_loss(s, i, t, row_weight=torch.ones(3, device="cuda")),
        lambda: A.teacher_loss(s, i, t, grad=torch.zeros(4, 49, device="cuda")), lambda: A.teacher_loss(s, i, t, grad=torch.zeros(4, 50, device="cuda", dtype=torch.bfloat16)),
        lambda: A.teacher_loss(s, i[:, :0], t[:, :0]), lambda: A.teacher_loss(s, i.repeat(1, 342), t.repeat(1, 342)), lambda: A.teacher_loss(s.t(), i, t),
        lambda: A.teacher_loss(s, i, t.t().contiguous().t()), lambda: A.teacher_grad(s, stats[:3], i, t), lambda: A.teacher_grad(s, stats, i, t, torch.ones(5, device="cuda")),
        lambda: A.teacher_grad(s, stats, i, t, out=torch.zeros(4, 50)), lambda: A.teacher_loss(s[:, :0], i, t),
    ]
    for n, f in enumerate(bad):
        with pytest.raises(A.AnnembedError):
            f()
            print("call", n, "went through")


def test_together(A):
    """a bank written in 8 bits, its graph's rows as the teacher's lists, an encoder's batch: logits, loss, gradients -- the whole chain in 64 bits.
    dlogits: as above; dq sums n of them times values held, so their tolerances add up times |p|"""
    rng = np.random.default_rng(11)
    n, dim, k, m = 900, 96, 8, 40
    centres = rng.normal(size=(6, dim))
    x = (centres[rng.integers(0, 6, n)] + 0.4 * rng.normal(size=(n, dim))).astype(np.float32) * 0.3
    bank = A.Points8(n, dim)
    for lo in range(0, n, 256):
        bank.write(torch.from_numpy(x[lo:lo + 256]).cuda(), first=lo)
    graph = A.KGraph.bruteforce_l2_points8(bank, k)
    proba, _ = A.to_proba_edges(graph, 1.0, 1.0).get()
    indptr, nbr, _ = graph.get_neighbours()
    batch = rng.permutation(n)[:m]
    idx = np.stack([nbr[indptr[b]:indptr[b + 1]] for b in batch]).astype(np.int64)
    p = np.stack([proba[indptr[b]:indptr[b + 1]] for b in batch]).astype(np.float32)
    q = torch.from_numpy(x[batch] + 0.05 * rng.normal(size=(m, dim)).astype(np.float32))
    logits = bank.product(q.cuda())
    pv, qv = U.values(x), U.values(q.numpy())
    want = qv @ pv.T
    off = dim * u * (np.abs(qv) @ np.abs(pv.T))
    assert (np.abs(n64(logits) - want) <= off).all()
    di, dt = dev(idx, p)
    loss, stats, dlogits = A.teacher_loss(logits, di, dt, grad=True)
    assert_close(logits.cpu(), idx, p, "proba", 1.0, None, {"loss": loss, "grad": dlogits}, torch.float32)
    dq = bank.product_grad(dlogits)
    wl, _, wg = U.teacher(want, idx, p)
    assert np.abs(n64(loss) - wl).max() <= 1e-4 and np.abs(n64(dq) - wg @ pv).max() <= 1e-4 * np.abs(wg @ pv).max()
    low = bank.product_grad(dlogits.bfloat16())
    size = np.abs(wg) @ np.abs(pv)
    assert (np.abs(n64(low) - n64(dq)) <= (2.0 ** -8 + 1e-5) * size + 1e-6).all()
    # a step against the gradient lowers what the loss is to first order
    step = 0.5
    moved = U.teacher(want - step * wg, idx, p)[0]
    assert (moved < wl).all()
