"""Graphs of points some of which have no distances: NaN coordinates, and norms or distances that f32 does not have.  The graph of the definition --
squared distances summed in f32, the smallest (distance, index) -- or, where a point has too few distances, a refusal, whatever the number of neighbours
and of points that are left; and the next graph is as it should be."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    import annembed_amd as A
    from annembed_amd import _lib
    _lib.load()
    return A


def graph(x, k):
    """neighbours of the definition, or None"""
    f = np.zeros((len(x), len(x)), np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        for t in range(x.shape[1]):
            d = x[:, None, t] - x[None, :, t]
            f += d * d
    np.fill_diagonal(f, np.nan)
    f[~np.isfinite(f)] = np.inf
    if (np.isfinite(f).sum(1) < k).any():
        return None
    return np.argsort(f, 1, kind="stable")[:, :k]


@pytest.mark.parametrize("n,left,k", [(700, 0, 1), (700, 0, 7), (10, 3, 3), (10, 3, 2), (300, 2, 1), (300, 200, 12), (300, 40, 40), (300, 41, 40), (200, 60, 60), (300, 299, 5)])
@pytest.mark.parametrize("bad", [np.nan, 1e30])
def test_points_without_distances(A, n, left, k, bad):
    rng = np.random.default_rng(n + left)
    x = rng.normal(size=(n, 20)).astype(np.float32)
    gone = rng.permutation(n)[left:]
    x[gone, rng.integers(0, 20, len(gone))] = bad
    bank = A.Points8(n, 20)
    bank.write(torch.from_numpy(x).cuda())
    for make, points in ((lambda: A.KGraph.bruteforce_l2(x, k), x), (lambda: A.KGraph.bruteforce_l2_points8(bank, k), bank.read().cpu().numpy())):
        want = graph(points, k)
        if want is None:
            with pytest.raises(A.AnnembedError):
                make()
        else:
            np.testing.assert_array_equal(make().get_neighbours()[1].reshape(n, k), want)
    x = rng.normal(size=(n, 20)).astype(np.float32)
    bank.write(torch.from_numpy(x).cuda())
    got = A.KGraph.bruteforce_l2_points8(bank, min(k, n - 1)).get_neighbours()
    want = A.KGraph.bruteforce_l2(bank.read().cpu().numpy(), min(k, n - 1)).get_neighbours()
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
