"""Both ends of the range in grouped products of float32 rows: finite products of large and of small numbers are finite and exact,
infinities and NaN come out as a product in 32 bits gives them, and sums that overflow become infinite, whichever kernel takes the
call.  The bounds are those of ``grouped_rows.sum_bound``."""
import pytest
import torch

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def ops():
    import qml_lightning_b200  # noqa: F401
    return torch.ops.qml_lightning_b200


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def same_kind(got, exact):
    """NaN where the definition gives NaN, the same infinity where it gives one (or a sum beyond the range), finite elsewhere."""
    want = exact.float()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], want[inf])


# (few rows, many rows) x (depths inside and beyond one stretch, odd widths)
@pytest.mark.parametrize('n', [60, 3000, 20001])
@pytest.mark.parametrize('K,N', [(64, 32), (63, 31), (200, 260), (336, 128)])
def test_infinities_keep_their_sign(n, K, N):
    g = gen(n + K)
    x, W = torch.randn(n, K, generator=g, device=DEV), torch.randn(2, K, N, generator=g, device=DEV)
    dy = torch.randn(n, N, generator=g, device=DEV)
    inf, nan = float('inf'), float('nan')
    x[3, 1], x[5, K - 1], x[7, 0], x[7, 1], x[9, 2], x[n - 1, 0] = inf, -inf, inf, -inf, nan, inf
    W[0, 2, 4], W[1, K - 1, N - 1], W[0, 1, 6] = inf, -inf, 0.0                       # an infinity times zero is NaN
    x[11, 2] = 0.0
    dy[2, 3], dy[4, 0], dy[n - 2, N - 1] = inf, nan, -inf
    x[13], x[15] = inf, nan                                                          # whole rows
    start = R.start_of([n // 2, n - n // 2], DEV)
    bound = R.groups_of(start, n)
    for got, parts in ((ops().grouped_matmul(x, W, start), [x[a:b].double() @ W[e].double() for e, (a, b) in enumerate(bound)]),
                       (ops().grouped_matmul(dy, W, start, True), [dy[a:b].double() @ W[e].double().T for e, (a, b) in enumerate(bound)])):
        exact = torch.cat(parts)
        same_kind(got, exact)
        ok = exact.isfinite()
        assert R.relative(got[ok], exact[ok]) < (max(K, N) ** 0.5 + 16) * R.U
    dW = ops().grouped_matmul_wgrad(x, dy, start)
    exact = torch.stack([x[a:b].double().T @ dy[a:b].double() for a, b in bound])
    same_kind(dW, exact)
    ok = exact.isfinite()
    assert not ok.any() or R.relative(dW[ok], exact[ok]) < (n ** 0.5 + 16) * R.U


@pytest.mark.parametrize('n', [60, 3000])
def test_sums_beyond_the_range(n):
    """Products whose sum leaves the range are infinite with its sign; their neighbours are untouched."""
    g = gen(5)
    K, N = 130, 48
    x, W = torch.rand(n, K, generator=g, device=DEV) + 0.5, torch.rand(1, K, N, generator=g, device=DEV) + 0.5
    x[10] *= 3e38 / 2
    x[11] *= -3e38 / 2
    start = R.start_of([n], DEV)
    y = ops().grouped_matmul(x, W, start)
    assert (y[10] == float('inf')).all() and (y[11] == -float('inf')).all()
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[10:12] = False
    exact, mag = R.product(x[rest], W, R.start_of([n - 2], DEV))
    R.assert_within(y[rest], exact, R.sum_bound(exact, mag, K, torch.float32), 'y')


@pytest.mark.parametrize('n', [60, 3000])
def test_largest_numbers(n):
    """Numbers that the nearest 8-bit significand lies beyond the range of."""
    top = torch.finfo(torch.float32).max
    x, W = torch.zeros(n, 70, device=DEV), torch.zeros(1, 70, 40, device=DEV)
    x[:, 0], x[1::2, 0], W[0, 0] = top, -top, 0.5
    x[:, 69], W[0, 69] = 1.0, 1.0
    start = R.start_of([n], DEV)
    exact, mag = R.product(x, W, start)
    y = ops().grouped_matmul(x, W, start)
    R.assert_within(y, exact, R.sum_bound(exact, mag, 2, torch.float32), 'y')
    dy = torch.zeros(n, 40, device=DEV)
    dy[1], dy[2, 3] = 0.5, 0.25
    exact, mag, terms = R.wgrad(x, dy, start)
    R.assert_within(ops().grouped_matmul_wgrad(x, dy, start), exact, R.sum_bound(exact, mag, terms, torch.float32), 'dW')


def test_everything_not_finite():
    """Training that has diverged: all values NaN, or all infinite, take no more than a moment and give what they should."""
    n, K, N = 30000, 336, 128
    start = R.start_of([n - 500, 500], DEV)
    ones = lambda v, *s: torch.full(s, v, device=DEV)  # noqa: E731
    for value in (float('nan'), float('inf')):
        y = ops().grouped_matmul(ones(value, n, K), ones(1.0, 2, K, N), start)
        dW = ops().grouped_matmul_wgrad(ones(value, n, K), ones(1.0, n, N), start)
        dx = ops().grouped_matmul(ones(1.0, n, N), ones(-value, 2, K, N), start, True)
        if value != value:
            assert y.isnan().all() and dW.isnan().all() and dx.isnan().all()
        else:
            assert (y == value).all() and (dW == value).all() and (dx == -value).all()
    from qml_lightning_b200 import cabi
    assert cabi.tc_timeouts() == 0


@pytest.mark.parametrize('n', [200, 3000])
@pytest.mark.parametrize('a,b', [(1e33, 1e-20), (1e37, 1e-30), (3e38, 1e-38), (1e-30, 1e20), (1e-37, 1e30), (1e18, 1e18)])
def test_values_near_the_ends_of_the_range(n, a, b):
    """Finite products of large and of small values are finite and as exact as others, for few rows and for many."""
    g = gen(4)
    K, N = 100, 64

    def values(size, *shape):                                          # magnitudes between a quarter of the size and the size
        v = torch.rand(shape, generator=g, device=DEV) * 0.75 + 0.25
        return v * torch.where(torch.rand(shape, generator=g, device=DEV) < 0.5, -1.0, 1.0) * size

    start = R.start_of([n // 2, n - n // 2 - 3], DEV)
    x, W, V, dy = values(a, n, K), values(b, 2, K, N), values(a, 2, K, N), values(b, n, N)
    tiny = 2.0 ** -126                                                 # results below the normal range carry fewer bits
    for name, got, (exact, mag, *terms), m in (('y', ops().grouped_matmul(x, W, start), R.product(x, W, start), K),
                                               ('dx', ops().grouped_matmul(dy, V, start, True), R.product(dy, V, start, True), N),
                                               ('dW', ops().grouped_matmul_wgrad(x, dy, start), R.wgrad(x, dy, start), 0),
                                               ('dW of exchanged operands', ops().grouped_matmul_wgrad(dy, x, start), R.wgrad(dy, x, start), 0)):
        assert bool((exact.abs() < 3e38).all())
        R.assert_within(got, exact, R.sum_bound(exact, mag, terms[0] if terms else m, torch.float32) + tiny * R.U, name)


def test_infinities_in_many_tiles():
    """More tiles per block than it keeps apart: infinities in the first, in the last, and in few between."""
    g = gen(6)
    n, K, N = 1500007, 6, 10
    x, W = torch.randn(n, K, generator=g, device=DEV), torch.randn(2, K, N, generator=g, device=DEV)
    start = R.start_of([n // 2, n - n // 2 - 4], DEV)
    for r, v in ((0, float('inf')), (700000, float('nan')), (1300000, -float('inf')), (1400001, 3e38), (n - 5, float('inf'))):
        x[r, r % K] = v
    y = ops().grouped_matmul(x, W, start)
    exact, _ = R.product(x, W, start)
    same_kind(y, exact)
    ok = exact.float().isfinite()                                      # (3e38 times a weight may leave the range of float32)
    size = x.double().abs().nan_to_num(0, 0).sum(1, keepdim=True) * W.abs().max()
    assert bool(((y.double() - exact).abs()[ok] <= 64 * R.U * size.expand_as(exact)[ok]).all())


def test_large_finite_values_cost_little():
    """Masks of 1e30 among ordinary rows, whose products are finite, take no more time than other rows."""
    n, K, N = 100000, 128, 64
    start = R.start_of([n // 2, n // 2], DEV)
    g = gen(7)
    x, W = torch.randn(n, K, generator=g, device=DEV), torch.randn(2, K, N, generator=g, device=DEV)

    def microseconds(x):
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            y = ops().grouped_matmul(x, W, start)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        assert y.isfinite().all()
        return sorted(times[2:])[3]

    masked = x.clone()
    masked[::2] = -1e30
    assert microseconds(masked) < 2.5 * microseconds(x)
