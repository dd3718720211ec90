"""Grouped products of float32 rows whose values lie many powers of ten apart along the depth of a sum.

Bounds.  u = 2^-24.  An operand enters as three bf16 numbers whose sum it is (8 + 8 + 8 bits, each rounded to nearest, so that the
second is at most 2^-9 and the third at most 2^-18 of it), and the six largest of the nine products are formed: what is left out is
at most (2 * 2^-27 + 2^-36) of a product, less than u / 2.  Sums of m terms whose additions may truncate are off by at most 2 m u
of the sum of the terms' magnitudes, so ``grouped_rows.sum_bound``, which grants 14 u for the operands, holds with room.  All
bounds are relative to the magnitudes of the very terms of a sum, whatever stands elsewhere in its rows.
"""
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


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


# few rows, and more rows than the kernel for few rows takes
@pytest.mark.parametrize('n', [200, 3000])
@pytest.mark.parametrize('ratio', [1e6, 1e8, 1e12, 1e18])
def test_features_of_different_magnitude(n, ratio):
    """Features that are `ratio` times larger than the others, with weights as much smaller: every product is of one size."""
    g = gen(1)
    K, N = 64, 96
    large = torch.zeros(K, dtype=torch.bool, device=DEV)
    large[[5, 40]] = True
    scale = torch.where(large, ratio, 1.0)
    x, W = randn(g, n, K) * scale, randn(g, 2, K, N) / scale.view(1, K, 1)
    start = R.start_of([n // 3, n - n // 3 - 5], DEV)
    y = ops().grouped_matmul(x, W, start)
    exact, mag = R.product(x, W, start)
    R.assert_within(y, exact, R.sum_bound(exact, mag, K, torch.float32), 'y')
    Wt, dy = (randn(g, 2, N, K) / scale), randn(g, n, K) * scale        # the sums of the transposed product run along the last dimension
    dx = ops().grouped_matmul(dy, Wt, start, True)
    exact, mag = R.product(dy, Wt, start, True)
    R.assert_within(dx, exact, R.sum_bound(exact, mag, K, torch.float32), 'dx')


@pytest.mark.parametrize('n', [200, 3000])
@pytest.mark.parametrize('ratio', [1e6, 1e8, 1e15])
def test_large_entries_that_meet_zeros(n, ratio):
    """One entry of a row, or of a matrix, is `ratio` times larger than the others and is multiplied by zero."""
    g = gen(2)
    K, N = 200, 40
    start = R.start_of([n - 9], DEV)
    for which in ('row', 'matrix', 'same stretch'):
        x, W = randn(g, n, K), randn(g, 1, K, N)
        k = 3 if which != 'same stretch' else 150
        if which == 'matrix':
            W[0, k] *= ratio
            x[:, k] = 0
        else:
            x[:, k] *= ratio
            W[0, k] = 0
        y = ops().grouped_matmul(x, W, start)
        exact, mag = R.product(x, W, start)
        R.assert_within(y, exact, R.sum_bound(exact, mag, K, torch.float32), which)
        assert R.relative(y, exact) < (K ** 0.5 + 16) * R.U


@pytest.mark.parametrize('ratio', [1e6, 1e8, 1e15])
@pytest.mark.parametrize('n,where', [(100, 0), (512, 0), (512, 448), (20000, 0), (20000, 10000)])
def test_gradient_with_large_rows_that_meet_zeros(n, where, ratio):
    """Sparse descriptors: some rows of dy are far larger than the others, and x is zero there."""
    g = gen(3)
    K, N = 48, 72
    x, dy = randn(g, n, K), randn(g, n, N)
    dy[where:where + 64] *= ratio
    x[where:where + 64, ::2] = 0
    start = R.start_of([n], DEV)
    for a, b, cols in ((x, dy, (slice(None, None, 2), slice(None))), (dy, x, (slice(None), slice(None, None, 2)))):
        dW = ops().grouped_matmul_wgrad(a, b, start)
        exact, mag, terms = R.wgrad(a, b, start)
        R.assert_within(dW, exact, R.sum_bound(exact, mag, terms, torch.float32), 'dW')
        part = (0,) + cols                                             # the results that no large row takes part in
        assert R.relative(dW[part], exact[part]) < (n ** 0.5 + 16) * R.U
