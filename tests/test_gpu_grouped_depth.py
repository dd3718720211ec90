"""Products of 16-bit rows whose sums are long: values of one sign, so that every rounding of a sum counts the same way.

Bound.  The tensor core truncates when it adds 16 products to a sum: at most 2 u = 2^-23 of the sum each time, in practice half of
that on average.  A piece of 16,384 values takes 1,024 such additions, 2^-13 at the most; the pieces are added in 32 bits, and the
result is rounded once, by at most h = eps / 2.  So a result is within h + 2^-13 + pieces * u of the exact sum, whatever the depth."""
import pytest
import torch

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def ops():
    import qml_lightning_b200  # noqa: F401
    return torch.ops.qml_lightning_b200


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('depth,out,n', [(16384, 40, 300), (16400, 40, 300), (40000, 24, 130), (131072, 40, 300), (131079, 33, 200),
                                         (262144, 272, 700), (1 << 20, 16, 130)])
def test_long_sums_of_one_sign(depth, out, n, dtype):
    g = torch.Generator(device=DEV).manual_seed(depth)
    start = R.start_of([n // 2, 0, n - n // 2 - 2], DEV)
    x = torch.rand(n, depth, generator=g, device=DEV).to(dtype)
    for transpose in (False, True):
        W = (torch.rand((3, out, depth) if transpose else (3, depth, out), generator=g, device=DEV) / depth).mul_(512).to(dtype)
        y = ops().grouped_matmul(x, W, start, transpose)
        exact, mag = R.product(x, W, start, transpose)
        bound = exact.abs() * (R.half_step(dtype) + 2.0 ** -13 + (depth // 16384 + 2) * R.U) * 1.001
        R.assert_within(y, exact, bound, f'{transpose}')
        assert torch.equal(y, ops().grouped_matmul(x, W, start, transpose))
    from qml_lightning_b200 import cabi
    assert cabi.tc_timeouts() == 0


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('depth,sizes,offset', [(16640, [20000, 20100], 0), (20001, [1500, 1250], 0), (17000, [300, 900], 3)])
def test_long_sums_of_large_groups_and_odd_rows(depth, sizes, offset, dtype):
    """The same for pairs of blocks (many deep rows), and for rows off the 16-byte boundaries; the ends of every group are compared."""
    g = torch.Generator(device=DEV).manual_seed(depth)
    n, out = sum(sizes) + 3, 256
    start = R.start_of(sizes, DEV)
    flat = torch.empty(n * depth + 8, dtype=dtype, device=DEV)
    x = flat[offset:offset + n * depth].view(n, depth)
    for a in range(0, n, 4096):
        x[a:a + 4096] = torch.rand(min(4096, n - a), depth, generator=g, device=DEV).to(dtype)
    bounds = R.groups_of(start, n)
    rows = torch.cat([torch.cat((torch.arange(a, a + 150), torch.arange(b - 150, b))) for a, b in bounds]).to(DEV)
    few = R.start_of([300] * len(sizes), DEV)
    for transpose in (False, True):
        W = (torch.rand((len(sizes), out, depth) if transpose else (len(sizes), depth, out), generator=g, device=DEV) / depth).mul_(512).to(dtype)
        y = ops().grouped_matmul(x, W, start, transpose)
        exact, mag = R.product(x[rows], W, few, transpose)
        bound = exact.abs() * (R.half_step(dtype) + 2.0 ** -13 + (depth // 16384 + 2) * R.U) * 1.001
        R.assert_within(y[rows], exact, bound, f'{transpose}')
        assert (y[-3:] == 0).all()
    from qml_lightning_b200 import cabi
    assert cabi.tc_timeouts() == 0
