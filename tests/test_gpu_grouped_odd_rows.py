"""Products of 16-bit rows that begin off the 16-byte boundaries: every small depth at every offset, with NaN all around the rows (what
belongs to a neighbour must not take part), and small groups of odd depth."""
import pytest
import torch

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def ops():
    import qml_lightning_b200  # noqa: F401
    return torch.ops.qml_lightning_b200


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('K', [1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 20])
def test_every_offset_of_shallow_rows(K, dtype):
    g = torch.Generator(device=DEV).manual_seed(K)
    for n, sizes in ((1, [1]), (9, [4, 5]), (200, [3, 0, 150, 47]), (2600, [1300, 1280])):
        N = 40
        W = torch.randn(len(sizes), K, N, generator=g, device=DEV).to(dtype)
        rows = torch.randn(n, K, generator=g, device=DEV).to(dtype)
        start = R.start_of(sizes, DEV)
        used = sum(sizes)
        rows[used:] = float('nan')
        exact, mag = R.product(rows[:used], W, start)
        for offset in range(9):
            flat = torch.full((n * K + 32,), float('nan'), dtype=dtype, device=DEV)
            x = flat[offset:offset + n * K].view(n, K)
            x.copy_(rows)
            y = ops().grouped_matmul(x, W, start)
            R.assert_within(y[:used], exact, R.sum_bound(exact, mag, K, dtype), f'{n} {offset}')
            assert (y[used:] == 0).all()
