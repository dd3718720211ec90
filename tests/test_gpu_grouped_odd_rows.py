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


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('K', [33, 130, 780, 781, 782])
@pytest.mark.parametrize('rows', [1, 20, 127, 130, 257, 513])
def test_small_groups_of_odd_depth(rows, K, dtype):
    """Groups around the sizes at which rows are copied to the 16-byte boundaries, with canaries behind the workspace."""
    from qml_lightning_b200 import _lib, cabi
    g = torch.Generator(device=DEV).manual_seed(rows + K)
    G, N = 9, 72
    sizes = [rows] * (G - 2) + [0, 2 * rows]
    n = sum(sizes) + 5
    x, W = torch.randn(n, K, generator=g, device=DEV).to(dtype), (torch.randn(G, K, N, generator=g, device=DEV) / K ** 0.5).to(dtype)
    x[-5:] = float('nan')
    start = R.start_of(sizes, DEV)
    lib, code, guard = _lib.load(), cabi._DTYPES[dtype], 4096
    nbytes = lib.qmlb_grouped_matmul_workspace_bytes(n, G, K, N, code, 0)
    ws = torch.full((nbytes + guard,), 85, dtype=torch.uint8, device=DEV)
    y = torch.full((n, N), 7.0, dtype=dtype, device=DEV)
    assert lib.qmlb_grouped_matmul(x.data_ptr(), W.data_ptr(), start.data_ptr(), code, n, G, K, N, 0, y.data_ptr(), ws.data_ptr(), nbytes,
                                   torch.cuda.current_stream().cuda_stream) == 0
    exact, mag = R.product(x[:-5], W, start)
    R.assert_within(y[:-5], exact, R.sum_bound(exact, mag, K, dtype), 'y')
    assert (y[-5:] == 0).all() and (ws[nbytes:] == 85).all()


@pytest.mark.parametrize('K', [781, 782])
def test_small_groups_of_odd_depth_cost_little(K):
    """64 groups of 20 rows: not much longer than at a depth that is a multiple of 8."""
    G = 64
    start = R.start_of([20] * G, DEV)

    def microseconds(K):
        x, W = torch.ones(20 * G, K, dtype=torch.bfloat16, device=DEV), torch.ones(G, K, 256, dtype=torch.bfloat16, device=DEV)
        times = []
        for i in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                ops().grouped_matmul(x, W, start)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 100)
        return sorted(times[2:])[3]

    assert microseconds(K) < 2.5 * microseconds(784)
