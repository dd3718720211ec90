"""Group bounds in 64 bits: values beyond 32 bits are clamped like all others outside the rows."""
import pytest
import torch

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


@pytest.mark.parametrize('dtype', R.TYPES)
def test_wide_bounds_are_clamped(dtype):
    import qml_lightning_b200  # noqa: F401
    ops = torch.ops.qml_lightning_b200
    g = torch.Generator(device=DEV).manual_seed(1)
    x, W, dy = (torch.randn(s, generator=g, device=DEV).to(dtype) for s in ((40, 24), (3, 24, 16), (40, 16)))
    want = torch.tensor([0, 10, 40, 40], dtype=torch.int32, device=DEV)
    for bounds in ([0, 10, 2 ** 32 + 5, 2 ** 40], [-2 ** 32 + 3, 10, 2 ** 31, 2 ** 62], [-2 ** 63, 10, 40, 2 ** 63 - 1]):
        start = torch.tensor(bounds, device=DEV)
        for got, ref in ((ops.grouped_matmul(x, W, start), ops.grouped_matmul(x, W, want)),
                         (ops.grouped_matmul(dy, W, start, True), ops.grouped_matmul(dy, W, want, True)),
                         (ops.grouped_matmul_wgrad(x, dy, start), ops.grouped_matmul_wgrad(x, dy, want))):
            assert torch.equal(got, ref), bounds
