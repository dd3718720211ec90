"""Orders in which most keys do not occur: the starts of a long run of absent keys are as right, and not much slower, than others."""
import pytest
import torch

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def order(keys, nkeys):
    import qml_lightning_b200  # noqa: F401
    return torch.ops.qml_lightning_b200.group_by_key(keys, nkeys)


def inputs(n, nkeys, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    spread = torch.randint(0, nkeys, (n,), generator=g, device=DEV)
    yield 'spread', spread
    yield 'all the first', torch.zeros_like(spread)
    yield 'all the last', torch.full_like(spread, nkeys - 1)
    yield 'all outside', torch.full_like(spread, -1)
    yield 'small', torch.randint(0, 5, (n,), generator=g, device=DEV)
    yield 'both ends', torch.where(spread % 2 == 0, spread % 7, nkeys - 1 - spread % 3)
    yield 'long gaps', spread // 4099 * 4099
    yield 'gaps of a thousand', (spread // 1000) * 1000 + 999


@pytest.mark.parametrize('n,nkeys', [(1, 600), (31, 1000), (4000, 64000), (8192, 131072), (20000, 20000), (70000, 1000000), (131072, 2000000),
                                     (131073, 2000000), (300001, 40000), (300001, 4000000)])
def test_starts_of_absent_keys(n, nkeys):
    for what, keys in inputs(n, nkeys):
        got, start = order(keys.clamp(max=nkeys - 1), nkeys)
        want, wstart = R.order_of(keys.clamp(max=nkeys - 1), nkeys)
        assert torch.equal(got, want) and torch.equal(start, wstart), what


@pytest.mark.parametrize('n,nkeys', [(65536, 1000000), (131072, 2000000), (500000, 8000000)])
def test_absent_keys_cost_little(n, nkeys):
    """Ten times the time of spread keys allows for the one block whose keys are all equal, not for a walk over the absent ones."""
    def microseconds(keys):
        for _ in range(3):
            order(keys, nkeys)
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            order(keys, nkeys)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        return sorted(times)[2]

    cases = dict(inputs(n, nkeys))
    base = microseconds(cases.pop('spread'))
    for what, keys in cases.items():
        assert microseconds(keys) < 10 * base, (what, base)
