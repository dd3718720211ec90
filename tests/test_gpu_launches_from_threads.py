"""Calls from several host threads at once whose launches of one kernel want different amounts of shared memory: every call succeeds
and gives what it gives alone."""
import threading

import pytest
import torch

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def calls(kind):
    import qml_lightning_b200  # noqa: F401
    ops = torch.ops.qml_lightning_b200
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s, dtype=torch.float32: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    if kind == 'order':
        for n, k in ((1500, 5), (40000, 300), (66000, 511), (9000, 4000)):
            keys = torch.randint(0, k, (n,), generator=g, device=DEV)
            yield lambda keys=keys, k=k: ops.group_by_key(keys, k)[0]
        return
    if kind == 'table gradient':
        for n, k, width in ((3000, 5, 3), (20000, 300, 256), (6000, 40, 1030)):
            keys, grad = torch.randint(0, k, (n,), generator=g, device=DEV), r(n, width)
            order, start = ops.group_by_key(keys, k)
            yield lambda a=(grad, keys, order, start, k): ops.embedding_grad(*a)
        return
    dtype = torch.float32 if kind.startswith('float32') else torch.bfloat16
    for groups, K, N in ((1, 64, 16), (900, 64, 128), (40, 128, 256)):
        n = 3000
        x, W, dy, start = r(n, K, dtype=dtype), r(groups, K, N, dtype=dtype), r(n, N, dtype=dtype), R.start_of([n // groups] * groups, DEV)
        if kind.endswith('gradient'):
            yield lambda a=(x, dy, start): ops.grouped_matmul_wgrad(*a)
        else:
            yield lambda a=(x, W, start): ops.grouped_matmul(*a)


@pytest.mark.parametrize('kind', ['order', 'table gradient', 'float32', 'float32 gradient', '16 bits', '16 bits gradient'])
def test_threads_with_different_sizes(kind):
    jobs = list(calls(kind))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    errors, begin = [], threading.Barrier(len(jobs))

    def work(job, expected):
        try:
            begin.wait(timeout=60)
            with torch.cuda.stream(torch.cuda.Stream(DEV)):
                for i in range(400):
                    got = job()
                    if i % 50 == 0:
                        assert torch.equal(got, expected)
                assert torch.equal(got, expected)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[:3]
