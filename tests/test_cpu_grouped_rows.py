"""Refusals of the grouped-row operators that need no GPU, and the oracle they are tested against."""
import ctypes

import pytest
import torch

from tests import grouped_rows as R


def lib():
    from qml_lightning_b200 import _lib
    return _lib.load()


DUMMY = ctypes.c_void_p(256)      # never dereferenced: every call below is refused before anything is launched


def refused(rc, word):
    assert rc == 1, rc
    assert word in lib().qmlb_last_error(), lib().qmlb_last_error()


def test_c_entries_refuse_bad_arguments():
    L = lib()
    refused(L.qmlb_group_by_key(None, 32, 5, 3, DUMMY, DUMMY, DUMMY, 1 << 20, None), b'null')
    refused(L.qmlb_group_by_key(DUMMY, 16, 5, 3, DUMMY, DUMMY, DUMMY, 1 << 20, None), b'32 or 64')
    refused(L.qmlb_group_by_key(DUMMY, 32, 1 << 31, 3, DUMMY, DUMMY, DUMMY, 1 << 20, None), b'2^31')
    refused(L.qmlb_group_by_key(DUMMY, 32, 5, 0, DUMMY, DUMMY, DUMMY, 1 << 20, None), b'number of keys')
    refused(L.qmlb_group_by_key(DUMMY, 32, 200000, 3, DUMMY, DUMMY, DUMMY, 16, None), b'scratch')
    refused(L.qmlb_group_by_key(DUMMY, 32, 1000, 3000, DUMMY, DUMMY, None, 0, None), b'scratch')
    refused(L.qmlb_embedding(None, 32, DUMMY, 0, 5, 3, 4, 1.0, DUMMY, None), b'null')
    refused(L.qmlb_embedding(DUMMY, 32, None, 0, 5, 3, 4, 1.0, DUMMY, None), b'null')
    refused(L.qmlb_embedding(DUMMY, 8, DUMMY, 0, 5, 3, 4, 1.0, DUMMY, None), b'32 or 64')
    refused(L.qmlb_embedding(DUMMY, 32, DUMMY, 3, 5, 3, 4, 1.0, DUMMY, None), b'element type')
    refused(L.qmlb_embedding(DUMMY, 32, DUMMY, 0, 5, 3, 0, 1.0, DUMMY, None), b'sizes')
    refused(L.qmlb_embedding_grad(None, 0, DUMMY, 32, DUMMY, DUMMY, 5, 3, 4, 1.0, DUMMY, DUMMY, 1 << 20, None), b'null')
    refused(L.qmlb_embedding_grad(DUMMY, 7, DUMMY, 32, DUMMY, DUMMY, 5, 3, 4, 1.0, DUMMY, DUMMY, 1 << 20, None), b'element type')
    refused(L.qmlb_embedding_grad(DUMMY, 0, DUMMY, 32, DUMMY, DUMMY, 5, 0, 4, 1.0, DUMMY, DUMMY, 1 << 20, None), b'sizes')
    refused(L.qmlb_embedding_grad(DUMMY, 0, DUMMY, 32, DUMMY, DUMMY, 5, 3, 4, 1.0, DUMMY, DUMMY, 8, None), b'scratch')
    refused(L.qmlb_grouped_matmul(None, DUMMY, DUMMY, 0, 5, 2, 4, 4, 0, DUMMY, DUMMY, 1 << 20, None), b'null')
    refused(L.qmlb_grouped_matmul(DUMMY, DUMMY, DUMMY, 5, 5, 2, 4, 4, 0, DUMMY, DUMMY, 1 << 20, None), b'element type')
    refused(L.qmlb_grouped_matmul(DUMMY, DUMMY, DUMMY, 0, 5, 0, 4, 4, 0, DUMMY, DUMMY, 1 << 20, None), b'groups')
    refused(L.qmlb_grouped_matmul(DUMMY, DUMMY, DUMMY, 0, 5, 1025, 4, 4, 0, DUMMY, DUMMY, 1 << 20, None), b'groups')
    refused(L.qmlb_grouped_matmul(DUMMY, DUMMY, DUMMY, 0, 5, 2, 0, 4, 0, DUMMY, DUMMY, 1 << 20, None), b'sizes')
    refused(L.qmlb_grouped_matmul(DUMMY, DUMMY, DUMMY, 0, 1 << 31, 2, 4, 4, 0, DUMMY, DUMMY, 1 << 20, None), b'rows')
    refused(L.qmlb_grouped_matmul_wgrad(DUMMY, None, DUMMY, 0, 5, 2, 4, 4, DUMMY, DUMMY, 1 << 20, None), b'null')
    refused(L.qmlb_grouped_matmul_wgrad(DUMMY, DUMMY, DUMMY, 9, 5, 2, 4, 4, DUMMY, DUMMY, 1 << 20, None), b'element type')
    refused(L.qmlb_grouped_matmul_wgrad(DUMMY, DUMMY, DUMMY, 0, 5, 2000, 4, 4, DUMMY, DUMMY, 1 << 20, None), b'groups')
    refused(L.qmlb_grouped_matmul_wgrad(DUMMY, DUMMY, DUMMY, 0, 5, 2, 4, -1, DUMMY, DUMMY, 1 << 20, None), b'sizes')


def test_scratch_sizes_grow_with_the_work():
    L = lib()
    assert L.qmlb_group_by_key_scratch_bytes(0, 5) == 0 and L.qmlb_group_by_key_scratch_bytes(1000, 5) == 0      # one launch, no scratch
    assert L.qmlb_grouped_matmul_workspace_bytes(21, 3, 336, 256, 0, 0) == 0 and L.qmlb_grouped_matmul_workspace_bytes(210000, 3, 336, 256, 0, 0) > 0
    assert L.qmlb_group_by_key_scratch_bytes(1 << 20, 5) < 8 << 20                 # one pass: counters only
    assert L.qmlb_group_by_key_scratch_bytes(1 << 20, 50000) >= 3 * 4 << 20        # two passes: pairs and sorted keys
    assert L.qmlb_embedding_grad_scratch_bytes(1 << 20, 100, 256) >= 2 * 256 * 4


def test_wrappers_refuse_cpu_tensors_and_wrong_types():
    from qml_lightning_b200 import cabi
    i, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 8)
    for call in (lambda: cabi.group_by_key(i, 3), lambda: cabi.embedding(i, f), lambda: cabi.embedding_grad(f, i, i, i),
                 lambda: cabi.grouped_matmul(f, f.view(2, 2, 8).transpose(1, 2).contiguous()[:, :8], torch.zeros(3, dtype=torch.int32)),
                 lambda: cabi.grouped_matmul_wgrad(f, f, i)):
        with pytest.raises(RuntimeError, match='CUDA'):
            call()
    with pytest.raises(RuntimeError, match='int32 or int64'):
        cabi.group_by_key(f, 3)
    with pytest.raises(RuntimeError, match='nkeys'):
        cabi.group_by_key(i, 0)
    with pytest.raises(RuntimeError, match='float32, float16 or bfloat16'):
        cabi.embedding(i, f.double())
    with pytest.raises(RuntimeError, match='columns'):
        cabi.grouped_matmul(f, torch.zeros(2, 5, 8), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match='one entry per group'):
        cabi.grouped_matmul(f, torch.zeros(2, 8, 8), i)
    ops = torch.ops.qml_lightning_b200
    for call in (lambda: ops.group_by_key(i, 3), lambda: ops.embedding(i, f, 1.0), lambda: ops.embedding_grad(f, i, i, i, 3, 1.0),
                 lambda: ops.grouped_matmul(f, torch.zeros(1, 8, 8), i), lambda: ops.grouped_matmul_wgrad(f, f, i)):
        with pytest.raises(RuntimeError, match='CUDA'):
            call()


def test_operator_schemas():
    import qml_lightning_b200  # noqa: F401
    get = torch._C._jit_get_schemas_for_operator
    names = {n: [a.name for a in get('qml_lightning_b200::' + n)[0].arguments]
             for n in ('group_by_key', 'embedding', 'embedding_grad', 'grouped_matmul', 'grouped_matmul_wgrad')}
    assert names == {'group_by_key': ['keys', 'nkeys'], 'embedding': ['indices', 'table', 'scale'],
                     'embedding_grad': ['grad', 'indices', 'order', 'group_start', 'rows', 'scale'],
                     'grouped_matmul': ['x', 'W', 'group_start', 'transpose'], 'grouped_matmul_wgrad': ['x', 'dy', 'group_start']}


def test_oracle_agrees_with_loops():
    """The 64-bit oracle of the GPU tests against loops over single rows."""
    g = torch.Generator().manual_seed(0)
    keys = torch.randint(-1, 5, (23,), generator=g)
    order, start = R.order_of(keys, 4)
    want = sorted(range(23), key=lambda i: (keys[i].item() if 0 <= keys[i] < 4 else 4, i))
    assert order.tolist() == want and start.tolist() == [sum(1 for k in keys.tolist() if 0 <= k < v) for v in range(5)]
    table, grad = torch.randn(4, 3, generator=g), torch.randn(23, 3, generator=g)
    out = R.lookup(keys, table, 2.0)
    total, mag, terms = R.lookup_grad(keys, grad, 4, 2.0)
    ref, refg = torch.zeros(23, 3, dtype=torch.float64), torch.zeros(4, 3, dtype=torch.float64)
    for i, k in enumerate(keys.tolist()):
        if 0 <= k < 4:
            ref[i] = 2 * table[k].double()
            refg[k] += 2 * grad[i].double()
    assert torch.equal(out, ref) and torch.allclose(total, refg, rtol=1e-14) and int(terms.sum()) == int(start[4])
    x, W, dy = torch.randn(23, 3, generator=g), torch.randn(4, 3, 2, generator=g), torch.randn(23, 2, generator=g)
    y, dW = torch.zeros(23, 2, dtype=torch.float64), torch.zeros(4, 3, 2, dtype=torch.float64)
    for e in range(4):
        for r in range(int(start[e]), int(start[e + 1])):
            y[r] = x[r].double() @ W[e].double()
            dW[e] += torch.outer(x[r].double(), dy[r].double())
    assert torch.allclose(R.product(x, W, start)[0], y, rtol=1e-14) and torch.allclose(R.wgrad(x, dy, start)[0], dW, rtol=1e-13, atol=1e-15)
