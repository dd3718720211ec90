"""Failure detection of the grouped products without a fault: a bounded wait that runs out.

A second copy of the library grants the first wait for operands of the issuing warps no polls at all (compile-time macro
``QMLB_TEST_FIRST_WAIT_POLLS`` = 0; every other wait keeps its limit).  That wait gives up before anything was issued to the
tensor cores; the other warps of the block see its flag and stop waiting, the block drains its copies, marks its results with
NaN, frees its tensor memory and counts the event.  The production library works on the same context right afterwards."""
import ctypes
import glob
import os
import subprocess

import pytest
import torch

from qml_lightning_b200 import _lib
from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, 'qml_lightning_b200')
FILES = ('grouped_tc', 'grouped_wgrad_tc', 'grouped_pair_tc')


@pytest.fixture(scope='module')
def impatient(tmp_path_factory):
    tmp = str(tmp_path_factory.mktemp('firstwait'))
    nvcc = '/usr/local/cuda/bin/nvcc' if os.path.exists('/usr/local/cuda/bin/nvcc') else 'nvcc'
    arch = ['-gencode', 'arch=compute_100a,code=sm_100a']
    objs = []
    jobs = []
    for f in FILES:
        objs.append(os.path.join(tmp, f + '.o'))
        jobs.append(subprocess.Popen([nvcc] + arch + ['-O3', '-std=c++17', '--expt-relaxed-constexpr', '-Xcompiler', '-fPIC', '-I', os.path.join(ROOT, 'include'),
                                                      '-I', os.path.join(PKG, 'csrc'), '-DQMLB_TEST_FIRST_WAIT_POLLS=0', '-c',
                                                      os.path.join(PKG, 'csrc', f + '.cu'), '-o', objs[-1]]))
    assert all(j.wait() == 0 for j in jobs)
    others = [o for o in sorted(glob.glob(os.path.join(PKG, 'build', '*.o'))) if os.path.basename(o)[:-2] not in FILES]
    assert others, 'the product library has to be built first (python qml_lightning_b200/build.py)'
    so = os.path.join(tmp, 'libqmlb200_firstwait.so')
    subprocess.run([nvcc, '-shared'] + arch + ['-o', so] + objs + others + ['-lcudart', '-lcublas'], check=True)
    lib = ctypes.CDLL(so)
    for name in ('qmlb_grouped_matmul', 'qmlb_grouped_matmul_wgrad', 'qmlb_tc_timeouts', 'qmlb_last_error'):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _lib.SIGNATURES[name]
    return lib


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_first_wait_runs_out_and_the_context_survives(impatient, dtype):
    product = _lib.load()
    g = torch.Generator(device=DEV).manual_seed(1)
    n, K, N = 4000, 128, 64
    x, dy = (torch.randn(n, c, generator=g, device=DEV).to(dtype) for c in (K, N))
    W = torch.randn(1, K, N, generator=g, device=DEV).to(dtype)
    start = R.start_of([n], DEV)
    code = {torch.float32: 0, torch.bfloat16: 2}[dtype]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def calls(lib):
        y, dW = torch.full((n, N), 7.0, device=DEV, dtype=dtype), torch.full((1, K, N), 7.0, device=DEV, dtype=dtype)
        nb = product.qmlb_grouped_matmul_workspace_bytes(n, 1, K, N, code, 0)
        wb = product.qmlb_grouped_matmul_wgrad_workspace_bytes(n, 1, K, N, code)
        ws = torch.empty(max(nb, wb), dtype=torch.uint8, device=DEV)
        assert lib.qmlb_grouped_matmul(x.data_ptr(), W.data_ptr(), start.data_ptr(), code, n, 1, K, N, 0, y.data_ptr(), ws.data_ptr(), nb, stream) == 0
        torch.cuda.synchronize()
        assert lib.qmlb_grouped_matmul_wgrad(x.data_ptr(), dy.data_ptr(), start.data_ptr(), code, n, 1, K, N, dW.data_ptr(), ws.data_ptr(), wb, stream) == 0
        torch.cuda.synchronize()
        return y, dW

    before = impatient.qmlb_tc_timeouts()
    y, dW = calls(impatient)                                   # returns: the waits are bounded
    assert impatient.qmlb_tc_timeouts() > before               # the events were counted
    assert bool(torch.isnan(y).all()) and bool(torch.isnan(dW).all())
    before = product.qmlb_tc_timeouts()
    y, dW = calls(product)                                     # same context, production limits
    assert product.qmlb_tc_timeouts() == before
    e, m = R.product(x, W, start)
    R.assert_within(y, e, R.sum_bound(e, m, K, dtype), 'y')
    e, m, t = R.wgrad(x, dy, start)
    R.assert_within(dW, e, R.sum_bound(e, m, t, dtype), 'dW')
