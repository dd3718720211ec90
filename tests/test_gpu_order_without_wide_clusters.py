"""Orders on a device that runs no clusters of sixteen blocks: a second copy of the library is told so (compile-time macro
``QMLB_TEST_NO_WIDE_CLUSTERS``) and takes smaller clusters, or separate launches, with the scratch that the library asks for."""
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


@pytest.fixture(scope='module')
def narrow(tmp_path_factory):
    tmp = str(tmp_path_factory.mktemp('narrow'))
    nvcc = '/usr/local/cuda/bin/nvcc' if os.path.exists('/usr/local/cuda/bin/nvcc') else 'nvcc'
    arch = ['-gencode', 'arch=compute_100a,code=sm_100a']
    obj, so = os.path.join(tmp, 'key_order.o'), os.path.join(tmp, 'libqmlb200_narrow.so')
    subprocess.run([nvcc] + arch + ['-O3', '-std=c++17', '--expt-relaxed-constexpr', '-Xcompiler', '-fPIC', '-I', os.path.join(ROOT, 'include'),
                                    '-I', os.path.join(PKG, 'csrc'), '-DQMLB_TEST_NO_WIDE_CLUSTERS', '-c', os.path.join(PKG, 'csrc', 'key_order.cu'),
                                    '-o', obj], check=True)
    others = [o for o in sorted(glob.glob(os.path.join(PKG, 'build', '*.o'))) if os.path.basename(o) != 'key_order.o']
    assert others, 'the product library has to be built first (python qml_lightning_b200/build.py)'
    subprocess.run([nvcc, '-shared'] + arch + ['-o', so, obj] + others + ['-lcudart', '-lcublas'], check=True)
    lib = ctypes.CDLL(so)
    for name in ('qmlb_group_by_key', 'qmlb_group_by_key_scratch_bytes', 'qmlb_last_error'):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _lib.SIGNATURES[name]
    return lib


@pytest.mark.parametrize('n', [100, 16385, 20000, 65536, 65537, 100003, 131072, 131073])
@pytest.mark.parametrize('nkeys', [1, 5, 511, 512, 1023, 1024, 50021, 1000000])
def test_order_without_wide_clusters(narrow, n, nkeys):
    g = torch.Generator(device=DEV).manual_seed(n + nkeys)
    product = _lib.load()
    nbytes = product.qmlb_group_by_key_scratch_bytes(n, nkeys)
    assert nbytes == narrow.qmlb_group_by_key_scratch_bytes(n, nkeys)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    guard = 4096
    for dtype in (torch.int32, torch.int64):
        keys = torch.randint(-1, nkeys + 1, (n,), generator=g, device=DEV).to(dtype)
        want, wstart = R.order_of(keys, nkeys)
        for lib in (narrow, product):
            order, start = torch.empty(n, dtype=torch.int32, device=DEV), torch.empty(nkeys + 1, dtype=torch.int32, device=DEV)
            scratch = torch.full((nbytes + guard,), 85, dtype=torch.uint8, device=DEV)
            rc = lib.qmlb_group_by_key(keys.data_ptr(), 32 if dtype == torch.int32 else 64, n, nkeys, order.data_ptr(), start.data_ptr(),
                                       scratch.data_ptr(), nbytes, stream)
            assert rc == 0, lib.qmlb_last_error()
            assert torch.equal(order, want) and torch.equal(start, wstart) and (scratch[nbytes:] == 85).all()
