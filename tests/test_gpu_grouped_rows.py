"""Operators on rows that belong to groups (order by key, table lookup and its gradient, one matrix per group) against
64-bit oracles, at the sizes, types, alignments and group shapes where they can go wrong.  The bounds are derived in
tests/grouped_rows.py."""
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


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def misaligned(t):
    """The same values at an address that is a multiple of the element size only."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    out = flat[1:].view(t.shape)
    assert out.is_contiguous() and (t.numel() == 0 or out.data_ptr() % 16 != 0)
    return out


# ---- order by key ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('nkeys', [1, 2, 3, 5, 31, 255, 300, 511, 1023, 1024, 50021, 1048575, 2100000])
@pytest.mark.parametrize('n', [1, 2, 31, 33, 257, 1024, 1025, 4095, 4097, 8193, 70001])
def test_order_is_stable(n, nkeys):
    g = gen(n * 7 + nkeys)
    for dtype in (torch.int32, torch.int64):
        keys = torch.randint(-1 if n % 2 else 0, nkeys + 1, (n,), generator=g, device=DEV).to(dtype)
        order, start = ops().group_by_key(keys, nkeys)
        want, wstart = R.order_of(keys, nkeys)
        assert order.dtype == torch.int32 and torch.equal(order, want)
        assert start.dtype == torch.int32 and torch.equal(start, wstart)


@pytest.mark.parametrize('n', [20000, 33000, 131072, 131073, 300000, 1234567])
@pytest.mark.parametrize('nkeys', [1, 2, 3, 5, 7, 8, 15, 16, 1000, 30011])
def test_order_of_many_skewed_keys(n, nkeys):
    g = gen(n + nkeys)
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    keys = (nkeys ** u - 1).int().clamp(max=nkeys - 1)              # small keys are frequent
    keys[torch.rand(n, generator=g, device=DEV) < 0.1] = -1
    order, start = ops().group_by_key(keys, nkeys)
    want, wstart = R.order_of(keys, nkeys)
    assert torch.equal(order, want) and torch.equal(start, wstart)


def test_order_of_special_inputs():
    from qml_lightning_b200 import cabi
    order, start = ops().group_by_key(torch.empty(0, dtype=torch.int32, device=DEV), 7)
    assert order.numel() == 0 and start.tolist() == [0] * 8
    big = torch.tensor([2 ** 62, -2 ** 63, 3, 2 ** 31 + 2, -1, 2 ** 32 + 1, 1, 4], device=DEV)     # only 3 and 1 are keys
    order, start = cabi.group_by_key(big, 4)
    assert order.tolist() == [6, 2, 0, 1, 3, 4, 5, 7] and start.tolist() == [0, 0, 1, 1, 2]
    low = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0], dtype=torch.int32, device=DEV)
    assert ops().group_by_key(low, 1)[0].tolist() == [2, 0, 1]
    for value in (-1, 0, 4):                                                                       # one value everywhere
        keys = torch.full((50000,), value, dtype=torch.int64, device=DEV)
        order, start = ops().group_by_key(keys, 5)
        assert torch.equal(order, torch.arange(50000, dtype=torch.int32, device=DEV))
        assert start.tolist() == [0 if value < 0 or v <= value else 50000 for v in range(6)]
    wide = torch.randint(0, 9, (64, 40), generator=gen(3), device=DEV, dtype=torch.int32)           # any shape counts flat
    assert torch.equal(ops().group_by_key(wide.t(), 9)[0], R.order_of(wide.t().contiguous(), 9)[0])
    nkeys = (1 << 30) + 5                                                                          # digits of a four-pass order
    keys = torch.randint(0, nkeys, (1000,), generator=gen(4), device=DEV)
    keys[:10] = keys[10:20]
    order, start = ops().group_by_key(keys, nkeys)
    assert torch.equal(order, torch.sort(keys, stable=True)[1].int())
    probe = torch.cat((keys, keys + 1, torch.tensor([0, nkeys], device=DEV)))
    assert torch.equal(start[probe].long(), torch.searchsorted(torch.sort(keys)[0], probe))


# ---- table lookup -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('width', [1, 2, 3, 8, 12, 64, 100, 127, 256, 1000, 2050])
def test_lookup_and_its_gradient(width, dtype):
    g = gen(width)
    for n, rows, outside in ((1, 1, 0), (7, 3, 0), (255, 120, 1), (1000, 3, 1), (5000, 1, 0), (3001, 7000, 1)):
        idx = torch.randint(-outside, rows + outside, (n,), generator=g, device=DEV)
        idx = idx.int() if n % 2 else idx
        table, grad = randn(g, rows, width, dtype=dtype), randn(g, n, width, dtype=dtype)
        if width == 64:
            table, grad = misaligned(table), misaligned(grad)
        scale = 1.7
        out = ops().embedding(idx, table, scale)
        exact = R.lookup(idx, table, scale)
        R.assert_within(out, exact, R.lookup_bound(exact, dtype), f'lookup {n} {rows}')
        order, start = ops().group_by_key(idx, rows)
        got = ops().embedding_grad(grad, idx, order, start, rows, scale)
        exact, mag, terms = R.lookup_grad(idx, grad, rows, scale)
        R.assert_within(got, exact, R.sum_bound(exact, mag, terms.view(-1, 1), dtype), f'gradient {n} {rows}')
        assert torch.equal(got, ops().embedding_grad(grad, idx, order, start, rows, scale))       # reproducible to the bit


@pytest.mark.parametrize('rows,skew', [(3, 1.0), (1, 0.0), (300, 0.0), (40000, 1.0)])
@pytest.mark.parametrize('n', [16384, 100003])
def test_gradient_of_long_segments(n, rows, skew):
    """Segments that begin, end or lie across the borders of the blocks, runs and pieces of the gradient's kernel."""
    g = gen(n + rows)
    for dtype, width in ((torch.float32, 40), (torch.bfloat16, 256), (torch.float32, 2), (torch.float16, 7)):
        w = torch.arange(1, rows + 1, device=DEV, dtype=torch.float64) ** -skew
        idx = torch.searchsorted(torch.cumsum(w, 0), torch.rand(n, generator=g, device=DEV, dtype=torch.float64) * w.sum()).clamp(max=rows - 1)
        grad = randn(g, n, width, dtype=dtype)
        order, start = ops().group_by_key(idx, rows)
        got = ops().embedding_grad(grad, idx, order, start, rows, 1.0)
        exact, mag, terms = R.lookup_grad(idx, grad, rows, 1.0)
        R.assert_within(got, exact, R.sum_bound(exact, mag, terms.view(-1, 1), dtype), f'{dtype} {width}')
        if dtype == torch.float32:        # far inside the worst case: the sums are split
            assert R.relative(got, exact) < 1e-6


def test_gradient_with_segments_of_chosen_lengths():
    g = gen(11)
    for lengths in ([128, 128, 128], [127, 1, 0, 0, 129, 255, 1, 1], [4096, 0, 4096, 1], [1, 8191, 1], [0, 0, 5000, 0], [31, 33, 64] * 40):
        idx = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), torch.tensor(lengths, device=DEV))
        idx = idx[torch.randperm(idx.numel(), generator=g, device=DEV)]
        for width, dtype in ((256, torch.float32), (4, torch.float32), (1024, torch.bfloat16)):
            grad = randn(g, idx.numel(), width, dtype=dtype)
            order, start = ops().group_by_key(idx, len(lengths))
            got = ops().embedding_grad(grad, idx, order, start, len(lengths), 0.5)
            exact, mag, terms = R.lookup_grad(idx, grad, len(lengths), 0.5)
            R.assert_within(got, exact, R.sum_bound(exact, mag, terms.view(-1, 1), dtype), str(lengths[:8]))


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('width', [4, 5, 7, 8, 9, 10, 15, 17, 18, 33, 301])
@pytest.mark.parametrize('n', [1, 2, 3, 29, 1000, 20001])
def test_lookup_of_odd_widths(n, width, dtype):
    """Rows that end anywhere in a 16-byte piece of the result: every element is its own, nothing behind the result is written,
    and rows that nothing names may hold anything."""
    from qml_lightning_b200 import cabi
    g = gen(n + width)
    rows = 37
    table = randn(g, rows, width, dtype=dtype)
    table[0] = float('nan')                                            # read for an index outside, and not used
    for bits in (torch.int32, torch.int64):
        idx = torch.randint(-1, rows + 2, (n,), generator=g, device=DEV, dtype=bits)
        idx[idx == 0] = -5
        flat = torch.full((n * width + 64,), 9.0, dtype=dtype, device=DEV)
        exact = R.lookup(idx, table, 1.5)
        out = cabi.embedding(idx, table, 1.5, out=flat[:n * width].view(n, width))
        R.assert_within(out, exact, R.lookup_bound(exact, dtype), f'{n} {width}')
        assert (flat[n * width:] == 9).all()
        shifted = flat[3:3 + n * width].view(n, width)                 # a result off the 16-byte boundary
        R.assert_within(cabi.embedding(idx, table, 1.5, out=shifted), exact, R.lookup_bound(exact, dtype), f'{n} {width} shifted')


def test_lookup_special_inputs():
    from qml_lightning_b200 import cabi
    table = randn(gen(0), 5, 6)
    assert ops().embedding(torch.empty(0, dtype=torch.int64, device=DEV), table, 1.0).shape == (0, 6)
    assert ops().embedding(torch.zeros(2, 3, dtype=torch.int32, device=DEV), table, 1.0).shape == (2, 3, 6)
    assert ops().embedding(torch.zeros(4, dtype=torch.int32, device=DEV), table[:0], 1.0).abs().sum() == 0       # an empty table
    assert ops().embedding(torch.zeros(4, dtype=torch.int32, device=DEV), table[:, :0], 1.0).shape == (4, 0)
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 31, 4], device=DEV)
    assert (ops().embedding(far, table, 1.0)[:3] == 0).all() and torch.equal(ops().embedding(far, table, 1.0)[3], table[4])
    # values that are not finite stay in the rows that name them
    table[2] = float('nan'); table[3] = float('inf')
    out = cabi.embedding(torch.tensor([0, 2, 3, -1, 1], device=DEV), table, -1.0)
    assert torch.equal(out[0], -table[0]) and out[1].isnan().all() and (out[2] == -float('inf')).all() and (out[3] == 0).all()
    grad = randn(gen(1), 4, 6)
    grad[3] = float('nan')
    idx = torch.tensor([0, 1, 0, -1], device=DEV)                    # the NaN belongs to a padded slot
    order, start = cabi.group_by_key(idx, 3)
    got = cabi.embedding_grad(grad, idx, order, start)
    assert torch.allclose(got[0], grad[0] + grad[2]) and torch.equal(got[1], grad[1]) and (got[2] == 0).all()
    none = torch.full((9,), -1, device=DEV)
    order, start = cabi.group_by_key(none, 3)
    assert (cabi.embedding_grad(randn(gen(2), 9, 6), none, order, start, out=torch.full((3, 6), 7.0, device=DEV)) == 0).all()
    order, start = cabi.group_by_key(none[:0], 3)
    assert (cabi.embedding_grad(randn(gen(2), 0, 6), none[:0], order, start, out=torch.full((3, 6), 7.0, device=DEV)) == 0).all()


def test_lookup_beyond_32_bit_offsets():
    """A table of 2.2e9 elements, and rows at its far end."""
    rows, width = 2200000, 1000
    table = torch.zeros(rows, width, dtype=torch.float16, device=DEV)
    table[-3:] = torch.arange(3 * width, device=DEV).view(3, width) % 97
    idx = torch.tensor([rows - 3, 0, rows - 1, rows - 2, rows], device=DEV)
    out = ops().embedding(idx, table, 1.0)
    assert torch.equal(out[0], table[-3]) and torch.equal(out[2], table[-1]) and torch.equal(out[3], table[-2])
    assert (out[1] == 0).all() and (out[4] == 0).all()
    order, start = ops().group_by_key(idx, rows)
    got = ops().embedding_grad(torch.ones(5, width, dtype=torch.float16, device=DEV), idx, order, start, rows, 1.0)
    assert (got[-3:] == 1).all() and (got[0] == 1).all() and int((got[1:-3].view(torch.int16) != 0).sum()) == 0


# ---- one matrix per group --------------------------------------------------------------------------------------------
SIZES = [
    [1], [0, 1, 0], [5, 0, 7], [127, 128, 129], [64, 0, 0, 1, 300], [1000], [33] * 20, [0, 0, 0], [2, 700, 1, 0, 90], [257, 255, 0, 512],
]


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('K,N', [(1, 1), (3, 5), (8, 16), (64, 64), (100, 70), (336, 256), (780, 128), (129, 257), (512, 1), (65, 520), (256, 336)])
def test_grouped_products(K, N, dtype):
    g = gen(K * 1000 + N)
    for sizes in SIZES:
        used = sum(sizes)
        n = used + (3 if len(sizes) % 2 else 0)                       # rows behind the last group
        if n == 0:
            n = 2
        start = R.start_of(sizes, DEV)
        x, dy = randn(g, n, K, dtype=dtype), randn(g, n, N, dtype=dtype)
        x[used:], dy[used:] = float('nan'), float('inf')              # and nothing reads them
        W = (randn(g, len(sizes), K, N) / K ** 0.5).to(dtype)
        what = f'{sizes} {K} {N} {dtype}'
        y = ops().grouped_matmul(x, W, start, False)
        exact, mag = R.product(x, W, start)
        R.assert_within(y, exact, R.sum_bound(exact, mag, K, dtype), 'y ' + what)
        dx = ops().grouped_matmul(dy, W, start, True)
        exact, mag = R.product(dy, W, start, True)
        R.assert_within(dx, exact, R.sum_bound(exact, mag, N, dtype), 'dx ' + what)
        dW = ops().grouped_matmul_wgrad(x, dy, start)
        exact, mag, terms = R.wgrad(x, dy, start)
        R.assert_within(dW, exact, R.sum_bound(exact, mag, terms, dtype), 'dW ' + what)
        assert torch.equal(dW, ops().grouped_matmul_wgrad(x, dy, start))             # reproducible to the bit


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('K,N,sizes,front', [
    (336, 256, [9000, 4000, 3001], 0), (780, 256, [5000, 1, 0, 2500, 777], 5), (96, 48, [20000], 0), (1000, 1032, [130, 260, 0, 3] * 8, 0),
    (72, 80, [1] * 1024, 0), (48, 2048, [600, 5000], 1), (2048, 40, [600, 5000], 0)])
def test_larger_grouped_products(K, N, sizes, front, dtype):
    """Several tiles in every direction, long sums over rows, up to 1,024 groups, groups that do not begin at row 0."""
    g = gen(K + N)
    n = front + sum(sizes) + 11
    start = R.start_of(sizes, DEV, front)
    x, dy, W = randn(g, n, K, dtype=dtype), randn(g, n, N, dtype=dtype), (randn(g, len(sizes), K, N) / K ** 0.5).to(dtype)
    y, dx, dW = ops().grouped_matmul(x, W, start, False), ops().grouped_matmul(dy, W, start, True), ops().grouped_matmul_wgrad(x, dy, start)
    for name, got, (exact, mag, *terms), m in (('y', y, R.product(x, W, start), K), ('dx', dx, R.product(dy, W, start, True), N),
                                               ('dW', dW, R.wgrad(x, dy, start), 0)):
        t = terms[0] if terms else m
        R.assert_within(got, exact, R.sum_bound(exact, mag, t, dtype), name)
        longest = int(t.max()) if terms else m
        # random signs: errors of the additions add up like their root; 16 u for runs of truncating additions, h of the result
        assert R.relative(got, exact) < (longest ** 0.5 + 16) * R.U + R.half_step(dtype)
    assert torch.equal(dW, ops().grouped_matmul_wgrad(x, dy, start)) and torch.equal(y, ops().grouped_matmul(x, W, start, False))
    assert (y[:front] == 0).all() and (y[-11:] == 0).all() and (dx[:front] == 0).all() and (dx[-11:] == 0).all()


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('K,N,sizes', [(136, 256, [30000, 9001, 2]), (64, 520, [20011, 5]), (520, 72, [39000]), (264, 264, [1, 21000, 0, 257, 128]),
                                       (48, 304, [38000, 255, 129]), (781, 40, [38001]),
                                       (776, 264, [20500, 1, 300]), (40, 1032, [6000, 5999])])
def test_products_of_large_groups(K, N, sizes, dtype):
    """Groups of tens of thousands of rows, tiles that end anywhere in a group, columns that end anywhere in a tile."""
    g = gen(K * 3 + N)
    n = sum(sizes) + 200
    start = R.start_of(sizes, DEV, 7)
    x, dy, W = randn(g, n, K, dtype=dtype), randn(g, n, N, dtype=dtype), (randn(g, len(sizes), K, N) / K ** 0.5).to(dtype)
    y, dx, dW = ops().grouped_matmul(x, W, start, False), ops().grouped_matmul(dy, W, start, True), ops().grouped_matmul_wgrad(x, dy, start)
    for name, got, (exact, mag, *terms), m in (('y', y, R.product(x, W, start), K), ('dx', dx, R.product(dy, W, start, True), N),
                                               ('dW', dW, R.wgrad(x, dy, start), 0)):
        R.assert_within(got, exact, R.sum_bound(exact, mag, terms[0] if terms else m, dtype), name)
        longest = int(terms[0].max()) if terms else m
        assert R.relative(got, exact) < (longest ** 0.5 + 16) * R.U + R.half_step(dtype)
    assert torch.equal(dW, ops().grouped_matmul_wgrad(x, dy, start)) and torch.equal(y, ops().grouped_matmul(x, W, start, False))
    from qml_lightning_b200 import cabi
    assert cabi.tc_timeouts() == 0


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('K,N', [(20, 12), (336, 256), (1100, 520)])
@pytest.mark.parametrize('sizes', [[0, 13, 0], [0, 200, 0], [0, 0, 2500, 0], [700, 0, 701, 0], [0, 9000, 0, 1], [0, 0]])
def test_every_result_is_written(sizes, K, N, dtype):
    """Whatever stood in the outputs and in the scratch, groups without rows have zero gradients, rows without a group zero rows."""
    from qml_lightning_b200 import cabi
    g = gen(K + len(sizes))
    used, front = sum(sizes), 2
    n = used + 5
    start = R.start_of(sizes, DEV, front)
    x, dy, W = randn(g, n, K, dtype=dtype), randn(g, n, N, dtype=dtype), (randn(g, len(sizes), K, N) / K ** 0.5).to(dtype)
    nan = lambda *shape: torch.full(shape, float('nan'), dtype=dtype, device=DEV)
    scratch = torch.full((1 << 24,), float('nan'), device=DEV)        # freed: what the calls below allocate comes from it
    del scratch
    dW = cabi.grouped_matmul_wgrad(x, dy, start, out=nan(len(sizes), K, N))
    y = cabi.grouped_matmul(x, W, start, out=nan(n, N))
    dx = cabi.grouped_matmul(dy, W, start, transpose=True, out=nan(n, K))
    for i, rows in enumerate(sizes):
        assert rows or (dW[i] == 0).all()
    for t in (y, dx):
        assert (t[:front] == 0).all() and (t[front + used:] == 0).all()
    for got, (exact, mag, *terms), m in ((y, R.product(x, W, start), K), (dx, R.product(dy, W, start, True), N), (dW, R.wgrad(x, dy, start), 0)):
        R.assert_within(got, exact, R.sum_bound(exact, mag, terms[0] if terms else m, dtype), f'{sizes} {K} {N}')


@pytest.mark.parametrize('dtype', R.TYPES)
def test_products_of_misaligned_tensors(dtype):
    g = gen(5)
    sizes, K, N = [70, 0, 200], 64, 128
    start = R.start_of(sizes, DEV)
    x, dy, W = randn(g, 270, K, dtype=dtype), randn(g, 270, N, dtype=dtype), randn(g, 3, K, N, dtype=dtype)
    y, dx, dW = ops().grouped_matmul(x, W, start, False), ops().grouped_matmul(dy, W, start, True), ops().grouped_matmul_wgrad(x, dy, start)
    for a, b, c in ((misaligned(x), W, dy), (x, misaligned(W), dy), (x, W, misaligned(dy)), (misaligned(x), misaligned(W), misaligned(dy))):
        e, m = R.product(x, W, start)
        R.assert_within(ops().grouped_matmul(a, b, start, False), e, R.sum_bound(e, m, K, dtype), 'y')
        e, m = R.product(dy, W, start, True)
        R.assert_within(ops().grouped_matmul(c, b, start, True), e, R.sum_bound(e, m, N, dtype), 'dx')
        e, m, t = R.wgrad(x, dy, start)
        R.assert_within(ops().grouped_matmul_wgrad(a, c, start), e, R.sum_bound(e, m, t, dtype), 'dW')
    from qml_lightning_b200 import cabi
    for got, want in ((cabi.grouped_matmul(x, W, start, out=misaligned(torch.zeros_like(y))), y),
                      (cabi.grouped_matmul(dy, W, start, transpose=True, out=misaligned(torch.zeros_like(dx))), dx),
                      (cabi.grouped_matmul_wgrad(x, dy, start, out=misaligned(torch.zeros_like(dW))), dW)):
        assert R.relative(got, want.double()) <= 2 * R.half_step(dtype)


@pytest.mark.parametrize('dtype', R.TYPES)
def test_products_keep_magnitudes_apart(dtype):
    """Rows and columns whose values differ by many powers of two: every row is as exact as if it were alone."""
    g = gen(6)
    K, N, n = 200, 96, 300
    start = R.start_of([150, 150], DEV)
    span = 6 if dtype == torch.float16 else 40
    x = (randn(g, n, K) * 2.0 ** torch.randint(-span, span, (n, 1), generator=g, device=DEV)).to(dtype)
    W = (randn(g, 2, K, N) * 2.0 ** torch.randint(-4, 4, (2, 1, N), generator=g, device=DEV)).to(dtype)
    y = ops().grouped_matmul(x, W, start, False)
    exact, mag = R.product(x, W, start)
    R.assert_within(y, exact, R.sum_bound(exact, mag, K, dtype), 'y')


@pytest.mark.parametrize('K,N', [(64, 32), (63, 32), (60, 31), (66, 36)])
def test_values_that_are_not_finite_stay_in_their_rows(K, N):
    g = gen(7)
    for dtype in R.TYPES:
        for n in (300, 3000):
            x, W = randn(g, n, K, dtype=dtype), randn(g, 2, K, N, dtype=dtype)
            start = R.start_of([130, n - 140], DEV)
            x[5], x[131, K - 2], x[n - 20, 0] = float('nan'), float('inf'), float('nan')
            W[0, 0, 7] = float('inf')
            y = ops().grouped_matmul(x, W, start, False)
            bad = ~torch.isfinite(y)
            assert bad[5].all() and bad[131].all() and bad[n - 20].all() and bad[:130, 7].all()
            bad[5], bad[131], bad[n - 20], bad[:130, 7] = False, False, False, False
            assert not bad.any()
            dy = randn(g, n, N, dtype=dtype)
            dy[77] = float('inf')
            bad = ~torch.isfinite(ops().grouped_matmul(dy, randn(g, 2, K, N, dtype=dtype), start, True))
            assert bad[77].all() and not bad[torch.arange(n, device=DEV) != 77].any()
            # a group's gradient is not touched by the rows of its neighbours
            dW = ops().grouped_matmul_wgrad(x, randn(g, n, N, dtype=dtype), R.start_of([5, 0, 100], DEV, 6))
            assert torch.isfinite(dW).all()


def test_bounds_outside_the_rows_are_clamped():
    """Bounds that no caller should pass lead to no access outside the tensors."""
    g = gen(8)
    for dtype in R.TYPES:
        x, W, dy = randn(g, 40, 24, dtype=dtype), randn(g, 3, 24, 16, dtype=dtype), randn(g, 40, 16, dtype=dtype)
        start = torch.tensor([-5, 10, 30, 1000], dtype=torch.int32, device=DEV)
        clamped = torch.tensor([0, 10, 30, 40], dtype=torch.int32, device=DEV)
        for got, want in ((ops().grouped_matmul(x, W, start, False), ops().grouped_matmul(x, W, clamped, False)),
                          (ops().grouped_matmul(dy, W, start, True), ops().grouped_matmul(dy, W, clamped, True)),
                          (ops().grouped_matmul_wgrad(x, dy, start), ops().grouped_matmul_wgrad(x, dy, clamped))):
            assert torch.equal(got, want)


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('n,K,N', [(100, 24, 16), (5000, 136, 72), (40000, 64, 48)])
def test_descending_bounds_stay_inside(n, K, N, dtype):
    """Groups that overlap, if their bounds were taken as they are, hold many times n rows: tiles, scratch and results keep their
    sizes, and what follows on the stream is right."""
    from qml_lightning_b200 import _lib, cabi
    g = gen(n)
    groups = 64
    x, dy, W = randn(g, n, K, dtype=dtype), randn(g, n, N, dtype=dtype), randn(g, groups, K, N, dtype=dtype)
    start = torch.tensor([0, n] * (groups // 2) + [0], dtype=torch.int32, device=DEV)
    code, lib, stream = cabi._DTYPES[dtype], _lib.load(), torch.cuda.current_stream().cuda_stream
    guard = 1 << 20

    def call(name, a, b, out_numel, *tail):
        nbytes = getattr(lib, name + '_workspace_bytes')(n, groups, K, N, code, *tail)
        ws = torch.full((nbytes + guard,), 85, dtype=torch.uint8, device=DEV)
        out = torch.full((out_numel + guard,), 3.0, dtype=dtype, device=DEV)
        assert getattr(lib, name)(a.data_ptr(), b.data_ptr(), start.data_ptr(), code, n, groups, K, N, *tail, out.data_ptr(), ws.data_ptr(),
                                  nbytes, stream) == 0
        assert (ws[nbytes:] == 85).all() and (out[out_numel:] == 3).all()

    call('qmlb_grouped_matmul', x, W, n * N, 0)
    call('qmlb_grouped_matmul', dy, W, n * K, 1)
    call('qmlb_grouped_matmul_wgrad', x, dy, groups * K * N)
    start = R.start_of([n // 3, 0, n // 2] + [0] * (groups - 3), DEV)
    exact, mag, terms = R.wgrad(x, dy, start)
    R.assert_within(ops().grouped_matmul_wgrad(x, dy, start), exact, R.sum_bound(exact, mag, terms, dtype), 'dW')
    assert cabi.tc_timeouts() == 0


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,K,N', [(2200001, 1000, 24), (2200003, 24, 1000)])
def test_products_beyond_32_bit_offsets(n, K, N, dtype):
    """Rows and results of 2.2e9 elements: groups at both ends, compared with the products of their rows alone."""
    g = gen(11)
    x, dy = torch.zeros(n, K, dtype=dtype, device=DEV), torch.zeros(n, N, dtype=dtype, device=DEV)
    W = (randn(g, 3, K, N) / K ** 0.5).to(dtype)
    start = R.start_of([300, n - 300 - 700, 693], DEV)
    parts = [(0, 300), (n - 700, n - 7)]
    for a, b in parts:
        x[a:b], dy[a:b] = randn(g, b - a, K, dtype=dtype), randn(g, b - a, N, dtype=dtype)
    dW = ops().grouped_matmul_wgrad(x, dy, start)
    assert (dW[1] == 0).all()
    for (a, b), e in zip(parts, (0, 2)):
        exact, mag, terms = R.wgrad(x[a:b], dy[a:b], R.start_of([b - a], DEV))
        R.assert_within(dW[e:e + 1], exact, R.sum_bound(exact, mag, terms, dtype), f'dW {e}')
    for transpose, rows, depth in ((False, x, K), (True, dy, N)):
        out = ops().grouped_matmul(rows, W, start, transpose)
        for (a, b), e in zip(parts, (0, 2)):
            exact, mag = R.product(rows[a:b], W[e:e + 1], R.start_of([b - a], DEV), transpose)
            R.assert_within(out[a:b], exact, R.sum_bound(exact, mag, depth, dtype), f'{transpose} {e}')
        assert int(out[300:n - 700].count_nonzero()) == 0 and int(out[n - 7:].count_nonzero()) == 0
        del out


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_matrices_beyond_32_bit_offsets(dtype):
    """1,024 matrices of 2.2e9 elements together, rows for the first and the last."""
    g = gen(12)
    G, K, N = 1024, 1050, 2056
    W = torch.zeros(G, K, N, dtype=dtype, device=DEV)
    W[0], W[-1] = randn(g, K, N, dtype=dtype), randn(g, K, N, dtype=dtype)
    for a, b in ((9, 11), (2000, 2500)):
        x, dy = randn(g, a + b, K, dtype=dtype), randn(g, a + b, N, dtype=dtype)
        start = R.start_of([a] + [0] * (G - 2) + [b], DEV)
        small, ends = R.start_of([a, b], DEV), torch.stack([W[0], W[-1]])
        for transpose, rows, depth in ((False, x, K), (True, dy, N)):
            exact, mag = R.product(rows, ends, small, transpose)
            R.assert_within(ops().grouped_matmul(rows, W, start, transpose), exact, R.sum_bound(exact, mag, depth, dtype), f'{a} {transpose}')
        dW = ops().grouped_matmul_wgrad(x, dy, start)
        exact, mag, terms = R.wgrad(x, dy, small)
        R.assert_within(torch.stack([dW[0], dW[-1]]), exact, R.sum_bound(exact, mag, terms, dtype), f'dW {a}')
        assert int(dW[1:-1].count_nonzero()) == 0
        del dW


def test_largest_number_of_keys():
    nkeys = 2 ** 31 - 2
    for n in (5, 150000):
        keys = torch.randint(0, nkeys, (n,), generator=gen(n), device=DEV)
        keys[0], keys[1], keys[3] = nkeys - 1, -1, nkeys
        order, start = ops().group_by_key(keys, nkeys)
        inside = (keys >= 0) & (keys < nkeys)
        ref = torch.sort(torch.where(inside, keys, torch.full_like(keys, nkeys)), stable=True)[1].int()
        assert torch.equal(order, ref)
        used = int(inside.sum())
        assert int(start[0]) == 0 and int(start[-1]) == used and int(start[-2]) == used - int((keys == nkeys - 1).sum())
        at = keys[ref[:used].long()]
        rank = torch.searchsorted(at, at)                                  # first position of the same key
        assert torch.equal(start[at].long(), rank)
        del start


def test_outputs_do_not_overlap_inputs():
    from qml_lightning_b200 import cabi
    x, W, start = torch.zeros(6, 8, device=DEV), torch.zeros(1, 8, 8, device=DEV), R.start_of([6], DEV)
    idx = torch.arange(6, device=DEV)
    order, first = cabi.group_by_key(idx, 6)
    for call in (lambda: cabi.grouped_matmul(x, W, start, out=x), lambda: cabi.grouped_matmul_wgrad(W[0], W[0], start, out=W),
                 lambda: cabi.embedding(idx, x, out=x), lambda: cabi.embedding_grad(x, idx, order, first, out=x)):
        with pytest.raises(RuntimeError, match='overlap'):
            call()


def test_empty_products():
    for dtype in R.TYPES:
        W = torch.ones(2, 3, 4, dtype=dtype, device=DEV)
        start = R.start_of([0, 0], DEV)
        assert ops().grouped_matmul(torch.ones(0, 3, dtype=dtype, device=DEV), W, start, False).shape == (0, 4)
        assert (ops().grouped_matmul(torch.ones(5, 3, dtype=dtype, device=DEV), W, start, False) == 0).all()
        assert (ops().grouped_matmul(torch.ones(5, 0, dtype=dtype, device=DEV), W[:, :0], R.start_of([2, 3], DEV), False) == 0).all()
        dW = ops().grouped_matmul_wgrad(torch.ones(0, 3, dtype=dtype, device=DEV), torch.ones(0, 4, dtype=dtype, device=DEV), start)
        assert dW.shape == (2, 3, 4) and (dW == 0).all()


def test_refusals():
    i = torch.zeros(4, dtype=torch.int32, device=DEV)
    x, W, start = torch.zeros(4, 8, device=DEV), torch.zeros(2, 8, 3, device=DEV), R.start_of([2, 2], DEV)
    for call, word in (
            (lambda: ops().group_by_key(x, 3), 'int32 or int64'), (lambda: ops().group_by_key(i, 0), 'nkeys'),
            (lambda: ops().group_by_key(i, 2 ** 31 - 1), 'nkeys'), (lambda: ops().embedding(i.cpu(), x, 1.0), 'CUDA'),
            (lambda: ops().embedding(i.float(), x, 1.0), 'int32 or int64'), (lambda: ops().embedding(i, x.double(), 1.0), 'float32, float16'),
            (lambda: ops().embedding(i, x[0], 1.0), 'rows, width'), (lambda: ops().embedding_grad(x[:3], i, i, i, 3, 1.0), 'shape of indices'),
            (lambda: ops().embedding_grad(x, i, i[:2], i, 3, 1.0), 'order'), (lambda: ops().embedding_grad(x, i, i, i, 9, 1.0), 'rows \\+ 1'),
            (lambda: ops().grouped_matmul(x, W.half(), start, False), 'dtype'), (lambda: ops().grouped_matmul(x, W, start, True), 'columns'),
            (lambda: ops().grouped_matmul(x, W, start[:2], False), 'one entry per group'),
            (lambda: ops().grouped_matmul(x, W[0], start, False), 'groups'), (lambda: ops().grouped_matmul(x, W.double(), start, False), 'dtype|float32'),
            (lambda: ops().grouped_matmul(x, torch.zeros(1025, 8, 3, device=DEV), torch.zeros(1026, dtype=torch.int32, device=DEV), False), '1024 groups'),
            (lambda: ops().grouped_matmul_wgrad(x, x[:3], start), 'number of rows'), (lambda: ops().grouped_matmul_wgrad(x, x.half(), start), 'dtype')):
        with pytest.raises(RuntimeError, match=word):
            call()


# ---- gradients, streams, graphs, and the operators together -------------------------------------------------------------
def layer(x, W, offset, element, groups):
    """A linear layer per element on unordered rows: ordered, gathered, multiplied, offset added; rows in element order."""
    order, start = ops().group_by_key(element, groups)
    rows = ops().embedding(order, x, 1.0)
    return ops().grouped_matmul(rows, W, start) + ops().embedding(element[order], offset, 2.0), order, start


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('n,K,N,groups', [(21, 48, 32, 3), (1000, 33, 17, 5), (3000, 128, 64, 40)])
def test_layer_and_its_gradients(n, K, N, groups, dtype):
    g = gen(n)
    element = torch.randint(-1, groups, (n,), generator=g, device=DEV, dtype=torch.int32)
    x, W, offset = (t.requires_grad_(True) for t in (randn(g, n, K, dtype=dtype), (randn(g, groups, K, N) / K ** 0.5).to(dtype),
                                                     randn(g, groups, N, dtype=dtype)))
    y, order, start = layer(x, W, offset, element, groups)
    dy = randn(g, n, N, dtype=dtype)
    dx, dW, doff = torch.autograd.grad(y, (x, W, offset), dy)
    with torch.no_grad():
        want, wstart = R.order_of(element, groups)
        assert torch.equal(order, want) and torch.equal(start, wstart)
        rows = x[order.long()]
        exact, mag = R.product(rows, W, start)
        off = R.lookup(element[order.long()], offset, 2.0)
        # both terms and their sum are rounded to the type
        R.assert_within(y, exact + off, R.sum_bound(exact, mag, K, dtype) + R.lookup_bound(off, dtype)
                        + 1.1 * R.half_step(dtype) * (exact + off).abs() + R.half_step(dtype) ** 2 * 4 * (exact.abs() + off.abs()), 'y')
        e, m = R.product(dy, W, start, True)
        back, bm = torch.empty_like(e), torch.empty_like(m)
        back[order.long()], bm[order.long()] = e, m
        R.assert_within(dx, back, R.sum_bound(back, bm, N, dtype), 'dx')
        e, m, t = R.wgrad(rows, dy, start)
        R.assert_within(dW, e, R.sum_bound(e, m, t, dtype), 'dW')
        e, m, t = R.lookup_grad(element[order.long()], dy, groups, 2.0)
        R.assert_within(doff, e, R.sum_bound(e, m, t.view(-1, 1), dtype), 'doffset')


def test_gradients_against_differences():
    """All operators are linear in each argument, so a difference over any step is the derivative up to rounding."""
    g = gen(20)
    n, K, N, groups = 200, 24, 20, 4
    element = torch.randint(-1, groups, (n,), generator=g, device=DEV)
    leaves = [randn(g, n, K), randn(g, groups, K, N), randn(g, groups, N)]
    dy = randn(g, n, N)
    grads = torch.autograd.grad(layer(*[t.requires_grad_(True) for t in leaves], element, groups)[0], leaves, dy)
    with torch.no_grad():
        f = lambda ts: (layer(*ts, element, groups)[0].double() * dy.double()).sum()  # noqa: E731
        size = float(layer(*[t.abs() for t in leaves], element, groups)[0].double().mul(dy.double().abs()).sum())
        for k, t in enumerate(leaves):
            d = randn(g, *t.shape)
            moved = [u + d if i == k else u for i, u in enumerate(leaves)]
            diff = float(f(moved) - f(leaves))
            assert abs(diff - float((grads[k].double() * d.double()).sum())) <= 64 * R.U * size


def test_second_derivatives():
    """Gradients of gradients (force training differentiates a gradient): against the same chain in 64-bit torch."""
    g = gen(21)
    n, K, N, groups = 60, 12, 10, 3
    element = torch.randint(-1, groups, (n,), generator=g, device=DEV)
    leaves = [randn(g, n, K), randn(g, groups, K, N), randn(g, groups, N)]

    def own(x, W, offset):
        return layer(x, W, offset, element, groups)[0]

    def plain(x, W, offset):
        order, start = R.order_of(element, groups)
        rows, el = x[order.long()], element[order.long()]
        ok = (el >= 0).unsqueeze(1)
        e = el.clamp(min=0)
        return torch.where(ok, torch.einsum('rk,rkn->rn', rows, W[e]) + 2 * offset[e], torch.zeros((), dtype=x.dtype, device=DEV))

    def penalty(f, ts):
        ts = [t.detach().clone().requires_grad_(True) for t in ts]
        energy = torch.tanh(f(*ts)).sum()
        dx, doff = torch.autograd.grad(energy, (ts[0], ts[2]), create_graph=True)
        return torch.autograd.grad((dx ** 2).sum() + (doff ** 3).sum(), ts)

    for a, b in zip(penalty(own, leaves), penalty(plain, [t.double() for t in leaves])):
        assert R.relative(a, b) < 1e-4       # tanh and cubes amplify the 32-bit roundings of the chain; a lost term is of order 1


def test_gradient_of_broadcast_and_transposed_tensors():
    g = gen(22)
    table = randn(g, 6, 10).requires_grad_(True)
    idx = torch.randint(0, 6, (7, 4), generator=g, device=DEV)
    grad, = torch.autograd.grad(ops().embedding(idx, table, 1.0).sum(), table)                     # an expanded gradient
    assert torch.equal(grad, torch.bincount(idx.reshape(-1), minlength=6).float().unsqueeze(1).expand(6, 10))
    W = randn(g, 2, 8, 12).transpose(1, 2).requires_grad_(True)                                     # not contiguous
    x = randn(g, 12, 30).t().requires_grad_(True)
    start = R.start_of([10, 20], DEV)
    y = ops().grouped_matmul(x, W, start)
    dx, dW = torch.autograd.grad(y.sum(), (x, W))
    ones = torch.ones_like(y)
    assert R.relative(y, R.product(x.detach(), W.detach(), start)[0]) < 1e-6
    assert R.relative(dx, R.product(ones, W.detach(), start, True)[0]) < 1e-6 and R.relative(dW, R.wgrad(x.detach(), ones, start)[0]) < 1e-6


def test_streams_run_apart():
    """The same operators on two streams at once, each with its own inputs."""
    g = gen(23)
    jobs = []
    for k in range(4):
        n, K, N, G = 4000 + 100 * k, 96, 64, 5
        jobs.append((randn(g, n, K, dtype=R.TYPES[k % 3]), (randn(g, G, K, N) / 10).to(R.TYPES[k % 3]), randn(g, G, N, dtype=R.TYPES[k % 3]),
                     torch.randint(-1, G, (n,), generator=g, device=DEV), G))
    with torch.no_grad():
        want = [layer(*j)[0] for j in jobs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(DEV) for _ in jobs]
        got = []
        for _ in range(3):
            got = []
            for s, j in zip(streams, jobs):
                with torch.cuda.stream(s):
                    got.append(layer(*j)[0])
        torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', R.TYPES)
def test_first_call_of_a_thread(dtype):
    """A backward pass runs in a thread of its own, whose first call to the device may be one of these."""
    import threading
    g = gen(30)
    x, W, dy = randn(g, 3000, 64, dtype=dtype), randn(g, 2, 64, 48, dtype=dtype), randn(g, 3000, 48, dtype=dtype)
    start = R.start_of([1000, 1900], DEV)
    keys = torch.randint(0, 9, (3000,), generator=g, device=DEV)

    def calls():
        order, first = ops().group_by_key(keys, 9)
        return [ops().grouped_matmul(x, W, start, False), ops().grouped_matmul(dy, W, start, True), ops().grouped_matmul_wgrad(x, dy, start), order,
                ops().embedding(keys, x, 1.0), ops().embedding_grad(x, keys, order, first, 9, 1.0)]

    want = calls()                                                    # the allocator has every block by now
    for k in range(len(want)):
        got, errors = [], []

        def work(k=k):
            try:
                first = [lambda: ops().grouped_matmul(x, W, start, False), lambda: ops().grouped_matmul(dy, W, start, True),
                         lambda: ops().grouped_matmul_wgrad(x, dy, start), lambda: ops().group_by_key(keys, 9)[0],
                         lambda: ops().embedding(keys, x, 1.0), lambda: ops().embedding_grad(x, keys, want[3], ops().group_by_key(keys, 9)[1], 9, 1.0)][k]
                got.append(first())
                torch.cuda.synchronize()
            except Exception as e:  # noqa: BLE001
                errors.append(e)
        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert not errors, errors
        assert torch.equal(got[0], want[k])


def test_captured_step_replays_on_new_inputs():
    """A whole step with its gradients in a CUDA graph; two graphs share nothing; no operator waits for the device."""
    g = gen(24)
    G, K, N = 5, 80, 48

    def make(n):
        return [randn(g, n, K).requires_grad_(True), (randn(g, G, K, N) / 9).requires_grad_(True), randn(g, G, N).requires_grad_(True),
                torch.randint(-1, G, (n,), generator=g, device=DEV, dtype=torch.int32), randn(g, n, N)]

    def step(x, W, offset, element, dy):
        y = layer(x, W, offset, element, G)[0]
        return (y,) + torch.autograd.grad(y, (x, W, offset), dy)

    states, graphs, outs = [make(3000), make(3000)], [], []
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            step(*s)
    torch.cuda.current_stream().wait_stream(side)
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    for round_ in range(2):
        fresh = [make(3000), make(3000)]
        with torch.no_grad():
            for s, f in zip(states, fresh):
                for a, b in zip(s, f):
                    a.copy_(b)
        torch.cuda.synchronize()
        pair = [torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)]
        for graph, stream in zip(graphs, pair):                       # both graphs at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, f in zip(outs, fresh):
            for a, b in zip(out, step(*f)):
                assert torch.equal(a, b)


def test_wrappers_of_the_c_abi_agree_with_the_operators():
    from qml_lightning_b200 import cabi
    g = gen(25)
    keys = torch.randint(-1, 6, (500,), generator=g, device=DEV)
    order, start = cabi.group_by_key(keys, 6)
    assert torch.equal(order, ops().group_by_key(keys, 6)[0]) and torch.equal(start, ops().group_by_key(keys, 6)[1])
    table, grad = randn(g, 6, 36), randn(g, 500, 36)
    assert torch.equal(cabi.embedding(keys, table, 3.0), ops().embedding(keys, table, 3.0))
    assert torch.equal(cabi.embedding_grad(grad, keys, order, start, 3.0), ops().embedding_grad(grad, keys, order, start, 6, 3.0))
    x, W, dy = randn(g, 500, 40), randn(g, 6, 40, 24), randn(g, 500, 24)
    assert torch.equal(cabi.grouped_matmul(x, W, start), ops().grouped_matmul(x, W, start, False))
    assert torch.equal(cabi.grouped_matmul(dy, W, start, transpose=True), ops().grouped_matmul(dy, W, start, True))
    assert torch.equal(cabi.grouped_matmul_wgrad(x, dy, start), ops().grouped_matmul_wgrad(x, dy, start))
    with pytest.raises(RuntimeError, match='contiguous'):
        cabi.grouped_matmul(x.t().contiguous().t(), W, start)
    with pytest.raises(RuntimeError, match='out must be'):
        cabi.grouped_matmul(x, W, start, out=torch.empty(3, 3, device=DEV))
