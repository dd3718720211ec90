"""Forward-mode derivatives of the differentiable operators on grouped rows: each map is linear in every argument, so a tangent is
one call of an operator of this family, and forward mode composes with reverse mode.  Tangents are compared with the formula in 64
bits."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests import grouped_rows as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def ops():
    import qml_lightning_b200  # noqa: F401
    return torch.ops.qml_lightning_b200


def data(dtype=torch.float32, n=300, K=24, N=20, G=4):
    g = torch.Generator(device=DEV).manual_seed(n)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    element = torch.randint(-1, G, (n,), generator=g, device=DEV)
    order, start = ops().group_by_key(element, G)
    return dict(x=r(n, K), dx=r(n, K), W=r(G, K, N), dW=r(G, K, N), g=r(n, N), dg=r(n, N), table=r(G, K), dtable=r(G, K), element=element,
                order=order, start=start, G=G, n=n, K=K, N=N)


def tangent(f, *pairs):
    with fwAD.dual_level():
        out = fwAD.unpack_dual(f(*[fwAD.make_dual(p, t) if t is not None else p for p, t in pairs]))
        assert out.tangent is not None, 'no tangent'
        return out.primal, out.tangent


@pytest.mark.parametrize('dtype', R.TYPES)
@pytest.mark.parametrize('needs_grad', [False, True])
def test_tangents(dtype, needs_grad):
    d = data(dtype)
    leaf = lambda t: t.clone().requires_grad_(True) if needs_grad else t  # noqa: E731
    primal, t = tangent(lambda a: ops().embedding(d['element'], a, 1.5), (leaf(d['table']), d['dtable']))
    assert torch.equal(primal, ops().embedding(d['element'], d['table'], 1.5)) and torch.equal(t, ops().embedding(d['element'], d['dtable'], 1.5))
    exact = R.lookup(d['element'], d['dtable'], 1.5)
    R.assert_within(t.detach(), exact, R.lookup_bound(exact, dtype), 'lookup')
    primal, t = tangent(lambda a: ops().embedding_grad(a, d['element'], d['order'], d['start'], d['G'], 0.5), (leaf(d['x']), d['dx']))
    exact, mag, terms = R.lookup_grad(d['element'], d['dx'], d['G'], 0.5)
    R.assert_within(t.detach(), exact, R.sum_bound(exact, mag, terms.view(-1, 1), dtype), 'gradient of the table')
    # products: one argument moving, or both (the sum of two rounded tangents is rounded once more)
    for transpose, rows, drows in ((False, 'x', 'dx'), (True, 'g', 'dg')):
        f = lambda a, W: ops().grouped_matmul(a, W, d['start'], transpose)  # noqa: E731,B023
        a, b = R.product(d[drows], d['W'], d['start'], transpose), R.product(d[rows], d['dW'], d['start'], transpose)
        m = d['N'] if transpose else d['K']
        for move_rows, move_W in ((1, 0), (0, 1), (1, 1)):
            primal, t = tangent(f, (leaf(d[rows]), d[drows] if move_rows else None), (leaf(d['W']), d['dW'] if move_W else None))
            assert torch.equal(primal, ops().grouped_matmul(d[rows], d['W'], d['start'], transpose))
            exact, mag = move_rows * a[0] + move_W * b[0], move_rows * a[1] + move_W * b[1]
            parts = move_rows * a[0].abs() + move_W * b[0].abs()
            R.assert_within(t.detach(), exact, R.sum_bound(parts, mag, m, dtype) + 1.1 * R.half_step(dtype) * exact.abs()
                            + 4 * R.half_step(dtype) ** 2 * parts, f'{transpose} {move_rows} {move_W}')
    f = lambda a, b: ops().grouped_matmul_wgrad(a, b, d['start'])  # noqa: E731
    a, b = R.wgrad(d['dx'], d['g'], d['start']), R.wgrad(d['x'], d['dg'], d['start'])
    primal, t = tangent(f, (leaf(d['x']), d['dx']), (leaf(d['g']), d['dg']))
    parts = a[0].abs() + b[0].abs()
    R.assert_within(t.detach(), a[0] + b[0], R.sum_bound(parts, a[1] + b[1], a[2], dtype) + 1.1 * R.half_step(dtype) * (a[0] + b[0]).abs()
                    + 4 * R.half_step(dtype) ** 2 * parts, 'gradient of the matrices')


def test_forward_over_reverse():
    """A Hessian-vector product: the tangent of a gradient, against the same chain differentiated twice in reverse."""
    d = data(n=120, K=12, N=10)

    def energy(x, W, table):
        rows = ops().embedding(d['order'], x)
        y = ops().grouped_matmul(rows, W, d['start']) + ops().grouped_matmul(ops().embedding(d['element'][d['order'].long()], table), W, d['start'])
        return torch.tanh(y).sum()

    leaves, moves = (d['x'], d['W'], d['table']), (d['dx'], d['dW'], d['dtable'])
    with fwAD.dual_level():
        duals = [fwAD.make_dual(p.clone().requires_grad_(True), t) for p, t in zip(leaves, moves)]
        got = [fwAD.unpack_dual(v).tangent for v in torch.autograd.grad(energy(*duals), duals, create_graph=True)]
    ts = [p.clone().requires_grad_(True) for p in leaves]
    grads = torch.autograd.grad(energy(*ts), ts, create_graph=True)
    want = torch.autograd.grad(sum((a * b).sum() for a, b in zip(grads, moves)), ts)
    for a, b in zip(got, want):
        assert a is not None and R.relative(a, b.double()) < 1e-4        # 32-bit chains through tanh; a lost term is of order 1


def test_other_transforms():
    """Batching runs the operator slice by slice; transforms that it does not take are refused, never answered without a derivative."""
    d = data()
    f = lambda t: ops().embedding(d['element'], t, 1.0)  # noqa: E731
    h = lambda a: ops().grouped_matmul(a, d['W'], d['start'])  # noqa: E731
    k = lambda a: ops().grouped_matmul_wgrad(a, d['g'], d['start'])  # noqa: E731
    for fn, a, b in ((f, d['table'], d['dtable']), (h, d['x'], d['dx']), (k, d['x'], d['dx'])):
        try:
            batched = torch.func.vmap(fn)(torch.stack([a, b]))
        except RuntimeError:
            pass
        else:
            assert torch.equal(batched, torch.stack([fn(a), fn(b)]))
        try:
            primal, t = torch.func.jvp(fn, (a,), (b,))
        except RuntimeError:
            pass
        else:
            assert torch.equal(primal, fn(a)) and torch.equal(t, fn(b))
        try:
            grad = torch.func.grad(lambda v: (fn(v) ** 2).sum())(a)
        except RuntimeError:
            pass
        else:
            leaf = a.clone().requires_grad_(True)
            assert torch.equal(grad, torch.autograd.grad((fn(leaf) ** 2).sum(), leaf)[0])
