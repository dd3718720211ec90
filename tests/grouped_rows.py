"""64-bit oracles and error bounds for the operators on rows that belong to groups.

Bounds.  u = 2^-24 is the unit roundoff of float32, h = eps / 2 that of the result's type.  A float32 sum of m terms in any
order, where every addition may also truncate (2 u instead of u), is off by at most 2 m u * sum|terms|; float32 operands
that enter a product as two fp16 parts x = h + l + r have |l| <= 2^-11 |x| and |r| <= 2^-11 |l| <= 2^-22 |x| = 4 u |x|; the
product h h' + h l' + l h' leaves out r x', x r' and l l', at most 3 * 2^-22 = 12 u of it.  (Parts below fp16's normal range are
off by 2^-39 of the largest value of their 64-value stretch, which these inputs keep far below 12 u of the sum.)  The result
is rounded once (h of its value).
"""
import torch

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def order_of(keys, nkeys):
    k = keys.reshape(-1).long()
    k = torch.where((k < 0) | (k >= nkeys), torch.full_like(k, nkeys), k)
    order = torch.sort(k, stable=True)[1]
    start = torch.searchsorted(k[order].contiguous(), torch.arange(nkeys + 1, device=k.device))
    return order.int(), start.int()


def lookup(indices, table, scale):
    idx = indices.reshape(-1).long()
    ok = (idx >= 0) & (idx < table.shape[0])
    out = torch.zeros(idx.numel(), table.shape[1], dtype=torch.float64, device=table.device)
    out[ok] = table.double()[idx[ok]] * scale
    return out.reshape(tuple(indices.shape) + (table.shape[1],))


def lookup_bound(exact, dtype):
    # the factor and the product are rounded to float32, the result once to its type (fp16: absolute below its normal range)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return exact.abs() * (half_step(dtype) + 2.1 * U) + tiny


def lookup_grad(indices, grad, rows, scale):
    """(exact, sum of absolute terms, terms per row)"""
    idx = indices.reshape(-1).long()
    ok = (idx >= 0) & (idx < rows)
    g = grad.reshape(idx.numel(), -1).double()[ok] * scale
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=grad.device)
    mag = torch.zeros_like(out).index_add_(0, idx[ok], g.abs())
    return out.index_add_(0, idx[ok], g), mag, torch.bincount(idx[ok], minlength=rows)


def sum_bound(exact, magnitude, terms, dtype):
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return magnitude * (2 * terms + 14) * U + exact.abs() * half_step(dtype) * 1.01 + tiny


def groups_of(start, n):
    s = [min(max(int(v), 0), n) for v in start.tolist()]
    return [(a, max(a, b)) for a, b in zip(s[:-1], s[1:])]


def product(x, W, start, transpose=False):
    """(exact, sum of absolute products)"""
    B = W.double().transpose(1, 2) if transpose else W.double()
    y = torch.zeros(x.shape[0], B.shape[2], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for g, (a, b) in enumerate(groups_of(start, x.shape[0])):
        y[a:b] = x[a:b].double() @ B[g]
        mag[a:b] = x[a:b].double().abs() @ B[g].abs()
    return y, mag


def wgrad(x, dy, start):
    """(exact, sum of absolute products, rows per group)"""
    bounds = groups_of(start, x.shape[0])
    dW = torch.zeros(len(bounds), x.shape[1], dy.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(dW)
    for g, (a, b) in enumerate(bounds):
        dW[g] = x[a:b].double().T @ dy[a:b].double()
        mag[g] = x[a:b].double().abs().T @ dy[a:b].double().abs()
    return dW, mag, torch.tensor([b - a for a, b in bounds], device=x.device).view(-1, 1, 1)


def assert_within(got, exact, bound, what=''):
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    off = (got.double() - exact).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values outside the bound, worst {float((off / bound.clamp(min=1e-300)).max()):.3g} times"


def relative(got, exact):
    norm = float(exact.norm())
    got = got.detach().double()
    return float((got - exact).norm()) / norm if norm else float(got.norm())


def start_of(sizes, device, front=0):
    out = [front]
    for s in sizes:
        out.append(out[-1] + s)
    return torch.tensor(out, dtype=torch.int32, device=device)
