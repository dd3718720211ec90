"""Timed cases of the operators on rows that belong to groups: rows ordered by key, table lookup with its gradient,
and matrix products with one matrix per group.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass, ``exact``
gives the same outputs in 64 bits.  With ``own`` false a pass is written in elementary torch operations, with ``own``
true it calls the operators of this package.

Kinds of cases
  group           group_by_key: stable order of n keys and the first position of every key
  embedding       embedding: out[i] = scale * table[index[i]], zero rows for an index outside the table
  embedding_step  the same and the gradient of the table for a given gradient of the result
  product         grouped_matmul: y[r] = x[r] W[g] for the rows r of group g, zero rows behind the last group
  product_step    the same and the gradients of x and W
  layer           one training step of a linear layer per element: rows ordered by element, gathered, multiplied by their
                  element's matrix, an element's offset added; gradients of rows, matrices and offsets
"""
import math

import torch

own = False

TYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
ELEMENT_SIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}
LARGEST_BYTES = 3.0e9       # what a drawn case may move and compute at most: below the largest listed ones
LARGEST_FLOPS = 2.4e11


def listed():
    return [
        # the atoms of one training batch (64 molecules of 21 atoms, 5 elements): what a host loop calls every few microseconds
        dict(name='group-training-batch', kind='group', n=1344, keys=5, skew=1.0, outside=0.0, wide=False),
        # the atom slots of 200,000 mixed molecules (4 to 29 atoms, a little padding): one pass over millions of keys
        dict(name='group-200k-molecules', kind='group', n=3300000, keys=5, skew=1.0, outside=0.02, wide=False),
        # token numbers of a large vocabulary, 64-bit as torch gives them
        dict(name='group-vocabulary', kind='group', n=262143, keys=50021, skew=1.0, outside=0.0, wide=True),
        # one molecule looks its atom types up: the smallest call, latency only
        dict(name='embedding-molecule', kind='embedding', n=21, keys=10, width=64, type='float32', skew=0.5, outside=0.0, wide=False),
        # a large table, rows of 2 KB, most rows read once
        dict(name='embedding-large-table', kind='embedding', n=65535, keys=100003, width=1024, type='bfloat16', skew=0.7, outside=0.01, wide=True),
        # 10,000 conformers of 21 atoms and 3 elements: every table row collects tens of thousands of gradient rows
        dict(name='embedding-step-conformers', kind='embedding_step', n=210000, keys=3, width=256, type='float32', skew=1.0, outside=0.0, wide=False),
        # training on tokens of a vocabulary: short segments, a few long ones, many empty
        dict(name='embedding-step-vocabulary', kind='embedding_step', n=32769, keys=30011, width=768, type='bfloat16', skew=1.0, outside=0.03, wide=True),
        # one molecule through the projection of its elements (336 descriptors to 256): the smallest product
        dict(name='product-molecule', kind='product', n=21, groups=3, K=336, N=256, type='float32', skew=1.0, behind=0.0),
        # 10,000 conformers of 21 atoms, 3 elements, in 32 bits
        dict(name='product-conformers', kind='product', n=210000, groups=3, K=336, N=256, type='float32', skew=1.0, behind=0.0),
        # 20,000 mixed molecules, 5 elements, 780 descriptors: rows of 1,560 bytes, which no 16-byte load can follow
        dict(name='product-step-mixed', kind='product_step', n=330001, groups=5, K=780, N=256, type='bfloat16', skew=1.0, behind=0.01),
        # many groups of ragged sizes, some of them empty, matrices that outweigh the rows
        dict(name='product-step-many-groups', kind='product_step', n=16383, groups=64, K=1024, N=2048, type='float16', skew=0.8, behind=0.0),
        # a training step of a linear layer per element in 32 bits, from unordered rows with padded slots
        dict(name='layer-step', kind='layer', n=26880, groups=5, K=336, N=128, type='float32', skew=1.0, outside=0.1),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w['bytes'] <= LARGEST_BYTES and w['flops'] <= LARGEST_FLOPS and w['flops'] * (8 if case.get('type') == 'float32' else 1) <= 6 * LARGEST_FLOPS:
            return case


def _draw(rng):
    kind = rng.choice(['group', 'embedding', 'embedding_step', 'product', 'product_step', 'layer'])
    skew = round(rng.uniform(0.0, 1.2), 2)
    few = rng.random() < 0.5
    if kind == 'group':
        return dict(kind=kind, n=_spread(rng, 1, 3300000), keys=_spread(rng, 1, 32) if few else _spread(rng, 33, 200000), skew=skew,
                    outside=rng.choice([0.0, 0.02, 0.3]), wide=rng.random() < 0.5)
    if kind in ('embedding', 'embedding_step'):
        return dict(kind=kind, n=_spread(rng, 1, 400000), keys=_spread(rng, 1, 120) if few else _spread(rng, 121, 120000),
                    width=_spread(rng, 1, 2048), type=rng.choice(list(TYPES)), skew=skew, outside=rng.choice([0.0, 0.02, 0.3]),
                    wide=rng.random() < 0.5)
    even = rng.choice([1, 2, 4, 8, 8, 8])
    shape = dict(n=_spread(rng, 1, 330000), groups=_spread(rng, 1, 8) if few else _spread(rng, 9, 96),
                 K=-(-_spread(rng, 16, 2048) // even) * even, N=-(-_spread(rng, 16, 2048) // even) * even, type=rng.choice(list(TYPES)), skew=skew)
    if kind == 'layer':
        return dict(kind=kind, outside=rng.choice([0.0, 0.1]), **dict(shape, n=min(shape['n'], 60000)))
    return dict(kind=kind, behind=rng.choice([0.0, 0.05]), **shape)


def work(case):
    k = case['kind']
    n = case['n']
    if k == 'group':
        return {'bytes': n * (8 if case['wide'] else 4) + 4 * n + 4 * (case['keys'] + 1), 'flops': n}
    size = ELEMENT_SIZE[case['type']]
    if k in ('embedding', 'embedding_step'):
        rows = n * case['width'] * size
        table = case['keys'] * case['width'] * size
        forward = min(rows, table) + rows + n * (8 if case['wide'] else 4)
        if k == 'embedding':
            return {'bytes': forward, 'flops': n * case['width']}
        return {'bytes': forward + rows + table, 'flops': 2 * n * case['width']}
    g, K, N = case['groups'], case['K'], case['N']
    x, y, W = n * K * size, n * N * size, g * K * N * size
    if k == 'product':
        return {'bytes': x + W + y + 4 * (g + 1), 'flops': 2 * n * K * N}
    if k == 'product_step':        # x, W and dy in, y, dx and dW out
        return {'bytes': 2 * (x + W + y) + 4 * (g + 1), 'flops': 6 * n * K * N}
    return {'bytes': 2 * (x + W + y) + 8 * n + 2 * g * N * size, 'flops': 6 * n * K * N + 2 * n * N}


def _keys(case, count, gen):
    """Keys of falling frequency (rank r with weight (r + 1) ** -skew), in a random assignment of ranks to keys."""
    weight = torch.arange(1, count + 1, dtype=torch.float64, device='cuda') ** -case['skew']
    edge = torch.cumsum(weight, 0)
    u = torch.rand(case['n'], generator=gen, device='cuda', dtype=torch.float64) * edge[-1]
    rank = torch.searchsorted(edge, u).clamp(max=count - 1)
    return torch.randperm(count, generator=gen, device='cuda')[rank]


def _normal(gen, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device='cuda') * spread).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    k, n = case['kind'], case['n']
    state = dict(case)
    if k in ('group', 'embedding', 'embedding_step'):
        keys = _keys(case, case['keys'], gen)
        if case['outside']:        # padded slots carry -1
            keys[torch.rand(n, generator=gen, device='cuda') < case['outside']] = -1
        state['index'] = keys if case['wide'] else keys.to(torch.int32)
        if k != 'group':
            dtype = TYPES[case['type']]
            state['scale'] = math.sqrt(case['width'])
            state['table'] = _normal(gen, (case['keys'], case['width']), dtype, 1 / math.sqrt(case['width'])).requires_grad_(k == 'embedding_step')
            if k == 'embedding_step':
                state['dout'] = _normal(gen, (n, case['width']), dtype)
        return state
    g, K, N, dtype = case['groups'], case['K'], case['N'], TYPES[case['type']]
    learned = k != 'product'
    # descriptors are densities: not negative, and larger in some columns than in others
    column = torch.rand(K, generator=gen, device='cuda') + 0.1
    x = torch.randn((n, K), generator=gen, device='cuda').abs_().mul_(column)
    state['x'] = x.to(dtype).requires_grad_(learned)
    state['W'] = _normal(gen, (g, K, N), dtype, 1 / math.sqrt(K)).requires_grad_(learned)
    if learned:
        state['dy'] = _normal(gen, (n, N), dtype)
    keys = _keys(case, g, gen)
    if k == 'layer':
        keys[torch.rand(n, generator=gen, device='cuda') < case['outside']] = -1
        state['element'] = keys.to(torch.int32)
        state['offset'] = _normal(gen, (g, N), dtype).requires_grad_(True)
        state['sizes'] = torch.bincount(keys[keys >= 0], minlength=g).tolist()
        return state
    rows = n - int(n * case['behind'])                   # the last rows of the buffer belong to no group
    sizes = torch.bincount(keys[:rows], minlength=g)
    state['sizes'] = sizes.tolist()
    state['start'] = torch.cat((sizes.new_zeros(1), torch.cumsum(sizes, 0))).to(torch.int32)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return _own_run(state) if own else _plain_run(state)


def _own_run(s):
    import qml_lightning_b200  # noqa: F401  (registers the operators)
    ops = torch.ops.qml_lightning_b200
    k = s['kind']
    if k == 'group':
        order, start = ops.group_by_key(s['index'], s['keys'])
        return {'order': order, 'start': start}
    if k == 'embedding':
        return {'out': ops.embedding(s['index'], s['table'], s['scale'])}
    if k == 'embedding_step':
        out = ops.embedding(s['index'], s['table'], s['scale'])
        dtable, = torch.autograd.grad(out, (s['table'],), s['dout'])
        return {'out': out.detach(), 'dtable': dtable}
    if k == 'product':
        return {'y': ops.grouped_matmul(s['x'], s['W'], s['start'])}
    if k == 'product_step':
        y = ops.grouped_matmul(s['x'], s['W'], s['start'])
        dx, dW = torch.autograd.grad(y, (s['x'], s['W']), s['dy'])
        return {'y': y.detach(), 'dx': dx, 'dW': dW}
    order, start = ops.group_by_key(s['element'], s['groups'])
    rows = ops.embedding(order, s['x'], 1.0)
    y = ops.grouped_matmul(rows, s['W'], start) + ops.embedding(s['element'][order], s['offset'], 1.0)
    dx, dW, doffset = torch.autograd.grad(y, (s['x'], s['W'], s['offset']), s['dy'])
    return {'order': order, 'y': y.detach(), 'dx': dx, 'dW': dW, 'doffset': doffset}


def _plain_group(index, keys):
    key = torch.where((index >= 0) & (index < keys), index, keys).long()
    order = torch.argsort(key, stable=True)
    count = torch.bincount(key, minlength=keys + 1)[:keys]
    return order.to(torch.int32), torch.cat((count.new_zeros(1), torch.cumsum(count, 0))).to(torch.int32)


def _plain_lookup(index, table, scale):
    inside = ((index >= 0) & (index < table.shape[0])).unsqueeze(1)
    row = table[index.clamp(0, table.shape[0] - 1)].float() * scale
    return torch.where(inside, row, torch.zeros_like(row)).to(table.dtype)


def _plain_lookup_grad(index, dout, keys, scale):
    inside = (index >= 0) & (index < keys)
    rows = torch.where(inside.unsqueeze(1), dout, torch.zeros_like(dout)).double()      # long sums
    total = torch.zeros((keys, dout.shape[1]), dtype=torch.float64, device=dout.device)
    return (total.index_add_(0, index.clamp(0, keys - 1), rows) * scale).to(dout.dtype)


def _plain_product(x, W, sizes, transpose):
    """Rows of every group times its matrix; there is no elementary operation over ragged groups, so they take turns."""
    B = W.transpose(1, 2) if transpose else W
    y = torch.zeros((x.shape[0], B.shape[2]), dtype=x.dtype, device=x.device)
    at = 0
    for g, size in enumerate(sizes):
        if size:
            y[at:at + size] = (x[at:at + size].float() @ B[g].float()).to(x.dtype)
        at += size
    return y


def _plain_product_wgrad(x, dy, sizes):
    """Long sums of non-negative descriptors: blocks of rows in 32 bits, the blocks added in 64."""
    dW = torch.zeros((len(sizes), x.shape[1], dy.shape[1]), dtype=x.dtype, device=x.device)
    at = 0
    for g, size in enumerate(sizes):
        if size:
            a, b = x[at:at + size].float(), dy[at:at + size].float()
            blocks = size // 4096
            total = (a[blocks * 4096:].T @ b[blocks * 4096:]).double()
            if blocks:
                a, b = (t[:blocks * 4096].view(blocks, 4096, -1) for t in (a, b))
                total = total + torch.bmm(a.transpose(1, 2), b).double().sum(0)
            dW[g] = total.to(x.dtype)
        at += size
    return dW


def _plain_run(s):
    with torch.no_grad():
        k = s['kind']
        if k == 'group':
            order, start = _plain_group(s['index'], s['keys'])
            return {'order': order, 'start': start}
        if k in ('embedding', 'embedding_step'):
            out = {'out': _plain_lookup(s['index'], s['table'], s['scale'])}
            if k == 'embedding_step':
                out['dtable'] = _plain_lookup_grad(s['index'], s['dout'], s['keys'], s['scale'])
            return out
        if k == 'product':
            return {'y': _plain_product(s['x'], s['W'], s['sizes'], False)}
        if k == 'product_step':
            return {'y': _plain_product(s['x'], s['W'], s['sizes'], False), 'dx': _plain_product(s['dy'], s['W'], s['sizes'], True),
                    'dW': _plain_product_wgrad(s['x'], s['dy'], s['sizes'])}
        order, _ = _plain_group(s['element'], s['groups'])
        rows = s['x'][order]
        element = s['element'][order]
        y = _plain_product(rows, s['W'], s['sizes'], False)
        y = (y.float() + _plain_lookup(element, s['offset'], 1.0).float()).to(y.dtype)
        dx = torch.zeros_like(s['x'])
        dx[order] = _plain_product(s['dy'], s['W'], s['sizes'], True)
        return {'order': order, 'y': y, 'dx': dx, 'dW': _plain_product_wgrad(rows, s['dy'], s['sizes']),
                'doffset': _plain_lookup_grad(element, s['dy'], s['groups'], 1.0)}


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------
def exact(case, seed):
    k = case['kind']
    if k == 'group':            # whole numbers only
        return None
    s = {name: v.detach() if isinstance(v, torch.Tensor) else v for name, v in prepare(case, seed).items()}
    if k in ('embedding', 'embedding_step'):
        # a zero row behind the table stands for every index outside it
        keys = case['keys']
        row = s['index'].long()
        row = torch.where((row < 0) | (row >= keys), torch.full_like(row, keys), row)
        table = torch.cat((s['table'].double(), torch.zeros((1, case['width']), dtype=torch.float64, device='cuda')))
        out = {'out': torch.index_select(table * s['scale'], 0, row)}
        if k == 'embedding_step':
            total = torch.zeros((keys + 1, case['width']), dtype=torch.float64, device='cuda')
            total.scatter_add_(0, row.unsqueeze(1).expand(-1, case['width']), s['dout'].double())
            out['dtable'] = total[:keys] * s['scale']
        return out
    n, g, N = case['n'], case['groups'], case['N']
    if k == 'layer':
        member = s['element'].long()
        order = torch.sort(torch.where(member < 0, torch.full_like(member, g), member), stable=True)[1]
        member = member[order]
    else:
        order = None
        edge = s['start'].long()
        member = torch.searchsorted(edge[1:], torch.arange(n, device='cuda'), right=True)
        member[member >= g] = -1
    x = s['x'].double() if order is None else s['x'].double()[order]
    y = torch.zeros((n, N), dtype=torch.float64, device='cuda')
    dx, dW = torch.zeros_like(x), torch.zeros((g, case['K'], N), dtype=torch.float64, device='cuda')
    doffset = torch.zeros((g, N), dtype=torch.float64, device='cuda')
    for e in range(g):
        rows = torch.nonzero(member == e)[:, 0]
        W = s['W'][e].double()
        y[rows] = torch.einsum('rk,kn->rn', x[rows], W)
        if k != 'product':
            dy = s['dy'][rows].double()
            dx[rows] = torch.einsum('rn,kn->rk', dy, W)
            dW[e] = torch.einsum('rk,rn->kn', x[rows], dy)
            if k == 'layer':
                y[rows] += s['offset'][e].double()
                doffset[e] = dy.sum(0)
    if k == 'product':
        return {'y': y}
    if k == 'product_step':
        return {'y': y, 'dx': dx, 'dW': dW}
    back = torch.empty_like(dx)
    back[order] = dx
    return {'order': None, 'y': y, 'dx': back, 'dW': dW, 'doffset': doffset}
