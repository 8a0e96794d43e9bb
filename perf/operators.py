"""A GCN layer's dense part with bias, activation and residual, and the optimiser step behind it, as cases that can be timed one by one.

Kinds of work:

  linear   y = act(x w + b) + r, forward alone (inference) or with the gradients of x, w, b and r (training); x, w, b, r in fp32, bf16 or fp16
  adamw    one AdamW step over all tensors of a model: its layers' weights and biases and, where the graph has no features, a learned table of
           node embeddings; states in 32 or in 8 bits, gradients clipped by their global norm where `max_norm` is not 0

Where `own` is false the operators run in their plain form, elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

PACKAGE = os.path.abspath('dist-gnn_b200')

# node counts and widths of coo_graph.synthetic.CONFIGS
PLUMBING = dict(feat=128, hidden=64, classes=10)
SPARSE_NODES, SPARSE = 2_449_029, dict(feat=100, hidden=256, classes=47)

BLOCK = 256                     # elements that share a scale where states are held in 8 bits
LARGEST = 448.0                 # of e4m3
ITEM = dict(f32=4, bf16=2, f16=2)
TYPE = dict(f32=torch.float32, bf16=torch.bfloat16, f16=torch.float16)
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=1e-2)


def _linear(rows, inner, cols, dtype, act, bias=True, residual=False, train=False, out_in=False):
    return dict(kind='linear', rows=rows, inner=inner, cols=cols, dtype=dtype, act=act, bias=bias, residual=residual, train=train, out_in=out_in)


def _adamw(feat, hidden, classes, layers, dtype, bits, max_norm, table_rows=0, table_width=0):
    return dict(kind='adamw', feat=feat, hidden=hidden, classes=classes, layers=layers, dtype=dtype, bits=bits, max_norm=max_norm,
                table_rows=table_rows, table_width=table_width)


def listed():
    return [
        # serving: the answer for one node, the smallest call there is
        dict(name='linear_one_f32', **_linear(1, 256, 256, 'f32', 'relu')),
        # serving: a few nodes through a wide layer whose weight lies as [out x in]
        dict(name='linear_few_bf16', **_linear(16, 1024, 1024, 'bf16', 'gelu', residual=True, out_in=True)),
        # evaluation of an eighth of the headline graph: the first layer, 100 features
        dict(name='linear_eval_f32', **_linear(306_128, 100, 256, 'f32', 'relu')),
        # a hidden layer of the default model on a ragged mid-sized graph
        dict(name='linear_train_f32', **_linear(150_001, 256, 256, 'f32', 'gelu', residual=True, train=True)),
        # wide odd features (602) and an odd class count (41), as the dense graph has them
        dict(name='linear_odd_f16', **_linear(232_965, 602, 41, 'f16', 'silu', train=True)),
        # a wide encoder in front of the graph: bound by the tensor cores
        dict(name='linear_wide_bf16', **_linear(65_536, 1024, 1024, 'bf16', 'silu', residual=True, train=True)),
        # a hidden residual layer over all nodes of the headline graph
        dict(name='linear_sparse_bf16', **_linear(SPARSE_NODES, 256, 256, 'bf16', 'gelu', residual=True, train=True)),
        # the smallest model's step: launches and host work count
        dict(name='adamw_plumbing', **_adamw(layers=2, dtype='f32', bits=32, max_norm=0.0, **PLUMBING)),
        # a deep residual model: 128 weights and biases
        dict(name='adamw_deep_8bit', **_adamw(layers=64, dtype='bf16', bits=8, max_norm=1.0, **SPARSE)),
        # the default model behind a table of 64 learned features a node
        dict(name='adamw_table', **_adamw(layers=3, dtype='f32', bits=32, max_norm=1.0, table_rows=SPARSE_NODES, table_width=64, **SPARSE)),
        # a table of 256 a node: what states in 8 bits are for
        dict(name='adamw_table_8bit', **_adamw(layers=3, dtype='bf16', bits=8, max_norm=0.0, table_rows=SPARSE_NODES, table_width=256, **SPARSE)),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.6:
        inner, cols = _log(rng, 1, 1024), _log(rng, 1, 1024)
        if rng.random() < 0.5:              # half of the widths are whole 16-byte pieces, as models have them
            inner, cols = inner + (-inner) % 8, cols + (-cols) % 8
        most = min(SPARSE_NODES, SPARSE_NODES * 256 * 256 // (inner * cols), SPARSE_NODES * 512 // (inner + cols))
        rows = _log(rng, 1, 512) if rng.random() < 0.3 else _log(rng, 512, most)
        train = rng.random() < 0.6
        # the gradient of ReLU is a step at zero: which side a pre-activation of 1e-7 is on is for the rounding of its sum to say, so that two right
        # answers differ there by a whole term.  The forward pass has no such places.
        act = rng.choice(['none', 'gelu', 'silu'] if train else ['none', 'relu', 'gelu', 'silu'])
        return _linear(rows, inner, cols, rng.choice(['f32', 'bf16', 'f16']), act, rng.random() < 0.8, rng.random() < 0.5, train, rng.random() < 0.3)
    layers, hidden = _log(rng, 1, 128), _log(rng, 8, 1024)
    hidden = min(hidden, int(math.sqrt(64e6 / layers)))
    width = _log(rng, 4, 256) if rng.random() < 0.5 else 0
    rows = _log(rng, 1_000, SPARSE_NODES) if width else 0
    return _adamw(_log(rng, 1, 602), hidden, rng.randint(2, 47), layers, rng.choice(['f32', 'bf16', 'f16']) if rows * width < 2e8 else 'bf16',
                  rng.choice([32, 8]) if rows * width < 2e8 else 8, rng.choice([0.0, 1.0, 100.0]), rows, width)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def _shapes(c):
    """Shapes of the model's tensors: the table, then every layer's weight [in x out] and bias."""
    widths = [c['table_width'] or c['feat']] + [c['hidden']] * (c['layers'] - 1) + [c['classes']]
    shapes = [(c['table_rows'], c['table_width'])] if c['table_rows'] else []
    for a, b in zip(widths, widths[1:]):
        shapes += [(a, b), (b,)]
    return shapes


def _whole(n):
    return n + (-n) % BLOCK


def prepare(case, seed):
    c = dict(case)
    return _prepare_linear(c, seed) if c['kind'] == 'linear' else _prepare_adamw(c, seed)


def _prepare_linear(c, seed):
    """Activations N(0, 1), weights N(0, 1 / inner) as an initialiser or a trained layer has them, gradients N(0, 1) / rows as a mean loss gives them."""
    gen, dtype = _gen(seed), TYPE[c['dtype']]
    rows, inner, cols = c['rows'], c['inner'], c['cols']

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, device='cuda', generator=gen) * scale).to(dtype)

    s = dict(case=c, x=randn(rows, inner))
    s['w'] = randn(cols, inner, scale=inner ** -0.5).t() if c['out_in'] else randn(inner, cols, scale=inner ** -0.5)
    s['b'] = randn(cols, scale=0.5) if c['bias'] else None
    s['r'] = randn(rows, cols) if c['residual'] else None
    # 16-bit training scales its loss so that gradients stay within the type
    s['dy'] = randn(rows, cols, scale=1.0 if dtype != torch.float32 else 1.0 / rows) if c['train'] else None
    if c['train']:
        for name in ('x', 'w', 'b', 'r'):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _prepare_adamw(c, seed):
    """A model in the middle of its training.  Every tensor starts on a block of its own inside one buffer a kind, so that the plain form can take
    them all at once; gradients of tensors differ by orders of magnitude, and a tenth of the table's rows have never had one."""
    gen, dtype = _gen(seed), TYPE[c['dtype']]
    shapes = _shapes(c)
    counts = [math.prod(s) for s in shapes]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + _whole(n))
    total = starts[-1]
    p, g = torch.zeros(total, device='cuda', dtype=dtype), torch.zeros(total, device='cuda', dtype=dtype)
    small = c['bits'] == 8
    kept = torch.float8_e4m3fn if small else torch.float32
    m, v = torch.zeros(total, device='cuda', dtype=kept), torch.zeros(total, device='cuda', dtype=kept)      # v: its root in 8 bits
    ms, vs = (torch.zeros(total // BLOCK, device='cuda'), torch.zeros(total // BLOCK, device='cuda')) if small else (None, None)
    for i, (shape, n, at) in enumerate(zip(shapes, counts, starts)):
        size = 10.0 ** -(2 + (i * 7 % 5) * 0.5)
        live = None
        if i == 0 and c['table_rows']:
            live = (torch.rand(shape[0], 1, device='cuda', generator=gen) > 0.1).float()

        def draws(kind):
            x = (torch.randn if kind == 'n' else torch.rand)(shape, device='cuda', generator=gen)
            return (x if live is None else x.mul_(live)).view(-1)

        p[at:at + n] = (torch.randn(shape, device='cuda', generator=gen) * 0.1).view(-1).to(dtype)
        g[at:at + n] = draws('n').mul_(size).to(dtype)
        mean, root = draws('n').mul_(0.3 * size), draws('u').mul_(0.9 * size)
        if not small:
            m[at:at + n], v[at:at + n] = mean, root.square_()
            continue
        end = at + _whole(n)
        for x, codes, scales in ((mean, m, ms), (root, v, vs)):
            wide = torch.zeros(end - at, device='cuda')
            wide[:n] = x
            wide = wide.view(-1, BLOCK)
            scale = wide.abs().amax(1) / LARGEST
            scales[at // BLOCK:end // BLOCK] = scale
            codes[at:end] = (wide / scale.clamp(min=1e-30)[:, None]).view(-1).to(kept)
    s = dict(case=c, p=p, g=g, m=m, v=v, ms=ms, vs=vs, step=100 + seed % 900, seed=seed % 10007)
    if own:
        s['optimizer'] = _optimizer(s, shapes, counts, starts)
    return s


def _optimizer(s, shapes, counts, starts):
    """The framework's optimiser on views of these buffers."""
    spmm_cpp = _framework()
    c = s['case']

    def views(t, unit=1):
        return [None if t is None else t[a // unit:(a + n + unit - 1) // unit] for a, n in zip(starts, counts)]

    params = []
    for w, g, shape in zip(views(s['p']), views(s['g']), shapes):
        params.append(torch.nn.Parameter(w.view(shape)))
        params[-1].grad = g.view(shape)
    opt = spmm_cpp.AdamW(params, lr=HYPER['lr'], betas=(HYPER['beta1'], HYPER['beta2']), eps=HYPER['eps'], weight_decay=HYPER['weight_decay'],
                         state_bits=c['bits'], max_norm=c['max_norm'] or None, seed=s['seed'])
    for q, m, v, ms, vs, shape in zip(params, views(s['m']), views(s['v']), views(s['ms'], BLOCK), views(s['vs'], BLOCK), shapes):
        opt.state[q] = dict(step=torch.tensor(s['step'], dtype=torch.int64, device='cuda'), exp_avg=m.view(shape), exp_avg_sq=v.view(shape))
        if c['bits'] == 8:
            opt.state[q] = dict(step=opt.state[q]['step'], exp_avg=m.view(shape), exp_avg_scale=ms, root=v.view(shape), root_scale=vs)
    return opt


def _framework():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import spmm_cpp
    return spmm_cpp


# ---- one pass ------------------------------------------------------------------------------------------------------------
def run(s):
    c = s['case']
    if c['kind'] == 'linear':
        return _linear_own(s) if own else _linear_plain(s)
    if own:
        s['optimizer'].step()
        norm = s['optimizer'].grad_norm
    else:
        norm = _adamw_plain(s)
    out = dict(p=s['p'], m=s['m'], v=s['v'])
    if c['bits'] == 8:
        out.update(m_scale=s['ms'], v_scale=s['vs'])
    if c['max_norm']:
        out['norm'] = norm
    return out


def _linear_own(s):
    c = s['case']
    linear = _framework().linear
    act = None if c['act'] == 'none' else c['act']
    if not c['train']:
        with torch.no_grad():
            return dict(y=linear(s['x'], s['w'], s['b'], residual=s['r'], activation=act))
    y = linear(s['x'], s['w'], s['b'], residual=s['r'], activation=act)
    names = [n for n in ('x', 'w', 'b', 'r') if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s['dy'])
    return dict({'d' + n: g for n, g in zip(names, grads)}, y=y)


def _linear_plain(s):
    c = s['case']
    with torch.no_grad():
        dtype = s['x'].dtype
        x, w = s['x'].float(), s['w'].float()
        z = x @ w
        if s['b'] is not None:
            z = z + s['b'].float()
        slope = None
        if c['act'] == 'relu':
            y, slope = z.clamp(min=0), (z > 0).float() if c['train'] else None
        elif c['act'] == 'gelu':
            half = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
            y, slope = z * half, half + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)) if c['train'] else None
        elif c['act'] == 'silu':
            gate = 1 / (1 + torch.exp(-z))
            y, slope = z * gate, gate * (1 + z * (1 - gate)) if c['train'] else None
        else:
            y = z
        if s['r'] is not None:
            y = y + s['r'].float()
        out = dict(y=y.to(dtype))
        if not c['train']:
            return out
        dz = s['dy'].float()
        if slope is not None:
            dz = dz * slope
        out['dx'] = (dz @ w.t()).to(dtype)
        # sums over up to millions of rows: in 64 bits above pieces of 4,096 rows
        piece, rows = 4096, x.size(0)
        whole = rows // piece * piece
        dw, db = x[whole:].t() @ dz[whole:], dz[whole:].sum(0, dtype=torch.float64)
        if whole:
            dw = dw.double() + torch.bmm(x[:whole].view(-1, piece, x.size(1)).transpose(1, 2), dz[:whole].view(-1, piece, dz.size(1))).sum(0, dtype=torch.float64)
            db = db + dz[:whole].sum(0, dtype=torch.float64)
        out['dw'] = dw.to(dtype)
        if s['b'] is not None:
            out['db'] = db.to(dtype)
        if s['r'] is not None:
            out['dr'] = s['dy']
        return out


# The rounding of 8-bit states is random, with numbers that are a function of the optimiser's seed, the step and the element's place: two rounds of
# xor-shift and product, in 32 bits that wrap around, for a pair of neighbours, 16 bits for each.
_PLACE, _ROUND1, _ROUND2, _STEP = 0x9E3779B1, 0x6A09E667, 0xBB67AE85, 0x3C6EF373


def _int32(v):
    v &= 0xFFFFFFFF
    return v - (1 << 32) if v >> 31 else v


def _mix(h):
    """Of an int32 tensor."""
    h = (h ^ ((h >> 16) & 0xFFFF)) * _int32(_ROUND1)
    h = (h ^ ((h >> 15) & 0x1FFFF)) * _int32(_ROUND2)
    return h ^ ((h >> 16) & 0xFFFF)


def _noise(n, seed, step):
    """A 16-bit number an element."""
    key = _mix(torch.tensor([_int32(seed + step * _STEP)], dtype=torch.int32, device='cuda'))
    h = _mix(torch.arange(n // 2, dtype=torch.int32, device='cuda') * _int32(_PLACE) + key)
    return torch.stack((h & 0xFFFF, (h >> 16) & 0xFFFF), dim=1).view(-1)


def _to_8_bits(x, noise, keep_positive):
    """(codes, scales): a block's largest magnitude is 448; between two neighbours of e4m3 the noise decides in proportion."""
    blocks = x.view(-1, BLOCK)
    most = blocks.abs().amax(1)
    scale = most * (1 / LARGEST)
    fine = ~(most < 1e-30)                            # a NaN stays one
    factor = torch.where(fine, LARGEST * (1 / most), torch.zeros_like(most))
    q = (blocks.abs() * factor[:, None]).view(-1).clamp(max=LARGEST)
    low = 2.0 ** -6                                   # below it e4m3 steps by 2^-9, as it does right above
    tiny = q < low
    bits = (torch.where(tiny, q + low, q).view(torch.int32) + (noise << 4)) & -0x100000
    y = bits.view(torch.float32)
    y = torch.where(tiny, y - low, y)
    if keep_positive:
        y = torch.where((y == 0) & (q > 0), torch.full_like(y, 2.0 ** -9), y)
    return torch.where(x < 0, -y, y).to(torch.float8_e4m3fn), torch.where(fine, scale, torch.zeros_like(scale))


def _adamw_plain(s):
    c = s['case']
    s['step'] += 1
    t, h, norm = s['step'], HYPER, None
    g = s['g'].float()
    if c['max_norm']:
        norm = g.double().square().sum().sqrt()       # a long sum
        g = g * (c['max_norm'] / (norm + 1e-6)).clamp(max=1.0).float()
        norm = norm.float()
    small = c['bits'] == 8
    if small:
        m = (s['m'].float().view(-1, BLOCK) * s['ms'][:, None]).view(-1)
        r = (s['v'].float().view(-1, BLOCK) * s['vs'][:, None]).view(-1)
        v = r * r
    else:
        m, v = s['m'], s['v']
    m = m * h['beta1'] + g * (1 - h['beta1'])
    v = v * h['beta2'] + g * g * (1 - h['beta2'])
    root = v.sqrt()
    p = s['p'].float() * (1 - h['lr'] * h['weight_decay'])
    p = p - m / (root * (1 / math.sqrt(1 - h['beta2'] ** t)) + h['eps']) * (h['lr'] / (1 - h['beta1'] ** t))
    s['p'].copy_(p)
    if small:
        noise = _noise(m.numel(), s['seed'], t)
        for x, codes, scales, positive in ((m, s['m'], s['ms'], False), (root, s['v'], s['vs'], True)):
            q, scale = _to_8_bits(x, noise, positive)
            codes.copy_(q)
            scales.copy_(scale)
    else:
        s['m'].copy_(m)
        s['v'].copy_(v)
    return norm


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    c, e = case, ITEM[case['dtype']]
    if c['kind'] == 'linear':
        M, K, N = c['rows'], c['inner'], c['cols']
        count = M * K + K * N + M * N + (N if c['bias'] else 0) + (M * N if c['residual'] else 0)
        if c['train']:                                # dy in; dx, dw, db out (the residual's gradient is dy itself)
            count += M * N + M * K + K * N + (N if c['bias'] else 0)
        return dict(bytes=e * count, flops=(6 if c['train'] else 2) * M * N * K)
    n = sum(math.prod(s) for s in _shapes(c))
    state = 4 if c['bits'] == 8 else 16               # two states in and out
    return dict(bytes=n * (3 * e + state) + (n // BLOCK * 16 if c['bits'] == 8 else 0), flops=20 * n)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False                             # inputs alone: no optimiser
    try:
        s = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return _exact_linear(s) if case['kind'] == 'linear' else _exact_adamw(s)


def _exact_linear(s):
    act = s['case']['act']
    x, w = s['x'].double(), s['w'].double()
    z = torch.matmul(x, w) if s['b'] is None else torch.addmm(s['b'].double(), x, w)
    if act == 'relu':
        y = torch.maximum(z, torch.zeros_like(z))
    elif act == 'gelu':
        y = z * torch.special.ndtr(z)
    elif act == 'silu':
        y = z * torch.sigmoid(z)
    else:
        y = z.clone()
    if s['r'] is not None:
        y += s['r'].double()
    out = dict(y=y)
    if s['dy'] is None:
        return out
    dz = s['dy'].double()
    if act == 'gelu':
        dz = dz * (torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    elif act == 'silu':
        gate = torch.sigmoid(z)
        dz = dz * (gate + z * gate * torch.sigmoid(-z))
    elif act == 'relu':
        dz = dz * (z > 0)
    out['dx'], out['dw'] = torch.matmul(dz, w.T), torch.matmul(x.T, dz)
    if s['b'] is not None:
        out['db'] = dz.sum(dim=0)
    if s['r'] is not None:
        out['dr'] = s['dy'].double()
    return out


def _exact_adamw(s):
    c, t = s['case'], s['step'] + 1
    b1, b2 = HYPER['beta1'], HYPER['beta2']
    grad, out = s['g'].double(), {}
    if c['max_norm']:
        norm = torch.linalg.vector_norm(grad)
        out['norm'] = norm
        if float(norm) + 1e-6 > c['max_norm']:
            grad *= c['max_norm'] / (norm + 1e-6)
    first, second = s['m'].double(), s['v'].double()
    if c['bits'] == 8:
        first, second = first * s['ms'].double().repeat_interleave(BLOCK), (second * s['vs'].double().repeat_interleave(BLOCK)) ** 2
    first = torch.lerp(first, grad, 1 - b1)
    second = second.mul_(b2).addcmul_(grad, grad, value=1 - b2)
    update = (first / (1 - b1 ** t)) / ((second / (1 - b2 ** t)).sqrt() + HYPER['eps'])
    out['p'] = (s['p'].double() * (1 - HYPER['lr'] * HYPER['weight_decay'])).sub_(update, alpha=HYPER['lr'])
    del update
    if c['bits'] == 32:
        return dict(out, m=first, v=second)
    noise = _noise(first.numel(), s['seed'], t).double() / 65536
    for name, value in (('m', first), ('v', second.sqrt_())):
        size = value.abs()
        top = size.view(-1, BLOCK).max(dim=1).values
        q = size / top.clamp(min=1e-30).repeat_interleave(BLOCK) * LARGEST
        grid = torch.exp2(torch.frexp(q).exponent.clamp(min=-5).double() - 4)           # the distance of e4m3's neighbours
        q = torch.floor(q / grid + noise).mul_(grid)
        if name == 'v':
            q = torch.where((q == 0) & (size > 0), torch.full_like(q, 2.0 ** -9), q)
        out[name], out[name + '_scale'] = torch.copysign(q, value), top / LARGEST
    return out
