"""Cases and plain forms of three operators of a training step with a large label set: layer norm, the softmax cross entropy
of a linear classifier, and the orthogonalised update of weight matrices.

`own` false: elementary torch operations in 32 bits (64 in long sums), rounded once to the inputs' type.  `own` true: the framework's calls
(`detector.layers.layer_norm`, `core.linear_cross_entropy`, `core.orthogonalize`).  `exact` computes the same in 64 bits."""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NS_EPS = 1e-7
LN_EPS = 1e-5
IGNORE = -100
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}
BYTES = {'fp32': 4, 'bf16': 2}


def _detector_matrices():
    """every weight matrix [Cout, Cin * taps] of the 50-layer backbone (16-channel stem), its four-level neck and the two shared
    layers of a bbox head (64 x 3 x 7 x 7 roi features -> 1024 -> 1024)"""
    out = [(16, 3 * 343)]
    cin = 16
    for stage, blocks in enumerate((3, 4, 6, 3)):
        planes = 16 * 2 ** stage
        for b in range(blocks):
            out += [(planes, cin), (planes, planes * 27), (planes * 4, planes)]
            if b == 0:
                out.append((planes * 4, cin))
            cin = planes * 4
    for c in (64, 128, 256, 512):
        out += [(64, c), (64, 64 * 27)]
    return out + [(1024, 64 * 3 * 7 * 7), (1024, 1024)]


def _shapes(case):
    if case['shapes'] == 'detector':
        return _detector_matrices()
    return [tuple(int(v) for v in s.split('x')) for s in case['shapes'].split(',')]


def listed():
    return [
        # one row of a head's activations, inference: launch latency
        {'name': 'norm_row', 'op': 'norm', 'rows': 1, 'cols': 1024, 'dtype': 'fp32', 'train': False},
        # the 512 sampled rois x 1024 features of a bbox head, forward + backward
        {'name': 'norm_rois', 'op': 'norm', 'rows': 512, 'cols': 1024, 'dtype': 'fp32', 'train': True},
        # odd row and column counts: nothing is a multiple of a vector load
        {'name': 'norm_ragged', 'op': 'norm', 'rows': 10007, 'cols': 1531, 'dtype': 'fp32', 'train': True},
        # the voxels of the finest pyramid map (40 x 128 x 128, 64 channels, channels last) in bf16 storage
        {'name': 'norm_voxels', 'op': 'norm', 'rows': 655360, 'cols': 64, 'dtype': 'bf16', 'train': True},
        # one row against a large label set, loss only: reads the classifier's weights once
        {'name': 'ce_row', 'op': 'ce', 'rows': 1, 'hidden': 1024, 'classes': 32768, 'dtype': 'bf16', 'bias': False, 'ignored': 0.0, 'train': False},
        # 512 sampled rois x 1024 features of a bbox head with about a thousand classes
        {'name': 'ce_rois', 'op': 'ce', 'rows': 512, 'hidden': 1024, 'classes': 1204, 'dtype': 'fp32', 'bias': True, 'ignored': 0.25, 'train': True},
        # odd sizes in all three directions, a third of the rows ignored
        {'name': 'ce_ragged', 'op': 'ce', 'rows': 3001, 'hidden': 515, 'classes': 20011, 'dtype': 'fp32', 'bias': True, 'ignored': 0.33, 'train': True},
        # a large batch over a large label set
        {'name': 'ce_large', 'op': 'ce', 'rows': 8192, 'hidden': 2048, 'classes': 131072, 'dtype': 'bf16', 'bias': False, 'ignored': 0.05, 'train': True},
        # one 3x3x3 convolution of the neck / RPN head: latency
        {'name': 'ortho_conv', 'op': 'ortho', 'shapes': '64x1728', 'dtype': 'fp32'},
        # odd sizes, tall and wide
        {'name': 'ortho_ragged', 'op': 'ortho', 'shapes': '777x2311,1301x333', 'dtype': 'fp32'},
        # all matrices of a detector in one update
        {'name': 'ortho_detector', 'op': 'ortho', 'shapes': 'detector', 'dtype': 'fp32'},
        # a large square matrix
        {'name': 'ortho_square', 'op': 'ortho', 'shapes': '4096x4096', 'dtype': 'bf16'},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('norm', 'ce', 'ortho'))
    dtype = rng.choice(('fp32', 'bf16'))
    if op == 'norm':
        cols = _log(rng, 16, 8192)
        rows = _log(rng, 1, min(655360, 41943040 // cols))
        return {'op': op, 'rows': rows, 'cols': cols, 'dtype': dtype, 'train': rng.random() < 0.75}
    if op == 'ce':
        hidden = _log(rng, 32, 2048)
        classes = _log(rng, 100, 131072)
        rows = _log(rng, 1, max(1, min(8192, (1 << 36) // classes // hidden)))
        return {'op': op, 'rows': rows, 'hidden': hidden, 'classes': classes, 'dtype': dtype, 'bias': rng.random() < 0.5,
                'ignored': rng.choice((0.0, 0.1, 0.5)), 'train': rng.random() < 0.75}
    shapes = ','.join('%dx%d' % (_log(rng, 16, 1536), _log(rng, 16, 6144)) for _ in range(rng.randint(1, 4)))
    return {'op': op, 'shapes': shapes, 'dtype': dtype}


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = DTYPES[case['dtype']]

    def randn(*shape):
        return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32)

    if case['op'] == 'norm':
        r, c = case['rows'], case['cols']
        s = {'x': (randn(r, c) * (0.5 + 2 * torch.rand((r, 1), generator=g, device='cuda')) + 0.5 * randn(r, 1)).to(dt),
             'w': (1 + 0.1 * randn(c)).to(dt), 'b': (0.1 * randn(c)).to(dt), 'dy': randn(r, c).to(dt) if case['train'] else None}
        leaves = ('x', 'w', 'b')
    elif case['op'] == 'ce':
        r, k, v = case['rows'], case['hidden'], case['classes']
        s = {'x': randn(r, k).to(dt), 'w': (randn(v, k) * (2.0 / math.sqrt(k))).to(dt), 'b': (0.5 * randn(v)).to(dt) if case['bias'] else None,
             'label': torch.randint(0, v, (r,), generator=g, device='cuda'),
             'row_weight': 0.25 + torch.rand((r,), generator=g, device='cuda')}
        dead = torch.rand((r,), generator=g, device='cuda') < case['ignored']
        dead[0] = False
        s['label'] = torch.where(dead, torch.full_like(s['label'], IGNORE), s['label'])
        leaves = ('x', 'w', 'b')
    else:
        # gradients of trained layers: a decaying spectrum under noise
        s = {'mats': []}
        for m, n in _shapes(case):
            k = max(1, min(m, n) // 8)
            s['mats'].append(((randn(m, k) @ randn(k, n)) * (1e-3 / math.sqrt(k)) + 5e-4 * randn(m, n)).to(dt))
        leaves = ()
    if case.get('train'):
        for name in leaves:
            if s[name] is not None:
                s[name].requires_grad_(True)
    s['case'] = case
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x, w, b = s['x'].float(), s['w'].float(), s['b'].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + LN_EPS)
    h = d * rstd
    out = {'y': (h * w + b).to(s['x'].dtype)}
    if s['dy'] is not None:
        dy = s['dy'].float()
        gh = dy * w
        out['dx'] = ((gh - gh.mean(1, keepdim=True) - h * (gh * h).mean(1, keepdim=True)) * rstd).to(s['x'].dtype)
        out['dw'] = (dy * h).sum(0).to(s['w'].dtype)
        out['db'] = dy.sum(0).to(s['b'].dtype)
    return out


def _plain_ce(s):
    x, w = s['x'].float(), s['w'].float()
    live = s['label'] != IGNORE
    label = torch.where(live, s['label'], torch.zeros_like(s['label'])).unsqueeze(1)
    rw = torch.where(live, s['row_weight'], torch.zeros_like(s['row_weight']))
    avg = (rw > 0).sum().clamp(min=1).float()
    z = x @ w.t()
    if s['b'] is not None:
        z = z + s['b'].float()
    zl = z.gather(1, label)
    top = z.amax(1, keepdim=True)
    p = z.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    loss = (((total.log() + top - zl).squeeze(1) * rw).double().sum() / avg).float().reshape(1)
    if not s['case']['train']:
        return {'loss': loss}
    p = p.mul_(1 / total)
    p = p.scatter_add_(1, label, torch.full_like(total, -1.0)).mul_((rw / avg).unsqueeze(1))
    out = {'loss': loss, 'dx': (p @ w).to(s['x'].dtype), 'dw': (p.t() @ x).to(s['w'].dtype)}
    if s['b'] is not None:
        out['db'] = p.sum(0).to(s['b'].dtype)
    return out


def _plain_ortho(s):
    a, b, c = COEFFICIENTS
    out = []
    for g in s['mats']:
        x = g.float()
        tall = x.size(0) > x.size(1)
        x = x.t() if tall else x
        x = x / ((x * x).sum().sqrt() + NS_EPS)
        for _ in range(STEPS):
            gram = x @ x.t()
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        out.append((x.t() if tall else x).to(g.dtype))
    return out


def run(state):
    op = state['case']['op']
    if not own:
        with torch.no_grad():
            return {'norm': _plain_norm, 'ce': _plain_ce, 'ortho': _plain_ortho}[op](state)
    from mr3d_amd.core import linear_cross_entropy, orthogonalize
    from mr3d_amd.detector.layers import layer_norm
    if op == 'ortho':
        return orthogonalize(state['mats'], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    train = state['case']['train']
    x, w, b = state['x'], state['w'], state['b']
    leaves = [t for t in (x, w, b) if t is not None]
    if op == 'norm':
        y = layer_norm(x, w, b, eps=LN_EPS)
        out = {'y': y.detach()}
        grads = torch.autograd.grad(y, leaves, state['dy']) if train else ()
    else:
        loss = linear_cross_entropy(x, w, state['label'], state['row_weight'], bias=b, ignore_index=IGNORE)
        out = {'loss': loss.detach()}
        grads = torch.autograd.grad(loss, leaves) if train else ()
    out.update(zip(('dx', 'dw', 'db'), grads))
    return out


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def _ortho_flops(m, n):
    """the cheaper of the direct form (a symmetric product costs half) and the one that iterates on the Gram matrix, touching the
    m x n matrix every third step"""
    m, n = min(m, n), max(m, n)
    direct = STEPS * (m * m * n + m ** 3 + 2 * m * m * n)
    rounds = -(-STEPS // 3)
    gram = rounds * 3 * m * m * n + (4 * STEPS - 3 * rounds) * m ** 3
    return float(min(direct, gram))


def work(case):
    e = BYTES[case['dtype']]
    if case['op'] == 'norm':
        n = case['rows'] * case['cols']
        return {'bytes': float(n * e * (4 if case['train'] else 2) + 4 * case['cols'] * e), 'flops': float(n * (20 if case['train'] else 8))}
    if case['op'] == 'ce':
        r, k, v = case['rows'], case['hidden'], case['classes']
        once = (r * k + v * k + (v if case['bias'] else 0)) * e
        return {'bytes': float(once * (2 if case['train'] else 1) + r * 12 + 4), 'flops': (6.0 if case['train'] else 2.0) * r * k * v}
    return {'bytes': float(sum(2 * m * n * e for m, n in _shapes(case))), 'flops': sum(_ortho_flops(m, n) for m, n in _shapes(case))}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case['op'] == 'norm':
            x, w, b = (s[k].double() for k in ('x', 'w', 'b'))
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            inv = 1.0 / torch.sqrt(var + LN_EPS)
            h = (x - mean) * inv
            out = {'y': torch.addcmul(b, h, w)}
            if case['train']:
                dy = s['dy'].double()
                t = dy * w
                c = x.size(1)
                out['dx'] = inv / c * (c * t - t.sum(1, keepdim=True) - h * (t * h).sum(1, keepdim=True))
                out['dw'] = torch.einsum('rc,rc->c', dy, h)
                out['db'] = dy.sum(0)
            return out
        if case['op'] == 'ce':
            w = s['w'].double()
            v, k = w.shape
            keep = (s['label'] != IGNORE).nonzero().squeeze(1)
            weight = s['row_weight'][keep].double()
            norm = max(1, int((weight > 0).sum()))
            loss = 0.0
            dx = torch.zeros((case['rows'], k), dtype=torch.float64, device='cuda')
            dw = torch.zeros_like(w)
            db = torch.zeros((v,), dtype=torch.float64, device='cuda')
            for rows, share in zip(keep.split(2048), weight.split(2048)):
                x = s['x'][rows].double()
                logp = x @ w.T
                if s['b'] is not None:
                    logp += s['b'].double()
                logp -= torch.logsumexp(logp, 1, keepdim=True)
                at = (torch.arange(len(rows), device='cuda'), s['label'][rows])
                loss = loss - (logp[at] * share).sum() / norm
                if case['train']:
                    logp.exp_()
                    logp[at] -= 1
                    logp *= (share / norm).unsqueeze(1)
                    dx[rows] = logp @ w
                    dw += logp.T @ x
                    db += logp.sum(0)
            out = {'loss': loss.reshape(1)}
            if case['train']:
                out.update(dx=dx, dw=dw)
                if s['b'] is not None:
                    out['db'] = db
            return out
        out = []
        a, b, c = COEFFICIENTS
        for g in s['mats']:
            # the same polynomial of the singular values, applied from the side where the Gram matrix is small
            x = g.double() / (torch.linalg.vector_norm(g.double()) + NS_EPS)
            for _ in range(STEPS):
                if x.size(0) <= x.size(1):
                    q = x @ x.T
                    x = a * x + b * (q @ x) + c * (q @ (q @ x))
                else:
                    q = x.T @ x
                    x = a * x + b * (x @ q) + c * ((x @ q) @ q)
            out.append(x)
        return out
