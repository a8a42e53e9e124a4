"""The operators of a training step behind the loader, as measurable cases.

A case is one pass through one of four operators:

* ``loss``    cross entropy of a batch of logits and its gradient: against class labels, against the ``[label,
              partner's label, lambda]`` rows of ``LabelMixup``, or against given class probabilities;
* ``norm``    the seam between two blocks of a residual network, forward and backward: the block's output goes
              through the norm behind it, a gate and the residual scale, is added to the stream, and the sum goes
              through the norm of the next block;
* ``rotary``  rotary positions of queries and keys, forward and backward: patches of an image by row and column, or
              places in a long sequence;
* ``adamw``   one AdamW step over all tensors of a network, with the moments in 32 or in 8 bits.

``run`` computes them from their formulas with elementary torch operations in 32 bits, or, where ``own`` is set, with
the calls of ``ffcv_b200.training``; ``exact`` computes them in 64 bits.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
SIZE = {'f32': 4, 'f16': 2, 'bf16': 2}

LR, BETAS, EPS, DECAY, SEED = 1e-3, (0.9, 0.999), 1e-8, 0.05, 17  # of the AdamW cases
CLIP = 1.0     # bound of the gradient's norm
STEPS = 1000   # steps made before the measured one
BLOCK = 256    # values that share one scale of an 8-bit moment
NORM_EPS = 1e-6
BASE = 10000.0  # of the rotary frequencies


def listed():
    return [
        # the loss of one batch of 32 x 32 images with ten classes and mixed labels
        dict(name='loss_512x10_mixed', op='loss', rows=512, classes=10, dtype='f32', target='mixed', smoothing=0.0, masked=False),
        # ... of one batch of the low-resolution training, with label smoothing
        dict(name='loss_1024x1000_mixed', op='loss', rows=1024, classes=1000, dtype='bf16', target='mixed', smoothing=0.1, masked=False),
        # pre-training on a label set of ImageNet-21k's kind, patches or crops of many images at once
        dict(name='loss_8192x21841', op='loss', rows=8192, classes=21841, dtype='bf16', target='labels', smoothing=0.0, masked=True),
        # a small network's seam: one request's 14 x 14 patches and a class token, plain residual, LayerNorm
        dict(name='norm_2x197x192', op='norm', batch=2, tokens=197, width=192, dtype='f32', norm='layer', post='none', gate='none', scale='none'),
        # 256 images of 224 x 224 pixels in 16 x 16 patches, residual scale per channel, LayerNorm
        dict(name='norm_256x197x768', op='norm', batch=256, tokens=197, width=768, dtype='bf16', norm='layer', post='none', gate='none', scale='vector'),
        # 64 images of 384 x 384 pixels in 8 x 8 patches, RMS norms before and after, a gate per image
        dict(name='norm_64x2305x1024', op='norm', batch=64, tokens=2305, width=1024, dtype='bf16', norm='rms', post='rms', gate='sample', scale='vector'),
        # queries and keys of a few images' patches by row and column
        dict(name='rotary_4x14x14', op='rotary', batch=4, rows=14, cols=14, heads=3, kv_heads=3, head_dim=64, rotary_dim=64,
             layout='half', axes=2, scaling='none', packed=False, dtype='f32'),
        # the same of a training batch, cut out of one fused projection, positions scaled down from a larger resolution
        dict(name='rotary_256x16x16', op='rotary', batch=256, rows=16, cols=16, heads=12, kv_heads=12, head_dim=64, rotary_dim=64,
             layout='interleaved', axes=2, scaling='linear', packed=True, dtype='bf16'),
        # one long sequence of tokens with shared key heads, half of every head, frequencies scaled by parts
        dict(name='rotary_2x32768', op='rotary', batch=2, rows=1, cols=32768, heads=32, kv_heads=8, head_dim=128, rotary_dim=64,
             layout='half', axes=1, scaling='ramp', packed=False, dtype='bf16'),
        # a linear classifier on top of a frozen network
        dict(name='adamw_head', op='adamw', layers=0, width=512, patch=4, classes=100, dtype='f32', bits=32, clip=False),
        # 148 tensors, 101 M values, all in 32 bits, the gradient's norm bounded
        dict(name='adamw_101m_clip', op='adamw', layers=12, width=832, patch=16, classes=1000, dtype='f32', bits=32, clip=True),
        # 292 tensors, 409 M values, bf16 weights with 32-bit masters and 8-bit moments
        dict(name='adamw8_409m', op='adamw', layers=24, width=1152, patch=16, classes=21841, dtype='bf16', bits=8, clip=False),
    ]


# The largest listed cases: bounds of the drawn ones.
MOST_LOGITS = 8192 * 21841
MOST_ACTIVATIONS = 64 * 2305 * 1024
MOST_ROTARY = 2 * 32768 * 40 * 128
MOST_WEIGHTS = 408_000_000


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['loss', 'norm', 'rotary', 'adamw'])
    dtype = rng.choice(['f32', 'bf16', 'bf16', 'f16'])
    if op == 'loss':
        target = rng.choice(['labels', 'mixed', 'mixed', 'soft'])
        masked = target == 'labels' and rng.random() < 0.3
        classes = _log_int(rng, 2, 130000)
        rows = min(_log_int(rng, 1, 16384), MOST_LOGITS // classes // (2 if dtype == 'f32' or target == 'soft' else 1))
        return dict(op=op, rows=rows, classes=classes, dtype=dtype, target=target,
                    smoothing=0.0 if masked else rng.choice([0.0, 0.0, 0.1]), masked=masked)
    if op == 'norm':
        width = _log_int(rng, 48, 8192)
        width -= width % 8 if rng.random() < 0.7 else 0
        tokens = _log_int(rng, 1, 4097)
        batch = max(1, min(_log_int(rng, 1, 512), MOST_ACTIVATIONS // (tokens * width) // (2 if dtype == 'f32' else 1)))
        return dict(op=op, batch=batch, tokens=tokens, width=width, dtype=dtype, norm=rng.choice(['layer', 'rms']),
                    post=rng.choice(['none', 'none', 'layer', 'rms']), gate=rng.choice(['none', 'none', 'sample', 'token']),
                    scale=rng.choice(['none', 'vector']))
    if op == 'rotary':
        axes = rng.choice([1, 2])
        rows, cols = (1, _log_int(rng, 1, 65536)) if axes == 1 else (_log_int(rng, 1, 64), _log_int(rng, 1, 64))
        head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        token = (heads + kv_heads) * head_dim * (2 if dtype == 'f32' else 1)
        cols = max(1, min(cols, MOST_ROTARY // (rows * token)))
        return dict(op=op, batch=max(1, min(_log_int(rng, 1, 512), MOST_ROTARY // (rows * cols * token))), rows=rows, cols=cols,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2]),
                    layout=rng.choice(['half', 'interleaved']), axes=axes, scaling=rng.choice(['none', 'linear', 'ntk', 'ramp']),
                    packed=rng.random() < 0.5, dtype=dtype)
    while True:
        case = dict(op=op, layers=rng.choice([0, 1, 2, 4, 6, 12, 24]), width=_log_int(rng, 32, 1280), patch=rng.choice([4, 8, 14, 16]),
                    classes=_log_int(rng, 2, 21841), dtype=dtype, bits=rng.choice([8, 32]), clip=False)
        case['clip'] = case['bits'] == 32 and rng.random() < 0.5
        if sum(math.prod(s) for s in _shapes(case)[0]) <= MOST_WEIGHTS // (2 if dtype == 'f32' else 1):
            return case


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    return {'loss': _prepare_loss, 'norm': _prepare_norm, 'rotary': _prepare_rotary, 'adamw': _prepare_adamw}[case['op']](case, gen)


def run(state):
    plain, theirs = {'loss': (_plain_loss, _own_loss), 'norm': (_plain_norm, _own_norm), 'rotary': (_plain_rotary, _own_rotary),
                     'adamw': (_plain_adamw, _own_adamw)}[state['op']]
    return theirs(state) if own else plain(state)


def work(case):
    return {'loss': _work_loss, 'norm': _work_norm, 'rotary': _work_rotary, 'adamw': _work_adamw}[case['op']](case)


def exact(case, seed):
    state = prepare(case, seed)
    return {'loss': _exact_loss, 'norm': _exact_norm, 'rotary': _exact_rotary, 'adamw': _exact_adamw}[case['op']](state)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device='cuda') * scale).to(dtype)


# ---- loss ------------------------------------------------------------------------------------------------------------

def _prepare_loss(case, gen):
    n, classes = case['rows'], case['classes']
    label = torch.randint(classes, (n,), generator=gen, device='cuda')
    logits = torch.randn((n, classes), generator=gen, device='cuda').mul_(2.0)
    right = torch.rand(n, generator=gen, device='cuda') < 0.6  # samples whose class the network has learnt
    logits[torch.arange(n, device='cuda'), label] += 6.0 * right
    if case['masked']:  # classes that a sample cannot have, and a sample without any; some samples without a label
        logits.masked_fill_(torch.rand((n, classes), generator=gen, device='cuda') < 0.2, -math.inf)
        logits[torch.arange(n, device='cuda'), label] = 3.0
        if n > 2:
            logits[n // 2] = -math.inf
            label[1:].masked_fill_(torch.rand(n - 1, generator=gen, device='cuda') < 0.05, -100)
    state = dict(op='loss', logits=logits.to(DTYPES[case['dtype']]), smoothing=case['smoothing'], target=case['target'],
                 ignore=-100 if case['masked'] else None)
    if case['target'] == 'labels':
        state['labels'] = label
    elif case['target'] == 'mixed':  # what LabelMixup makes: own label, the label of the sample before, lambda
        lam = torch.rand(n, generator=gen, device='cuda')
        state['mixed'] = torch.stack([label.float(), label.roll(1).float(), lam], 1)
    else:
        state['soft'] = torch.softmax(torch.randn((n, classes), generator=gen, device='cuda'), 1)
    return state


def _plain_loss(s):
    x = s['logits'].float()
    n, classes = x.shape
    column = torch.arange(classes, device=x.device)
    counted, rows = None, float(n)
    if s['target'] == 'labels':
        p = (column == s['labels'][:, None]).float()
        if s['ignore'] is not None:
            counted = (s['labels'] != s['ignore'])[:, None].float()
            rows = counted.sum()
    elif s['target'] == 'mixed':
        own_label, other, lam = (s['mixed'][:, k:k + 1] for k in range(3))
        p = lam * (column == own_label) + (1 - lam) * (column == other)
    else:
        p = s['soft']
    target = p * (1 - s['smoothing']) + s['smoothing'] / classes
    total = target.sum(1, keepdim=True)
    top = x.amax(1, keepdim=True)
    empty = top == -math.inf
    e = torch.exp(x - torch.where(empty, 0.0, top))
    mass = e.sum(1, keepdim=True)
    lse = top + torch.log(mass)
    each = total * lse - torch.where(target > 0, target * x, 0.0).sum(1, keepdim=True)
    grad = total * e / mass - target
    if counted is not None:
        each, grad = torch.where(counted > 0, each, 0.0), grad * counted
    each, grad = torch.where(empty, 0.0, each), torch.where(empty, 0.0, grad)
    return {'loss': each.sum() / rows, 'grad': (grad / rows).to(s['logits'].dtype)}


def _own_loss(s):
    from ffcv_b200 import training
    loss, grad = training.cross_entropy_with_grad(s['logits'], label_smoothing=s['smoothing'], ignore_index=s['ignore'],
                                                  **{s['target']: s[s['target']]})
    return {'loss': loss, 'grad': grad}


def _exact_loss(s):
    x = s['logits'].double()
    n, classes = x.shape
    keep = torch.isfinite(x).any(1)
    if s['target'] == 'labels':
        labelled = s['labels'] != s['ignore'] if s['ignore'] is not None else torch.ones_like(keep)
        rows = int(labelled.sum())
        keep = keep & labelled
        picks = [(s['labels'].clamp(min=0), torch.ones(n, dtype=torch.float64, device=x.device))]
    else:
        rows = n
        if s['target'] == 'mixed':
            lam = s['mixed'][:, 2].double()
            picks = [(s['mixed'][:, 0].long(), lam), (s['mixed'][:, 1].long(), 1 - lam)]
    log_p = torch.log_softmax(torch.where(keep[:, None], x, 0.0), 1)
    grad = torch.exp(log_p)
    eps = s['smoothing']
    if s['target'] == 'soft':
        each = -(1 - eps) * (s['soft'].double() * log_p).sum(1)
        mass = (1 - eps) * s['soft'].double().sum(1) + eps
        grad = grad * mass[:, None] - (1 - eps) * s['soft'].double()
    else:
        each = torch.zeros(n, dtype=torch.float64, device=x.device)
        for label, weight in picks:
            each -= (1 - eps) * weight * log_p.gather(1, label[:, None])[:, 0]
            grad.scatter_add_(1, label[:, None], -(1 - eps) * weight[:, None])
    if eps > 0:
        each -= eps * log_p.mean(1)
        grad -= eps / classes
    each = torch.where(keep, each, 0.0)
    return {'loss': each.sum() / rows, 'grad': torch.where(keep[:, None], grad, 0.0) / rows}


def _work_loss(case):
    values = case['rows'] * case['classes']
    row = {'labels': 8, 'mixed': 12, 'soft': 4 * case['classes']}[case['target']]
    return {'bytes': 2 * values * SIZE[case['dtype']] + case['rows'] * row + 4, 'flops': 8 * values}


# ---- norm ------------------------------------------------------------------------------------------------------------

def _prepare_norm(case, gen):
    dtype, (b, t, d) = DTYPES[case['dtype']], (case['batch'], case['tokens'], case['width'])
    stream = torch.randn((b, t, d), generator=gen, device='cuda') * (1 + 3 * torch.rand(d, generator=gen, device='cuda')) + 0.3
    s = dict(op='norm', norm=case['norm'], post=case['post'], x=stream.to(dtype), h=_randn(gen, b, t, d, dtype=dtype, scale=0.7),
             dy=_randn(gen, b, t, d, dtype=dtype, scale=1e-2), dz=_randn(gen, b, t, d, dtype=dtype, scale=1e-2),
             weight=1 + _randn(gen, d, scale=0.2), bias=None, post_weight=None, post_bias=None, gate=None, scale=None)
    if case['norm'] == 'layer':
        s['bias'] = _randn(gen, d, scale=0.1)
    if case['post'] != 'none':
        s['post_weight'] = 1 + _randn(gen, d, scale=0.2)
    if case['post'] == 'layer':
        s['post_bias'] = _randn(gen, d, scale=0.1)
    if case['gate'] != 'none':
        s['gate'] = _randn(gen, b, 1 if case['gate'] == 'sample' else t, d, dtype=dtype, scale=0.5)
    if case['scale'] == 'vector':
        s['scale'] = 0.1 + _randn(gen, d, scale=0.02)
    return s


def _normed(a, kind):
    """The normalised values and 1 / (standard deviation or root mean square) of rows."""
    if kind == 'layer':
        a = a - a.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((a * a).mean(-1, keepdim=True) + NORM_EPS)
    return a * r, r


def _normed_back(g, a, r, kind):
    """The gradient before a norm: g is the gradient of the normalised values a."""
    g = g - a * (g * a).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == 'layer' else 0.0)
    return g * r


def _plain_norm(s):
    dtype, width = s['x'].dtype, s['x'].shape[-1]
    x, h, dy, dz = (s[k].float() for k in ('x', 'h', 'dy', 'dz'))
    gate = 1.0 if s['gate'] is None else s['gate'].float()
    scale = 1.0 if s['scale'] is None else s['scale']
    inner, inner_r = (h, None) if s['post'] == 'none' else _normed(h, s['post'])
    u = inner if s['post_weight'] is None else inner * s['post_weight']
    u = u if s['post_bias'] is None else u + s['post_bias']
    y = x + u * (gate * scale)
    outer, outer_r = _normed(y, s['norm'])
    z = outer * s['weight']
    z = z if s['bias'] is None else z + s['bias']
    out = {'y': y.to(dtype), 'z': z.to(dtype)}

    dx = dy + _normed_back(dz * s['weight'], outer, outer_r, s['norm'])
    du = dx * (gate * scale)
    dh = du if s['post_weight'] is None else _normed_back(du * s['post_weight'], inner, inner_r, s['post'])
    out.update(dx=dx.to(dtype), dh=dh.to(dtype), dweight=(dz * outer).reshape(-1, width).sum(0))
    if s['bias'] is not None:
        out['dbias'] = dz.reshape(-1, width).sum(0)
    if s['post_weight'] is not None:
        out['dpost_weight'] = (du * inner).reshape(-1, width).sum(0)
    if s['post_bias'] is not None:
        out['dpost_bias'] = du.reshape(-1, width).sum(0)
    if s['gate'] is not None:
        dgate = dx * u * scale
        out['dgate'] = (dgate.sum(1, keepdim=True) if s['gate'].shape[1] < x.shape[1] else dgate).to(dtype)
    if s['scale'] is not None:
        out['dscale'] = (dx * u * gate).reshape(-1, width).sum(0)
    return out


def _own_norm(s):
    from ffcv_b200 import training
    how = dict(norm=s['norm'], weight=s['weight'], bias=s['bias'], post_norm=None if s['post'] == 'none' else s['post'],
               post_weight=s['post_weight'], post_bias=s['post_bias'], gate=s['gate'], scale=s['scale'], eps=NORM_EPS)
    y, z, stats = training.norm_residual_forward(s['x'], s['h'], **how)
    grads = training.norm_residual_backward(s['dy'], s['dz'], s['x'], s['h'], stats, **how)
    out = {'y': y, 'z': z}
    out.update({'d' + name: g for name, g in grads.items()})
    return out


def _exact_norm(s):
    names = [k for k in ('x', 'h', 'weight', 'bias', 'post_weight', 'post_bias', 'gate', 'scale') if s[k] is not None]
    v = {k: s[k].double().requires_grad_() for k in names}

    def norm(a, kind, weight, bias):
        mean = a.mean(-1, keepdim=True) if kind == 'layer' else 0.0
        out = (a - mean) * torch.rsqrt(((a - mean) ** 2).mean(-1, keepdim=True) + NORM_EPS) * weight
        return out if bias is None else out + bias

    u = v['h']
    if s['post'] != 'none':
        u = norm(u, s['post'], v['post_weight'], v.get('post_bias'))
    if 'gate' in v:
        u = u * v['gate']
    if 'scale' in v:
        u = u * v['scale']
    y = v['x'] + u
    z = norm(y, s['norm'], v['weight'], v.get('bias'))
    grads = torch.autograd.grad([y, z], [v[k] for k in names], [s['dy'].double(), s['dz'].double()])
    return {'y': y.detach(), 'z': z.detach(), **{'d' + k: g for k, g in zip(names, grads)}}


def _work_norm(case):
    rows, d, size = case['batch'] * case['tokens'], case['width'], SIZE[case['dtype']]
    streams = 8 + {'none': 0, 'sample': 2 / case['tokens'], 'token': 2}[case['gate']]
    params = 1 + (case['norm'] == 'layer') + (case['post'] != 'none') + (case['post'] == 'layer') + (case['scale'] == 'vector')
    return {'bytes': streams * rows * d * size + 8 * d * params, 'flops': (30 + 14 * (case['post'] != 'none')) * rows * d}


# ---- rotary ----------------------------------------------------------------------------------------------------------

def _frequencies(case):
    """Radians per unit of position of every pair, and the factor of the rotated values, in 64 bits."""
    dim, factor, length = case['rotary_dim'] // case['axes'], 4.0, 4096
    base = BASE * factor ** (dim / (dim - 2)) if case['scaling'] == 'ntk' else BASE
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    amplitude = 1.0
    if case['scaling'] == 'linear':
        f = f / factor
    elif case['scaling'] == 'ramp':  # turns over the original length: few are interpolated, many kept
        keep = ((length * f / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        f = f * ((1 - keep) / factor + keep)
        amplitude = 0.1 * math.log(factor) + 1
    return f, amplitude


def _prepare_rotary(case, gen):
    dtype, b, t = DTYPES[case['dtype']], case['batch'], case['rows'] * case['cols']
    heads, kv_heads, dim = case['heads'], case['kv_heads'], case['head_dim']
    s = dict(op='rotary', half=case['layout'] == 'half', rotary_dim=case['rotary_dim'])
    for name in ('', 'd'):
        if case['packed']:  # queries, keys and values as one projection makes them
            fused = _randn(gen, b, t, heads + 2 * kv_heads, dim, dtype=dtype)
            s[name + 'q'], s[name + 'k'] = fused[:, :, :heads], fused[:, :, heads:heads + kv_heads]
        else:
            s[name + 'q'], s[name + 'k'] = _randn(gen, b, t, heads, dim, dtype=dtype), _randn(gen, b, t, kv_heads, dim, dtype=dtype)
    f, s['amplitude'] = _frequencies(case)
    if case['axes'] == 2:  # the patches' rows and columns
        s['positions'] = torch.cartesian_prod(torch.arange(case['rows']), torch.arange(case['cols'])).cuda()
        length = max(case['rows'], case['cols'])
    else:  # several documents in a row, each counted from its beginning
        place = torch.arange(t, device='cuda')
        first = torch.randint(t, (b, 1), generator=gen, device='cuda')
        s['positions'] = torch.where(place >= first, place - first, place).contiguous()
        length = t
    # what a program without the operator keeps: sines and cosines of all positions
    angle = torch.outer(torch.arange(length, dtype=torch.float64), f)
    s['cos'], s['sin'] = angle.cos().float().cuda(), angle.sin().float().cuda()
    s['f'] = f.cuda()
    if own:
        from ffcv_b200 import training
        s['rotary'] = training.RotaryPositions(dim, rotary_dim=case['rotary_dim'], base=BASE, layout=case['layout'], axes=case['axes'],
                                               scaling=case['scaling'], factor=4.0, original_length=4096)
    return s


def _rotated(a, cos, sin, s):
    r = s['rotary_dim']
    x, rest = a[..., :r].float(), a[..., r:]
    u, v = (x[..., :r // 2], x[..., r // 2:]) if s['half'] else (x[..., 0::2], x[..., 1::2])
    p, q = (u * cos - v * sin) * s['amplitude'], (u * sin + v * cos) * s['amplitude']
    turned = torch.cat([p, q], -1) if s['half'] else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([turned.to(a.dtype), rest], -1)


def _plain_rotary(s):
    at = s['positions']
    pick = lambda table: (table[at] if table.shape[1] * 2 == s['rotary_dim'] else table[at].flatten(-2))[..., None, :]  # noqa: E731
    cos, sin = pick(s['cos']), pick(s['sin'])
    return {'q': _rotated(s['q'], cos, sin, s), 'k': _rotated(s['k'], cos, sin, s),
            'dq': _rotated(s['dq'], cos, -sin, s), 'dk': _rotated(s['dk'], cos, -sin, s)}


def _own_rotary(s):
    q, k = s['rotary'].rotate(s['q'], s['k'], s['positions'])
    dq, dk = s['rotary'].rotate(s['dq'], s['dk'], s['positions'], transpose=True)
    return {'q': q, 'k': k, 'dq': dq, 'dk': dk}


def _exact_rotary(s):
    angle = s['positions'].double()[..., None] * s['f']
    if s['f'].numel() * 2 != s['rotary_dim']:
        angle = angle.flatten(-2)
    turn = torch.polar(torch.full_like(angle, s['amplitude']), angle)[..., None, :]
    out = {}
    for name, turned_by in (('q', turn), ('k', turn), ('dq', turn.conj()), ('dk', turn.conj())):
        a = s[name].double()
        r = s['rotary_dim']
        x = a[..., :r]
        x = x.unflatten(-1, (2, r // 2)).transpose(-1, -2) if s['half'] else x.unflatten(-1, (r // 2, 2))
        x = torch.view_as_real(torch.view_as_complex(x.contiguous()) * turned_by)
        x = x.transpose(-1, -2) if s['half'] else x
        out[name] = torch.cat([x.flatten(-2), a[..., r:]], -1)
    return out


def _work_rotary(case):
    tokens = case['batch'] * case['rows'] * case['cols']
    heads = tokens * (case['heads'] + case['kv_heads'])
    where = 16 * case['rows'] * case['cols'] if case['axes'] == 2 else 8 * tokens
    return {'bytes': 4 * heads * case['head_dim'] * SIZE[case['dtype']] + where, 'flops': 2 * 3 * heads * case['rotary_dim']}


# ---- adamw -----------------------------------------------------------------------------------------------------------

def _shapes(case):
    """The tensors of a small image transformer: matrices, which decay, and vectors, which do not."""
    w, matrices, vectors = case['width'], [], []
    if case['layers']:
        matrices.append((w, 3 * case['patch'] ** 2))
        vectors.append((w,))
    for _ in range(case['layers']):
        matrices += [(3 * w, w), (w, w), (4 * w, w), (w, 4 * w)]
        vectors += [(3 * w,), (w,), (4 * w,), (w,), (w,), (w,), (w,), (w,)]
    matrices.append((case['classes'], w))
    vectors.append((case['classes'],))
    return matrices + vectors, len(matrices)


def _prepare_adamw(case, gen):
    dtype = DTYPES[case['dtype']]
    shapes, matrices = _shapes(case)
    counts = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for c in counts:  # every tensor begins a block
        starts.append(total)
        total += -(-c // BLOCK) * BLOCK
    used = torch.ones(total, dtype=torch.bool, device='cuda')
    for start, c in zip(starts, counts):
        used[start + c:start + -(-c // BLOCK) * BLOCK] = False
    magnitude = torch.exp(1.5 * torch.randn(total // BLOCK, 1, generator=gen, device='cuda')) * 1e-3  # of the blocks' gradients

    def values(scale):
        v = torch.randn((total // BLOCK, BLOCK), generator=gen, device='cuda') * scale
        return v.view(-1).masked_fill_(~used, 0.0)

    master = values(0.02)
    s = dict(op='adamw', bits=case['bits'], clip=CLIP if case['clip'] else None, decayed=starts[matrices], step=STEPS,
             params=master.to(dtype), grads=values(magnitude).to(dtype), master=None if dtype == torch.float32 else master)
    m, v = values(magnitude * 0.3), values(magnitude).square_().add_(1e-12).masked_fill_(~used, 0.0)
    if case['bits'] == 8:
        s['m'], m_scale = _to_eight(m, torch.float8_e4m3fn, 7)
        s['v'], v_scale = _to_eight(v, torch.float8_e5m2, 14)
        s['scales'] = torch.stack([m_scale, v_scale], 1)
    else:
        s['m'], s['v'], s['scales'] = m, v, None
    if own:
        from ffcv_b200 import training
        views = [s['params'][a:a + c].view(shape) for a, c, shape in zip(starts, counts, shapes)]
        params = [torch.nn.Parameter(p) for p in views]
        for p, a, c, shape in zip(params, starts, counts, shapes):
            p.grad = s['grads'][a:a + c].view(shape)
        groups = [dict(params=params[:matrices]), dict(params=params[matrices:], weight_decay=0.0)]
        opt = training.AdamW(groups, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case['bits'],
                             max_grad_norm=s['clip'], seed=SEED)
        saved = opt.state_dict()
        for i, (a, c, shape) in enumerate(zip(starts, counts, shapes)):
            entry = dict(step=STEPS, exp_avg=s['m'][a:a + c].view(shape), exp_avg_sq=s['v'][a:a + c].view(shape))
            if case['bits'] == 8:
                entry['scales'] = s['scales'][a // BLOCK:-(-(a + c) // BLOCK)]
            if s['master'] is not None:
                entry['master'] = s['master'][a:a + c].view(shape)
            saved['state'][i] = entry
        opt.load_state_dict(saved)
        s.update(opt=opt, m=None, v=None, scales=None, master=None)
    return s


def _to_eight(values, dtype, top):
    """Blocks of values in 8 bits, and their scales: powers of two that bring the largest to 2^top .. 2^(top + 1)."""
    blocks = values.view(-1, BLOCK)
    scale = _power(torch.frexp(blocks.abs().amax(1))[1] - 1) * 2.0 ** -top
    return (blocks / scale[:, None]).to(dtype).view(-1), scale


def _power(exponent):
    """2^exponent, -127 < exponent < 128."""
    return ((exponent + 127) << 23).view(torch.float32)


def _mix(x):
    """A 32-bit hash of 32-bit whole numbers: a multiplication between two, and a shift on either side of the second."""
    x = (x * 0xE4C6EF2B) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x87EA99B3) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _step_key(seed, step):
    return _mix(_mix((seed + 1) & 0xFFFFFFFF) ^ (step & 0xFFFFFFFF))


def _plain_adamw(s):
    s['step'] += 1
    t, (b1, b2), dtype = s['step'], BETAS, s['params'].dtype
    g = s['grads'].float()
    out = {}
    if s['clip'] is not None:
        out['grad_norm'] = torch.sqrt((g * g).sum())
        g = g * torch.clamp(s['clip'] / (out['grad_norm'] + 1e-6), max=1.0)
    if s['bits'] == 8:
        scales = s['scales']
        m = (s['m'].float().view(-1, BLOCK) * scales[:, :1]).view(-1)
        v = (s['v'].float().view(-1, BLOCK) * scales[:, 1:]).view(-1)
    else:
        m, v = s['m'], s['v']
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    w = s['params'].float() if s['master'] is None else s['master']
    update = m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + EPS)
    w[:s['decayed']] *= 1 - LR * DECAY
    w -= update * (LR / (1 - b1 ** t))
    if s['bits'] == 8:
        place = torch.arange(m.numel(), device='cuda')
        noise = _mix((place + _step_key(SEED, t)) & 0xFFFFFFFF)
        s['m'], m_scale = _round_to_eight(m, (noise & 0xFFFF) << 4, 7, 120, 20, torch.float8_e4m3fn)
        s['v'], v_scale = _round_to_eight(v, (noise >> 16) << 5, 14, 112, 21, torch.float8_e5m2)
        s['scales'] = out['scales'] = torch.stack([m_scale, v_scale], 1)
    else:
        s['m'], s['v'] = m, v
    if s['master'] is not None:
        out['master'] = w
    s['params'].copy_(w)
    return {'params': s['params'], 'm': s['m'], 'v': s['v'], **out}


def _round_to_eight(values, noise, top, bias, dropped, dtype):
    """Stochastic rounding to an 8-bit type. A block's largest value is brought to 2^top .. 2^(top + 1) by a power of two; the
    exponent is then lowered by the difference of the two types' biases, so that the upper bits of the 32-bit number, its
    own denormals among them, are those of the 8-bit one, and noise is added to the bits that are dropped."""
    blocks = values.view(-1, BLOCK)
    exponent = (blocks.abs().amax(1).view(torch.int32) >> 23).clamp(min=1) - 127
    bits = ((blocks.abs() * _power(-exponent)[:, None]) * 2.0 ** (top - bias)).view(torch.int32)
    code = (bits + noise.view(-1, BLOCK).int()) >> dropped
    if dtype == torch.float8_e5m2:  # a second moment above zero stays above zero
        code = torch.maximum(code, (blocks > 0).int())
    code = code | ((blocks < 0).int() << 7)
    scale = _power(exponent) * 2.0 ** -top
    return code.to(torch.uint8).view(dtype).view(-1), scale


def _own_adamw(s):
    opt = s['opt']
    opt.step()
    out = {'params': s['params'], 'm': opt.exp_avg, 'v': opt.exp_avg_sq}
    if s['clip'] is not None:
        out['grad_norm'] = opt.grad_norm
    if s['bits'] == 8:
        out['scales'] = opt.scales
    if opt.master is not None:
        out['master'] = opt.master
    return out


def _exact_adamw(s):
    t, (b1, b2) = s['step'] + 1, BETAS
    g = s['grads'].double()
    out = {}
    if s['clip'] is not None:
        out['grad_norm'] = g.norm()
        g = g * min(1.0, s['clip'] / (float(out['grad_norm']) + 1e-6))
    m, v = s['m'].double(), s['v'].double()
    if s['bits'] == 8:
        m, v = (a.view(-1, BLOCK) * s['scales'][:, k, None].double() for k, a in enumerate((m, v)))
    m, v = m.view(-1).lerp(g, 1 - b1), v.view(-1).lerp(g * g, 1 - b2)
    w = (s['params'] if s['master'] is None else s['master']).double()
    decay = torch.ones_like(w)
    decay[:s['decayed']] -= LR * DECAY
    w = torch.addcdiv(w * decay, m, (v / (1 - b2 ** t)).sqrt() + EPS, value=-LR / (1 - b1 ** t))
    out.update(params=w)
    if s['master'] is not None:
        out['master'] = w
    if s['bits'] == 8:
        noise = _mix((torch.arange(m.numel(), device='cuda') + _step_key(SEED, t)) & 0xFFFFFFFF)
        steps = []
        for name, a, part, top, low, digits in (('m', m, noise & 0xFFFF, 7, -6, 3), ('v', v, noise >> 16, 14, -14, 2)):
            a = a.view(-1, BLOCK)
            scale = torch.exp2((torch.frexp(a.abs().amax(1))[1] - 1 - top).double())
            a = a / scale[:, None]
            step = torch.exp2((torch.frexp(a)[1] - 1).clamp(min=low).double() - digits)  # between neighbours around a
            size = torch.floor(a.abs() / step + part.view(-1, BLOCK) / 65536.0) * step
            if name == 'v':
                size = torch.where(a > 0, size.clamp(min=2.0 ** (low - digits)), size)
            out[name] = (size * torch.sign(a)).view(-1)
            steps.append(scale)
        out['scales'] = torch.stack(steps, 1)
    else:
        out.update(m=m, v=v)
    return out


def _work_adamw(case):
    weights, size = sum(math.prod(s) for s in _shapes(case)[0]), SIZE[case['dtype']]
    each = 3 * size + (0 if size == 4 else 8) + (16 if case['bits'] == 32 else 4 + 16 / BLOCK)
    return {'bytes': each * weights, 'flops': (14 if case['bits'] == 32 else 40) * weights}
