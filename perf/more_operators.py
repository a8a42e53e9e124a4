"""More operators of a training step behind the loader, as measurable cases.

A case is one pass through one of three operators:

* ``head``     a classifier of many classes and its cross entropy, with the gradients of hidden values, weights and bias: the
               logits are the product of both and are not kept;
* ``distill``  the loss of a batch of logits against a teacher's largest logits, with or without the loss against labels
               beside it, and its gradient;
* ``group``    group norm of images that lie channels last with an activation behind it, forward and backward, or forward alone.

``run`` computes them from their formulas with elementary torch operations in 32 bits, or, where ``own`` is set, with
the calls of ``ffcv_b200.training``; ``exact`` computes them in 64 bits.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
SIZE = {'f32': 4, 'f16': 2, 'bf16': 2}
IGNORE = -100
EPS = 1e-5  # of the group norm
SCALE = {'f32': 1.0, 'f16': 4096.0, 'bf16': 1.0}  # of the losses' gradients, which 16 bits with a small exponent could not hold


def listed():
    return [
        # the last layer of a small network on a small batch, mixed labels with smoothing
        dict(name='head_64x1000x384', op='head', rows=64, classes=1000, width=384, dtype='bf16', target='mixed', smoothing=0.1,
             bias=True, ignored=0.0),
        # the last, incomplete batch of an epoch over a label set of ImageNet-21k's kind
        dict(name='head_1021x21841x768', op='head', rows=1021, classes=21841, width=768, dtype='bf16', target='labels', smoothing=0.0,
             bias=True, ignored=0.0),
        # pre-training on the same set, crops of many images at once
        dict(name='head_8192x21841x1024', op='head', rows=8192, classes=21841, width=1024, dtype='bf16', target='labels', smoothing=0.0,
             bias=False, ignored=0.0),
        # masked patches: 256 images of 14 x 14 patches, each predicted as one of 8192 visual tokens, where it was hidden
        dict(name='head_50176x8192x768_masked', op='head', rows=50176, classes=8192, width=768, dtype='f16', target='labels',
             smoothing=0.0, bias=True, ignored=0.6),
        # a batch of 32 x 32 images with ten classes, the teacher's best three
        dict(name='distill_512x10_3', op='distill', rows=512, classes=10, kept=3, dtype='f32', temperature=2.0, hard=0.5,
             target='labels', smoothing=0.0, ragged=False),
        # a batch of the low-resolution training, mixed labels, the teacher's best ten
        dict(name='distill_1024x1000_10', op='distill', rows=1024, classes=1000, kept=10, dtype='bf16', temperature=1.0, hard=0.5,
             target='mixed', smoothing=0.1, ragged=False),
        # pre-training on many classes from stored logits alone; some samples have fewer of them, or none
        dict(name='distill_8192x21841_64', op='distill', rows=8192, classes=21841, kept=64, dtype='bf16', temperature=2.0, hard=0.0,
             target='labels', smoothing=0.0, ragged=True),
        # a still larger label set, an odd number of samples, a temperature between whole numbers
        dict(name='distill_1531x50021_200', op='distill', rows=1531, classes=50021, kept=200, dtype='f16', temperature=3.5, hard=0.3,
             target='labels', smoothing=0.0, ragged=True),
        # the last stage of a convolutional network on two images
        dict(name='group_2x7x7x512', op='group', batch=2, height=7, width=7, channels=512, groups=32, dtype='f32', activation='silu',
             direction='both'),
        # its first stage on a training batch of 224 x 224 images
        dict(name='group_256x56x56x256', op='group', batch=256, height=56, width=56, channels=256, groups=32, dtype='bf16',
             activation='silu', direction='both'),
        # images that are not square, groups of 30 channels
        dict(name='group_97x28x30x480', op='group', batch=97, height=28, width=30, channels=480, groups=16, dtype='f16', activation='gelu',
             direction='both'),
        # the decoder of an image autoencoder at full resolution
        dict(name='group_4x512x512x128_forward', op='group', batch=4, height=512, width=512, channels=128, groups=32, dtype='bf16',
             activation='silu', direction='forward'),
    ]


# The largest listed cases: bounds of the drawn ones.
MOST_PRODUCTS = 8192 * 21841 * 1024
MOST_LOGITS = 8192 * 21841
MOST_PIXELS = 256 * 56 * 56 * 256


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['head', 'distill', 'group'])
    if op == 'head':
        width = _log_int(rng, 16, 4096)
        width -= width % 8 if width > 8 and rng.random() < 0.8 else 0
        classes = _log_int(rng, 2, 65536)
        target = rng.choice(['labels', 'labels', 'mixed'])
        return dict(op=op, rows=min(_log_int(rng, 1, 65536), MOST_PRODUCTS // (classes * width), MOST_LOGITS * 2 // classes), classes=classes, width=width,
                    dtype=rng.choice(['bf16', 'bf16', 'f16']), target=target, smoothing=rng.choice([0.0, 0.0, 0.1]), bias=rng.random() < 0.5,
                    ignored=rng.choice([0.0, 0.0, 0.15, 0.6]) if target == 'labels' else 0.0)
    dtype = rng.choice(['f32', 'bf16', 'bf16', 'f16'])
    if op == 'distill':
        classes = _log_int(rng, 2, 130000)
        return dict(op=op, rows=min(_log_int(rng, 1, 16384), MOST_LOGITS // classes // (2 if dtype == 'f32' else 1)), classes=classes,
                    kept=min(classes, _log_int(rng, 1, 256)), dtype=dtype, temperature=rng.choice([1.0, 2.0, 3.5, 4.0]),
                    hard=rng.choice([0.0, 0.3, 0.5]), target=rng.choice(['labels', 'mixed']), smoothing=rng.choice([0.0, 0.1]),
                    ragged=rng.random() < 0.5)
    groups = rng.choice([1, 2, 3, 4, 8, 16, 32, 32])
    share = rng.choice([4, 8, 12, 16, 32, 64]) if rng.random() < 0.8 else rng.randint(1, 40)
    height, width = _log_int(rng, 1, 512), _log_int(rng, 1, 512)
    height = max(height, -(-64 // (width * share)))  # (a group of few values has hardly any gradient)
    width = max(1, min(width, MOST_PIXELS // (height * groups * share * 2)))
    sample = height * width * groups * share * (2 if dtype == 'f32' else 1)
    return dict(op=op, batch=max(1, min(_log_int(rng, 1, 512), MOST_PIXELS // sample)), height=height, width=width,
                channels=groups * share, groups=groups, dtype=dtype,
                activation=rng.choice(['none', 'silu', 'gelu']),  # (relu's slope jumps at 0, where rounding decides)
                direction=rng.choice(['both', 'both', 'forward']))


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    return {'head': _prepare_head, 'distill': _prepare_distill, 'group': _prepare_group}[case['op']](case, gen)


def run(state):
    plain, theirs = {'head': (_plain_head, _own_head), 'distill': (_plain_distill, _own_distill), 'group': (_plain_group, _own_group)}[state['op']]
    return theirs(state) if own else plain(state)


def work(case):
    return {'head': _work_head, 'distill': _work_distill, 'group': _work_group}[case['op']](case)


def exact(case, seed):
    state = prepare(case, seed)
    return {'head': _exact_head, 'distill': _exact_distill, 'group': _exact_group}[case['op']](state)


def _randn(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device='cuda').mul_(scale)


def _targets(case, gen, n, classes):
    """One class per sample, and as the case has it: labels, or the [label, label of the sample before, lambda] rows of ``LabelMixup``."""
    label = torch.randint(classes, (n,), generator=gen, device='cuda')
    if case['target'] == 'labels':
        return label, {'labels': label}
    return label, {'mixed': torch.stack([label.float(), label.roll(1).float(), torch.rand(n, generator=gen, device='cuda')], 1)}


def _target_rows(s, classes, dtype):
    """The targets as probabilities per class."""
    column = torch.arange(classes, device='cuda')
    if 'labels' in s:
        p = (column == s['labels'][:, None]).to(dtype)
    else:
        first, second, lam = (s['mixed'][:, k:k + 1].to(dtype) for k in range(3))
        p = lam * (column == first) + (1 - lam) * (column == second)
    return p * (1 - s['smoothing']) + s['smoothing'] / classes


# ---- head ------------------------------------------------------------------------------------------------------------

def _ignored_rows(case):
    return int(case['ignored'] * case['rows'])


def _prepare_head(case, gen):
    n, classes, width = case['rows'], case['classes'], case['width']
    dtype = DTYPES[case['dtype']]
    weight = _randn(gen, classes, width, scale=2.0 / math.sqrt(width))
    label, target = _targets(case, gen, n, classes)
    hidden = _randn(gen, n, width)  # what a norm gives, moved towards the class where the network has learnt it
    learnt = torch.rand((n, 1), generator=gen, device='cuda') < 0.6
    hidden += 1.5 * learnt * weight[label]
    bias = _randn(gen, classes, scale=0.3).to(dtype) if case['bias'] else None
    ignored = _ignored_rows(case)
    if ignored:  # patches that were not hidden
        label[torch.randperm(n, generator=gen, device='cuda')[:ignored]] = IGNORE
    return dict(op='head', hidden=hidden.to(dtype), weight=weight.to(dtype), bias=bias, smoothing=case['smoothing'],
                ignore=IGNORE if ignored else None, scale=SCALE[case['dtype']], **target)


def _plain_head(s):
    x, w = s['hidden'].float(), s['weight'].float()
    z = x @ w.t()
    if s['bias'] is not None:
        z = z + s['bias'].float()
    target = _target_rows(s, w.shape[0], torch.float32)
    total = target.sum(1, keepdim=True)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    mass = e.sum(1, keepdim=True)
    each = total * torch.log(mass) - (target * (z - top)).sum(1, keepdim=True)
    grad = total * e / mass - target
    rows = float(x.shape[0])
    if s['ignore'] is not None:
        counted = (s['labels'] != s['ignore'])[:, None].float()
        rows = counted.sum().clamp(min=1.0)
        each, grad = each * counted, grad * counted
    grad = grad * (s['scale'] / rows)
    dtype = s['hidden'].dtype
    out = {'loss': each.sum() / rows, 'hidden': (grad @ w).to(dtype), 'weight': (grad.t() @ x).to(dtype)}
    if s['bias'] is not None:
        out['bias'] = grad.sum(0).to(dtype)
    return out


def _own_head(s):
    from ffcv_b200 import training
    loss, hidden, weight, bias = training.linear_cross_entropy_with_grad(
        s['hidden'], s['weight'], s.get('labels'), mixed=s.get('mixed'), bias=s['bias'], label_smoothing=s['smoothing'], ignore_index=s['ignore'],
        grad_scale=s['scale'])
    out = {'loss': loss, 'hidden': hidden, 'weight': weight}
    if bias is not None:
        out['bias'] = bias
    return out


def _exact_head(s):
    x, w = s['hidden'].double(), s['weight'].double()
    z = torch.mm(x, w.t())
    if s['bias'] is not None:
        z += s['bias'].double()
    lse = torch.logsumexp(z, 1)
    n, classes = z.shape
    row = torch.arange(n, device='cuda')
    if 'labels' in s:
        kept = torch.ones(n, dtype=torch.bool, device='cuda') if s['ignore'] is None else s['labels'] != s['ignore']
        picks = [(s['labels'].clamp(min=0), torch.ones(n, dtype=torch.float64, device='cuda'))]
    else:
        kept, lam = torch.ones(n, dtype=torch.bool, device='cuda'), s['mixed'][:, 2].double()
        picks = [(s['mixed'][:, 0].long(), lam), (s['mixed'][:, 1].long(), 1 - lam)]
    smoothing, share = s['smoothing'], kept.double() / kept.sum().clamp(min=1)
    each = lse - smoothing * z.mean(1)
    grad = torch.exp(z - lse[:, None]) - smoothing / classes
    for label, weight in picks:
        each = each - (1 - smoothing) * weight * z[row, label]
        grad[row, label] -= (1 - smoothing) * weight
    grad *= share[:, None] * s['scale']
    out = {'loss': (each * share).sum(), 'hidden': torch.mm(grad, w), 'weight': torch.mm(grad.t(), x)}
    if s['bias'] is not None:
        out['bias'] = grad.sum(0)
    return out


def _work_head(case):
    n, classes, width = case['rows'], case['classes'], case['width']
    values = 2 * (n * width + classes * width) + (2 * classes if case['bias'] else 0)
    targets = n * (8 if case['target'] == 'labels' else 12)
    return {'bytes': SIZE[case['dtype']] * values + targets, 'flops': 6 * (n - _ignored_rows(case)) * classes * width}


# ---- distill ---------------------------------------------------------------------------------------------------------

def _prepare_distill(case, gen):
    n, classes, kept = case['rows'], case['classes'], case['kept']
    dtype = DTYPES[case['dtype']]
    label, target = _targets(case, gen, n, classes)
    teacher = _randn(gen, n, classes, scale=2.0)
    teacher[torch.arange(n, device='cuda'), label] += 6.0
    student = (teacher * 0.7).add_(_randn(gen, n, classes)).to(dtype)
    best, where = teacher.topk(kept, 1)
    if case['ragged']:  # samples with fewer stored logits, or none, are filled up with class -1
        count = torch.randint(0, kept + 1, (n, 1), generator=gen, device='cuda')
        count[1:][torch.rand((n - 1, 1), generator=gen, device='cuda') < 0.7] = kept
        none = torch.arange(kept, device='cuda') >= count
        best, where = best.masked_fill(none, 0.0), where.masked_fill(none, -1)
    # as they come out of a data set: 16 bits, or 32 with logits of 32, and classes of 32 bits
    return dict(op='distill', logits=student, teacher=best.to(torch.float32 if dtype == torch.float32 else torch.float16), classes=where.int(),
                temperature=case['temperature'], hard=case['hard'], smoothing=case['smoothing'], scale=SCALE[case['dtype']],
                **target)


def _plain_distill(s):
    z, tau, hard = s['logits'].float(), s['temperature'], s['hard']
    n, classes = z.shape
    there = s['classes'] >= 0
    where = s['classes'].long().clamp(min=0)
    t = torch.where(there, s['teacher'].float() / tau, -math.inf)
    most = t.amax(1, keepdim=True)
    q = torch.exp(t - torch.where(most == -math.inf, 0.0, most))
    given = q.sum(1, keepdim=True)
    any_ = (given > 0).float()
    q = torch.where(given > 0, q / given, 0.0)
    top = z.amax(1, keepdim=True)
    e = torch.exp((z - top) / tau)
    mass = e.sum(1, keepdim=True)
    log_p = (z.gather(1, where) - top) / tau - torch.log(mass)
    each = tau * tau * torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)) - log_p), 0.0).sum(1, keepdim=True)
    grad = (any_ * e / mass).scatter_add_(1, where, -q) * tau
    if hard:
        target = _target_rows(s, classes, torch.float32)
        total = target.sum(1, keepdim=True)
        e = torch.exp(z - top)
        mass = e.sum(1, keepdim=True)
        other = total * torch.log(mass) - (target * (z - top)).sum(1, keepdim=True)
        each = (1 - hard) * each + hard * other
        grad = (1 - hard) * grad + hard * (total * e / mass - target)
    return {'loss': each.sum() / n, 'grad': (grad * (s['scale'] / n)).to(s['logits'].dtype)}


def _own_distill(s):
    from ffcv_b200 import training
    targets = {k: s[k] for k in ('labels', 'mixed') if k in s} if s['hard'] else {}
    loss, grad = training.distillation_with_grad(s['logits'], s['teacher'], s['classes'], temperature=s['temperature'], hard_weight=s['hard'],
                                                 label_smoothing=s['smoothing'] if s['hard'] else 0.0, grad_scale=s['scale'], **targets)
    return {'loss': loss, 'grad': grad}


def _exact_distill(s):
    z, tau, hard = s['logits'].double().requires_grad_(), s['temperature'], s['hard']
    n, classes = z.shape
    t = (s['teacher'].double() / tau).masked_fill(s['classes'] < 0, -math.inf)
    q = torch.softmax(t, 1).nan_to_num(0.0)
    where = s['classes'].long().clamp(min=0)
    log_p = torch.log_softmax(z / tau, 1)
    loss = tau ** 2 * (torch.xlogy(q, q) - q * log_p.gather(1, where)).sum() / n
    if hard:
        log_p = torch.log_softmax(z, 1)
        row = torch.arange(n, device='cuda')
        if 'labels' in s:
            right = log_p[row, s['labels']]
        else:
            lam = s['mixed'][:, 2].double()
            right = lam * log_p[row, s['mixed'][:, 0].long()] + (1 - lam) * log_p[row, s['mixed'][:, 1].long()]
        loss = (1 - hard) * loss - hard * ((1 - s['smoothing']) * right + s['smoothing'] * log_p.mean(1)).sum() / n
    loss.backward()
    return {'loss': loss.detach(), 'grad': z.grad * s['scale']}


def _work_distill(case):
    n, classes, size = case['rows'], case['classes'], SIZE[case['dtype']]
    entries = n * case['kept'] * (size + 4)
    targets = 0 if not case['hard'] else n * (8 if case['target'] == 'labels' else 12)
    return {'bytes': 2 * size * n * classes + entries + targets, 'flops': (16 if case['hard'] else 8) * n * classes}


# ---- group norm ------------------------------------------------------------------------------------------------------

def _prepare_group(case, gen):
    shape = (case['batch'], case['height'], case['width'], case['channels'])
    dtype = DTYPES[case['dtype']]
    level = _randn(gen, shape[0], 1, 1, shape[3])  # what a convolution gives: channels with means and scales of their own
    x = _randn(gen, *shape).mul_(torch.exp(_randn(gen, 1, 1, 1, shape[3], scale=0.3))).add_(level).to(dtype).permute(0, 3, 1, 2)
    state = dict(op='group', x=x, groups=case['groups'], activation=None if case['activation'] == 'none' else case['activation'],
                 weight=(1 + _randn(gen, shape[3], scale=0.2)).to(dtype), bias=_randn(gen, shape[3], scale=0.2).to(dtype))
    if case['direction'] == 'both':
        state['dy'] = _randn(gen, *shape).to(dtype).permute(0, 3, 1, 2)
    return state


def _plain_group(s):
    x, groups, kind = s['x'], s['groups'], s['activation']
    n, channels, height, width = x.shape
    rows = x.permute(0, 2, 3, 1).reshape(n, height * width, groups, channels // groups).float()
    w, b = (s[k].float().view(groups, -1) for k in ('weight', 'bias'))
    mean = rows.mean((1, 3), keepdim=True)
    rows = rows - mean
    rstd = 1 / torch.sqrt((rows * rows).mean((1, 3), keepdim=True) + EPS)
    hat = rows * rstd
    a = hat * w + b

    def back(t):  # to the order of x
        return t.reshape(n, height, width, channels).to(x.dtype).permute(0, 3, 1, 2)

    if kind == 'silu':
        gate = 1 / (1 + torch.exp(-a))
        y, slope = a * gate, gate * (1 + a * (1 - gate))
    elif kind == 'gelu':
        gate = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        y, slope = a * gate, gate + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    else:
        y, slope = a, torch.ones_like(a)
    if 'dy' not in s:
        return {'y': back(y)}
    da = s['dy'].permute(0, 2, 3, 1).reshape(rows.shape).float() * slope
    dhat = da * w
    dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    return {'y': back(y), 'dx': back(dx), 'dweight': (da * hat).sum((0, 1)).view(-1).to(x.dtype), 'dbias': da.sum((0, 1)).view(-1).to(x.dtype)}


def _own_group(s):
    from ffcv_b200 import training
    how = dict(weight=s['weight'], bias=s['bias'], activation=s['activation'], eps=EPS)
    y, stats = training.group_norm_act_forward(s['x'], s['groups'], **how)
    if 'dy' not in s:
        return {'y': y}
    grads = training.group_norm_act_backward(s['dy'], s['x'], stats, s['groups'], **how)
    return {'y': y, 'dx': grads['x'], 'dweight': grads['weight'], 'dbias': grads['bias']}


def _exact_group(s):
    x, w, b = (s[k].double().requires_grad_('dy' in s) for k in ('x', 'weight', 'bias'))
    n, channels = x.shape[:2]
    flat = x.reshape(n, s['groups'], -1)
    var, mean = torch.var_mean(flat, 2, keepdim=True, correction=0)
    a = ((flat - mean) * torch.rsqrt(var + EPS)).view(x.shape) * w[:, None, None] + b[:, None, None]
    act = {None: lambda v: v, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}[s['activation']]
    y = act(a)
    if 'dy' not in s:
        return {'y': _last(y, s['x'])}
    y.backward(s['dy'].double())
    return {'y': _last(y.detach(), s['x']), 'dx': _last(x.grad, s['x']), 'dweight': w.grad, 'dbias': b.grad}


def _last(t, like):
    """A tensor in another one's order in memory."""
    return torch.empty_strided(like.shape, like.stride(), dtype=t.dtype, device=t.device).copy_(t)


def _work_group(case):
    values = case['batch'] * case['height'] * case['width'] * case['channels']
    both = case['direction'] == 'both'
    return {'bytes': SIZE[case['dtype']] * ((4 if both else 2) * values + (4 if both else 2) * case['channels']), 'flops': (40 if both else 15) * values}
