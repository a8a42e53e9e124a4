"""AdamW over many tensors: against the formula in 64 bits with 32-bit moments, bit for bit against the same
arithmetic in plain operations with 8-bit ones.

Tolerances: moments are two products and a sum: 2^-22 of the terms' size.  An update is a quotient of them, of size lr / (1 - b1^t)
times at most 1 / sqrt(1 - b2): off by 2^-20 of itself; the weight by 2^-23 of itself and that."""
import math

import numpy as np
import pytest
import torch as ch

pytestmark = pytest.mark.gpu

TYPES = [ch.float32, ch.bfloat16, ch.float16]
BLOCK = 256
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def params_of(shapes, dtype, seed=0):
    gen = ch.Generator('cuda').manual_seed(seed)
    return [ch.nn.Parameter(ch.randn(s, generator=gen, device='cuda').to(dtype)) for s in shapes], gen


def set_grads(params, gen, scale=1.0):
    for p in params:
        p.grad = (ch.randn(p.shape, generator=gen, device='cuda') * scale).to(p.dtype)


class Formula:
    """One tensor's state in 64 bits."""

    def __init__(self, p, lr, betas, eps, weight_decay):
        self.w, self.t = p.detach().double().clone(), 0
        self.m, self.v = ch.zeros_like(self.w), ch.zeros_like(self.w)
        self.lr, self.betas, self.eps, self.wd = lr, betas, eps, weight_decay

    def step(self, g, clip=1.0):
        self.t += 1
        b1, b2 = self.betas
        g = g.double() * clip
        self.m, self.v = b1 * self.m + (1 - b1) * g, b2 * self.v + (1 - b2) * g * g
        u = self.m / (1 - b1 ** self.t) / ((self.v / (1 - b2 ** self.t)).sqrt() + self.eps)
        self.w = self.w * (1 - self.lr * self.wd) - self.lr * u

    def check(self, opt, p, steps):
        s = opt.state[p]
        big_g = float(self.v.max().sqrt()) * 10 / math.sqrt(1 - self.betas[1]) if self.v.numel() else 0.0
        assert bool(((s['exp_avg'].double() - self.m).abs() <= steps * 2.0 ** -22 * big_g).all())
        assert bool(((s['exp_avg_sq'].double() - self.v).abs() <= steps * 2.0 ** -20 * self.v + 1e-30).all())
        w = s['master'] if 'master' in s else p.detach()
        room = steps * (2.0 ** -23 * self.w.abs() + 2.0 ** -18 * self.lr * 10) + 2.0 ** -23 * steps
        assert bool(((w.double() - self.w).abs() <= room).all()), float(((w.double() - self.w).abs() / room).max())
        if 'master' in s:
            assert ch.equal(p.detach(), s['master'].to(p.dtype))


SHAPES = [(1,), (3, 5), (255,), (256,), (257,), (64, 33), (8192,), (8193,), (70, 301), (0,), (2, 3, 3, 3), (40000,)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('clip', [None, 0.5, 1e6])
def test_32_bit_moments(dtype, clip):
    from ffcv_b200.training import AdamW
    params, gen = params_of(SHAPES, dtype)
    opt = AdamW([dict(params=params[:5]), dict(params=params[5:], weight_decay=0.0, lr=1e-2)], **HYPER, max_grad_norm=clip)
    want = [Formula(p, HYPER['lr'] if i < 5 else 1e-2, HYPER['betas'], HYPER['eps'], 0.1 if i < 5 else 0.0) for i, p in enumerate(params)]
    for step in range(4):
        set_grads(params, gen, 0.01 * 10 ** step)
        norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
        factor = 1.0 if clip is None else min(1.0, clip / (norm + 1e-6))
        opt.step()
        for w, p in zip(want, params):
            w.step(p.grad, factor)
        if clip is not None:
            assert abs(float(opt.grad_norm) - norm) < 1e-5 * norm
    for w, p in zip(want, params):
        w.check(opt, p, 40)


@pytest.mark.parametrize('count', [63, 64, 65, 1023, 1024, 1025, 2500])
def test_many_tensors_some_without_a_gradient(count):
    """More tensors than one launch takes, and more different step counts than one launch has room for."""
    from ffcv_b200.training import AdamW
    params, gen = params_of([(5 + i % 7,) for i in range(count)], ch.float32)
    opt = AdamW(params, **HYPER, max_grad_norm=1e9)
    want = [Formula(p, HYPER['lr'], HYPER['betas'], HYPER['eps'], HYPER['weight_decay']) for p in params]
    for step in range(30):
        set_grads(params, gen)
        for i, p in enumerate(params):  # tensor i begins to learn in step i mod 25
            if step < i % 25:
                p.grad = None
        opt.step()
        for w, p in zip(want, params):
            if p.grad is not None:
                w.step(p.grad)
    for i in range(0, count, 7):
        want[i].check(opt, params[i], 300)
    assert [opt.state_dict()['state'][i]['step'] for i in range(25)] == [30 - i for i in range(25)]


def test_memory_formats_alignment_and_moved_tensors():
    from ffcv_b200.training import AdamW
    gen = ch.Generator('cuda').manual_seed(2)
    r = lambda *s: ch.randn(s, generator=gen, device='cuda')  # noqa: E731
    flat = r(1000)
    params = [ch.nn.Parameter(r(8, 6, 5, 5).to(memory_format=ch.channels_last)), ch.nn.Parameter(r(30, 20).t()),
              ch.nn.Parameter(flat[1:401]), ch.nn.Parameter(flat[402:406]), ch.nn.Parameter(r(333))]
    opt = AdamW(params, **HYPER)
    want = [Formula(p, HYPER['lr'], HYPER['betas'], HYPER['eps'], HYPER['weight_decay']) for p in params]
    for step in range(5):
        for p in params:
            p.grad = r(*p.shape)  # (not always in the parameter's order)
        if step == 2:  # a parameter that was given other memory
            params[4].data = params[4].data.clone()
        if step == 3:
            params[4].grad = r(334)[1:]
        opt.step()
        for w, p in zip(want, params):
            w.step(p.grad)
    for w, p in zip(want, params):
        w.check(opt, p, 50)


def mix(x):
    x = (x * 0xE4C6EF2B) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x87EA99B3) & 0xFFFFFFFF
    return x ^ (x >> 16)


def rounded(v, noise, top, bias, dropped, dtype):
    """As the kernel rounds, in numpy's 32-bit arithmetic."""
    v = v.reshape(-1, BLOCK)
    e = np.maximum(np.abs(v).max(1).view(np.int32) >> 23, 1) - 127
    down = np.ldexp(np.float32(1), -e).astype(np.float32)[:, None]
    bits = ((np.abs(v) * down) * np.float32(2.0 ** (top - bias))).view(np.int32)
    code = (bits + noise.reshape(-1, BLOCK).astype(np.int32)) >> dropped
    if dtype == ch.float8_e5m2:
        code = np.maximum(code, v > 0)
    code = (code | ((v < 0) << 7)).astype(np.uint8)
    return ch.from_numpy(code.reshape(-1)).view(dtype), np.ldexp(np.float32(1), e - top).astype(np.float32)


class Eight:
    """The flat state of 8 bits in plain 32-bit operations on the CPU."""

    def __init__(self, opt):
        self.m, self.v, self.scales = opt.exp_avg.cpu(), opt.exp_avg_sq.cpu(), opt.scales.cpu()

    def step(self, g, b1, b2, seed, t):
        f = np.float32
        m = (self.m.float().view(-1, BLOCK) * self.scales[:, :1]).view(-1).numpy()
        v = (self.v.float().view(-1, BLOCK) * self.scales[:, 1:]).view(-1).numpy()
        m = m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * g) * f(1 - b2)
        key = mix(mix((seed + 1) & 0xFFFFFFFF) ^ t)
        noise = mix((np.arange(g.size, dtype=np.uint64) + np.uint64(key)) & np.uint64(0xFFFFFFFF))
        self.m, ms = rounded(m, (noise & np.uint64(0xFFFF)) << np.uint64(4), 7, 120, 20, ch.float8_e4m3fn)
        self.v, vs = rounded(v, (noise >> np.uint64(16)) << np.uint64(5), 14, 112, 21, ch.float8_e5m2)
        self.scales = ch.from_numpy(np.stack([ms, vs], 1))
        return m, v


def flat_of(opt, params, tensors):
    flat = np.zeros(opt.exp_avg.numel(), np.float32)
    for p, t, start in zip(params, tensors, opt._start):
        flat[start:start + p.numel()] = t.detach().float().cpu().numpy().reshape(-1)
    return flat


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_8_bit_moments(dtype):
    from ffcv_b200.training import AdamW
    params, gen = params_of(SHAPES, dtype, 3)
    opt = AdamW(params, **HYPER, state_bits=8, seed=5)
    b1, b2 = HYPER['betas']
    plain = Eight(opt)
    w = flat_of(opt, params, params).astype(np.float64)
    for t in range(1, 7):
        set_grads(params, gen, 10.0 ** -t)
        params[3].grad[7] = 0.0
        params[5].grad[::3] *= 1e-7  # values far below their block's largest
        params[8].grad.zero_() if t < 3 else None
        opt.step()
        m, v = plain.step(flat_of(opt, params, [p.grad for p in params]), b1, b2, 5, t)
        with np.errstate(invalid='ignore', divide='ignore'):
            u = m.astype(np.float64) / (1 - b1 ** t) / (np.sqrt(v.astype(np.float64) / (1 - b2 ** t)) + HYPER['eps'])
        w = w * (1 - HYPER['lr'] * HYPER['weight_decay']) - HYPER['lr'] * u
        assert ch.equal(opt.exp_avg.view(ch.uint8).cpu(), plain.m.view(ch.uint8))
        assert ch.equal(opt.exp_avg_sq.view(ch.uint8).cpu(), plain.v.view(ch.uint8))
        assert ch.equal(opt.scales.cpu(), plain.scales)
    masters = [opt.state[p]['master'] if 'master' in opt.state[p] else p for p in params]
    got = flat_of(opt, params, masters)
    assert np.all(np.abs(got - w) <= 6 * (2.0 ** -22 * np.abs(w) + 2.0 ** -18 * HYPER['lr'] * 10))
    for p in params:
        if 'master' in opt.state[p]:
            assert ch.equal(p.detach(), opt.state[p]['master'].to(dtype))


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_8_bit_moments_of_many_values(dtype):
    """As many as have their chunks worked on in turns, with tensors that end inside a turn, and a gradient at an odd place."""
    from ffcv_b200.training import AdamW
    shapes = [(1100, 2900), (7,), (1301, 1303), (8192,), (8193 + 255,), (2048 + 256,), (90001,), (6, 2048), (0,)]
    assert sum(math.prod(s) for s in shapes) > 148 * 4 * 8192
    params, gen = params_of(shapes, dtype, 6)
    opt = AdamW(params, **HYPER, state_bits=8, seed=11, max_grad_norm=1e9)
    b1, b2 = HYPER['betas']
    plain = Eight(opt)
    w = flat_of(opt, params, params).astype(np.float64)
    for t in range(1, 4):
        set_grads(params, gen, 10.0 ** -t)
        params[6].grad = ch.randn(90002, generator=gen, device='cuda').to(dtype)[1:]
        opt.step()
        m, v = plain.step(flat_of(opt, params, [p.grad for p in params]), b1, b2, 11, t)
        with np.errstate(invalid='ignore', divide='ignore'):
            u = m.astype(np.float64) / (1 - b1 ** t) / (np.sqrt(v.astype(np.float64) / (1 - b2 ** t)) + HYPER['eps'])
        w = w * (1 - HYPER['lr'] * HYPER['weight_decay']) - HYPER['lr'] * u
        assert ch.equal(opt.exp_avg.view(ch.uint8).cpu(), plain.m.view(ch.uint8))
        assert ch.equal(opt.exp_avg_sq.view(ch.uint8).cpu(), plain.v.view(ch.uint8))
        assert ch.equal(opt.scales.cpu(), plain.scales)
    masters = [opt.state[p]['master'] if 'master' in opt.state[p] else p for p in params]
    got = flat_of(opt, params, masters)
    assert np.all(np.abs(got - w) <= 3 * (2.0 ** -22 * np.abs(w) + 2.0 ** -18 * HYPER['lr'] * 10))
    for p in params:
        if 'master' in opt.state[p]:
            assert ch.equal(p.detach(), opt.state[p]['master'].to(dtype))


def test_8_bit_moments_follow_their_averages():
    """Thousands of steps of a constant gradient: the second moment comes to g^2, which it would not if values were rounded
    to the nearest, and a value's mean over many equal ones is right.  A step moves a value by up to (1 - b2) g^2 and rounding by a
    quarter of it with the chance that keeps the mean: a variance of at most 0.25 * 0.001 per step over 500 steps, so the mean of 4096
    values is within 5 * sqrt(0.125 / 4096) = 3 %."""
    from ffcv_b200.training import AdamW
    p = ch.nn.Parameter(ch.zeros(4096, device='cuda'))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    p.grad = ch.full_like(p, 0.3)
    p.grad[::256] = 3.0  # the blocks' largest
    for _ in range(6000):
        opt.step()
    v = opt.exp_avg_sq.float() * opt.scales[:, 1].repeat_interleave(256)
    m = opt.exp_avg.float() * opt.scales[:, 0].repeat_interleave(256)
    rest = ch.ones(4096, dtype=ch.bool, device='cuda')
    rest[::256] = False
    assert abs(float(v[rest].mean()) / 0.09 - 1) < 0.03 + math.exp(-6)
    assert abs(float(m[rest].mean()) / 0.3 - 1) < 0.02
    assert float(v[rest].std()) / 0.09 < 0.5


@pytest.mark.parametrize('bits', [8, 32])
def test_steps_that_are_not_made(bits):
    """With a bound, a gradient that is not finite changes nothing; without one, it goes where arithmetic takes it."""
    from ffcv_b200.training import AdamW
    for bad in (math.inf, math.nan):
        params, gen = params_of([(300,), (20, 30)], ch.float32)
        opt = AdamW(params, **HYPER, state_bits=bits, max_grad_norm=1.0)
        set_grads(params, gen)
        opt.step()
        before = [t.clone() for t in (*params, opt.exp_avg.view(ch.uint8), opt.exp_avg_sq.view(ch.uint8))]
        params[0].grad[5] = bad
        opt.step()
        assert not math.isfinite(float(opt.grad_norm))
        assert all(ch.equal(a, b) for a, b in zip(before, (*params, opt.exp_avg.view(ch.uint8), opt.exp_avg_sq.view(ch.uint8))))
        free = AdamW(params, **HYPER, state_bits=bits)
        free.step()
        assert not bool(ch.isfinite(params[0][5])) or bits == 8
        free.step()
        assert not bool(ch.isfinite(params[0][5])) and bool(ch.isfinite(params[0][256:]).all()) and bool(ch.isfinite(params[1]).all())


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_state_dict(bits, dtype, tmp_path):
    from ffcv_b200.training import AdamW
    shapes = [(300,), (20, 30), (7,)]

    def make():
        params, _ = params_of(shapes, dtype, 6)
        return params, AdamW([dict(params=params[:1]), dict(params=params[1:], lr=1e-2)], **HYPER, state_bits=bits, seed=9)

    a, opt_a = make()
    gen = ch.Generator('cuda').manual_seed(8)
    for step in range(3):
        set_grads(a, gen)
        if step == 1:
            a[2].grad = None
        opt_a.step()
    opt_a.param_groups[0]['lr'] = 1e-4
    ch.save(dict(opt=opt_a.state_dict(), params=a), tmp_path / 'state.pt')
    saved = ch.load(tmp_path / 'state.pt', weights_only=False)
    b, opt_b = make()
    for p, q in zip(b, saved['params']):
        p.data.copy_(q.data)
    opt_b.load_state_dict(saved['opt'])
    assert opt_b.param_groups[0]['lr'] == 1e-4 and opt_b._steps.tolist() == [3, 3, 2]
    for p, q in zip(a, b):
        p.grad = ch.randn(p.shape, generator=gen, device='cuda').to(dtype)
        q.grad = p.grad.clone()
    opt_a.step()
    opt_b.step()
    assert all(ch.equal(p, q) for p, q in zip(a, b)) and ch.equal(opt_a.exp_avg_sq.view(ch.uint8), opt_b.exp_avg_sq.view(ch.uint8))
    other = AdamW(make()[0], state_bits=bits)
    with pytest.raises(ValueError):
        other.load_state_dict(opt_a.state_dict())


def test_goes_on_from_torch_and_with_its_schedulers():
    from ffcv_b200.training import AdamW
    a, gen = params_of([(100, 3), (50,)], ch.float32)
    b = [ch.nn.Parameter(p.detach().clone()) for p in a]
    theirs = ch.optim.AdamW(a, **HYPER)
    for _ in range(3):
        set_grads(a, gen)
        theirs.step()
    ours = AdamW(b, **HYPER)
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    ours.load_state_dict(theirs.state_dict())
    plans = [ch.optim.lr_scheduler.CosineAnnealingLR(o, 10) for o in (theirs, ours)]
    for _ in range(5):
        set_grads(a, gen)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        for o, plan in zip((theirs, ours), plans):
            o.step()
            plan.step()
        assert theirs.param_groups[0]['lr'] == ours.param_groups[0]['lr']
    for p, q in zip(a, b):
        assert ch.allclose(p, q, rtol=1e-5, atol=1e-6)


def test_groups_added_later_keep_the_state():
    from ffcv_b200.training import AdamW
    for bits, dtype in ((32, ch.bfloat16), (8, ch.float32)):
        params, gen = params_of([(300,), (20, 30), (513,)], dtype)
        opt = AdamW(params[:2], **HYPER, state_bits=bits)
        set_grads(params, gen)
        opt.step()
        before = [opt.state[params[1]][k].view(ch.uint8).clone() for k in ('exp_avg', 'exp_avg_sq')]
        opt.add_param_group(dict(params=[params[2]], lr=1.0))
        assert all(ch.equal(opt.state[params[1]][k].view(ch.uint8), v) for k, v in zip(('exp_avg', 'exp_avg_sq'), before))
        assert opt._steps.tolist() == [1, 1, 0]
        loss = opt.step(lambda: 7)
        assert loss == 7 and opt._steps.tolist() == [2, 2, 1]


def test_autograd_sees_the_step():
    """A backward pass that needs a weight as it was before the step says so."""
    from ffcv_b200.training import AdamW
    p = ch.nn.Parameter(ch.ones(8, device='cuda'))
    opt = AdamW([p])
    x = ch.ones(8, device='cuda', requires_grad=True)
    y = (x * p).sum()
    p.grad = ch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


def test_learns_in_mixed_precision():
    """Least squares: with either state the loss falls to a hundredth."""
    from ffcv_b200.training import AdamW
    for bits in (32, 8):
        ch.manual_seed(0)
        net = ch.nn.Sequential(ch.nn.Linear(16, 64), ch.nn.GELU(), ch.nn.Linear(64, 4)).cuda().bfloat16()
        x, y = ch.randn(256, 16, device='cuda').bfloat16(), None
        y = ch.stack([x[:, 0] * x[:, 1], x[:, 2], x[:, 3] ** 2, x[:, 4] - x[:, 5]], 1).float()
        opt = AdamW(net.parameters(), lr=1e-2, weight_decay=0.0, state_bits=bits, max_grad_norm=1.0)
        losses = []
        for _ in range(600):
            opt.zero_grad()
            loss = (net(x).float() - y).square().mean()
            loss.backward()
            opt.step()
            losses.append(loss.detach())
        assert float(losses[-1]) < 0.02 * float(losses[0])


def test_refusals():
    from ffcv_b200.training import AdamW
    p = ch.nn.Parameter(ch.zeros(4, device='cuda'))
    for kw, kind in ((dict(state_bits=16), ValueError), (dict(max_grad_norm=0.0), ValueError), (dict(lr=-1.0), ValueError), (dict(betas=(1.0, 0.9)), ValueError),
                     (dict(eps=-1.0), ValueError), (dict(weight_decay=-0.1), ValueError)):
        with pytest.raises(kind):
            AdamW([p], **kw)
    for bad, kind in ((ch.nn.Parameter(ch.zeros(4)), TypeError), (ch.nn.Parameter(ch.zeros(4, device='cuda', dtype=ch.float64)), TypeError),
                      (ch.nn.Parameter(ch.zeros(4, device='cuda').half()), TypeError), (ch.nn.Parameter(ch.zeros(8, device='cuda')[::2]), ValueError)):
        with pytest.raises(kind):
            AdamW([p, bad])
    opt = AdamW([p])
    opt.param_groups[0]['lr'] = -1.0
    p.grad = ch.zeros_like(p)
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[0]['lr'] = 1.0
    with pytest.raises(ValueError):
        opt.load_state_dict(AdamW([p], state_bits=8).state_dict())
