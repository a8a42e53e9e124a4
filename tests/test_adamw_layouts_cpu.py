"""Parameters that are other tensors than when the optimizer was made, on the host: the step's arithmetic is the formula in numpy.

Tolerances.  32 bits: the stand-in computes in 64 bits and rounds once per step, as the formula here does not: 2^-23 of the weights and
of the update per step.  8 bits: e4m3 and e5m2 are off by 2^-4 and 2^-3 of a moment per rounding to the nearest, or by 2^-10 and 2^-17 of
their block's largest."""
import math

import pytest
import torch as ch

from adamw_host import on_the_host

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


class Formula:
    def __init__(self, p):
        self.w, self.t = p.detach().double().clone(), 0
        self.m, self.v = ch.zeros_like(self.w), ch.zeros_like(self.w)

    def step(self, g):
        self.t += 1
        b1, b2 = HYPER['betas']
        g = g.double()
        self.m, self.v = b1 * self.m + (1 - b1) * g, b2 * self.v + (1 - b2) * g * g
        u = self.m / (1 - b1 ** self.t) / ((self.v / (1 - b2 ** self.t)).sqrt() + HYPER['eps'])
        self.w = self.w * (1 - HYPER['lr'] * HYPER['weight_decay']) - HYPER['lr'] * u

    def near(self, w):
        return bool(((w.double() - self.w).abs() <= self.t * 2.0 ** -23 * (self.w.abs() + 1)).all())


def same(p, changed):
    """A parameter with its values in another order in memory, or in other memory."""
    if changed == 'channels_last':
        p.data = p.data.to(memory_format=ch.channels_last)
    elif changed == 'transposed':
        p.data = p.data.transpose(0, 1).contiguous().transpose(0, 1)
    elif changed == 'back and forth':
        p.data = p.data.to(memory_format=ch.channels_last)
        p.data = p.data.contiguous()
    else:
        p.data = p.data.clone()


@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
@pytest.mark.parametrize('changed', ['channels_last', 'transposed', 'back and forth', 'cloned'])
@pytest.mark.parametrize('later', [False, True])
def test_another_order_in_memory(monkeypatch, dtype, changed, later):
    """Moments and masters stay with their values, whenever the order changes, and with a group that is added after it."""
    AdamW, lib = on_the_host(monkeypatch)
    gen = ch.Generator().manual_seed(0)
    params = [ch.nn.Parameter(ch.randn(s, generator=gen).to(dtype)) for s in ((300,), (4, 6, 5, 5), (3, 2, 9, 11))]
    opt = AdamW(params[:2] if later else params, **HYPER)
    want = [Formula(p) for p in params]
    for step in range(5):
        if step == 2:
            same(params[1], changed)
            if later:
                opt.add_param_group(dict(params=[params[2]], lr=HYPER['lr']))
        for p, w in zip(params, want):
            if p is params[2] and later and step < 2:
                continue
            p.grad = ch.randn(p.shape, generator=gen).to(dtype)
            w.step(p.grad)
        opt.step()
    for p, w in zip(params, want):
        assert w.near(opt.state[p]['master'] if dtype != ch.float32 else p.detach())
        if dtype != ch.float32:
            assert ch.equal(p.detach(), opt.state[p]['master'].to(dtype))


def test_the_order_of_values_at_the_same_address(monkeypatch):
    """``p.data = p.data.t()``: other values of the same memory, which the address does not show."""
    AdamW, lib = on_the_host(monkeypatch)
    p = ch.nn.Parameter(ch.randn(7, 7))
    opt, g = AdamW([p], **HYPER), ch.randn(7, 7)
    p.grad = g
    opt.step()
    m = opt.state[p]['exp_avg'].clone()
    p.grad = None
    p.data = p.data.t()
    want = Formula(p)  # (the state stays with rows and columns as the parameter has them now)
    want.t, want.m, want.v = 1, m.double(), opt.state[p]['exp_avg_sq'].double().clone()
    p.grad = ch.randn(7, 7)
    want.step(p.grad)
    opt.step()
    assert want.near(p.detach())


@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_another_order_with_moments_of_8_bits(monkeypatch, dtype):
    """The moments are rounded once more, each to a number of its own size."""
    AdamW, lib = on_the_host(monkeypatch)
    gen = ch.Generator().manual_seed(1)
    p = ch.nn.Parameter(ch.randn((6, 30, 5, 3), generator=gen).to(dtype))
    opt = AdamW([p], **HYPER, state_bits=8)
    spread = ch.exp(ch.randn(p.shape, generator=gen))
    for _ in range(3):
        p.grad = (ch.randn(p.shape, generator=gen) * spread).to(dtype)
        opt.step()

    def moments():
        out = []
        for k, name in enumerate(('exp_avg', 'exp_avg_sq')):
            codes = opt.state[p][name]
            flat = ch.as_strided(codes, (codes.numel(),), (1,)).float() * opt.state[p]['scales'][:, k].repeat_interleave(256)[:codes.numel()]
            out.append(ch.as_strided(flat, codes.shape, codes.stride()).contiguous())
        return out

    before, weights = moments(), (opt.state[p]['master'] if dtype != ch.float32 else p.detach()).contiguous().clone()
    p.data = p.data.to(memory_format=ch.channels_last)
    p.grad = None
    opt.step()  # (no gradient: nothing but the order changes)
    assert opt.state[p]['exp_avg'].stride() == p.stride()
    for was, now, own, most in zip(before, moments(), (2.0 ** -4, 2.0 ** -3), (2.0 ** -10, 2.0 ** -17)):
        assert bool(((now - was).abs() <= own * was.abs() + most * was.abs().max()).all())
        assert bool(((now > 0) == (was > 0)).all())
    now = opt.state[p]['master'] if dtype != ch.float32 else p.detach()
    assert ch.equal(now, weights) and ch.equal(p.detach().contiguous(), weights.to(dtype))


@pytest.mark.parametrize('bits', [8, 32])
def test_parameters_that_are_no_longer_what_they_were(monkeypatch, bits):
    """Fewer or more values, other shapes and types, gaps: refused before anything is done, and before a group is added."""
    AdamW, lib = on_the_host(monkeypatch)
    whole = ch.randn(8, 6)
    for new, kind in ((whole[:4], ValueError), (ch.randn(9, 6), ValueError), (whole.view(6, 8), ValueError), (whole.view(48), ValueError),
                      (ch.randn(8, 12)[:, ::2], ValueError), (ch.randn(6, 1).t().expand(8, 6), ValueError), (whole.bfloat16(), TypeError), (whole.half(), TypeError)):
        p, other = ch.nn.Parameter(whole.clone()), ch.nn.Parameter(ch.randn(5))
        opt = AdamW([p, other], **HYPER, state_bits=bits)
        other.grad, p.grad = ch.randn(5), ch.randn(8, 6)
        opt.step()
        steps, before = lib.steps, other.detach().clone()
        p.grad = None
        p.data = new
        with pytest.raises(kind):
            opt.step()
        with pytest.raises(kind):
            opt.add_param_group(dict(params=[ch.nn.Parameter(ch.randn(3))]))
        assert lib.steps == steps and ch.equal(other.detach(), before) and len(opt.param_groups) == 1 and opt._steps.tolist() == [1, 1]
        p.data = whole.clone()
        opt.step()
        assert lib.steps == steps + 1


def test_gradients_that_are_no_longer_what_they_were(monkeypatch):
    """A gradient whose memory was exchanged for less of it."""
    AdamW, lib = on_the_host(monkeypatch)
    p = ch.nn.Parameter(ch.randn(8, 6))
    opt = AdamW([p], **HYPER)
    for new, kind in ((ch.randn(4, 6), ValueError), (ch.randn(8, 1).expand(8, 6), None), (ch.randn(8, 6).half(), TypeError), (ch.randn(6, 8).t(), None)):
        p.grad = ch.randn(8, 6)
        opt.step()
        steps = lib.steps
        p.grad.data = new
        if kind is None:
            want, t = Formula(p), opt._steps[0]
            want.t, want.m, want.v = int(t), *(opt.state[p][k].double().clone() for k in ('exp_avg', 'exp_avg_sq'))
            want.step(new)
            opt.step()
            assert lib.steps == steps + 1 and want.near(p.detach())
        else:
            with pytest.raises(kind):
                opt.step()
            assert lib.steps == steps


def test_frozen_between_steps_and_in_other_modes(monkeypatch):
    """What does not change the memory does not disturb a step."""
    AdamW, lib = on_the_host(monkeypatch)
    p = ch.nn.Parameter(ch.randn(40))
    opt, want = AdamW([p], **HYPER), None
    want = Formula(p)
    for step in range(6):
        p.grad = ch.randn(40)
        p.requires_grad_(step % 2 == 0)
        want.step(p.grad)
        if step == 3:
            with ch.autocast('cpu'):
                opt.step()
        else:
            opt.step()
    assert lib.steps == 6 and want.near(p.detach()) and math.isclose(want.t, 6)


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_state_saved_in_another_order(monkeypatch, bits, dtype):
    """A network that was trained with its channels last goes on with them first: moments in 8 bits have a scale per block of
    neighbours in memory, which are others then."""
    AdamW, lib = on_the_host(monkeypatch)
    gen = ch.Generator().manual_seed(2)
    p = ch.nn.Parameter(ch.randn((5, 30, 4, 3), generator=gen).to(dtype).to(memory_format=ch.channels_last))
    opt = AdamW([p], **HYPER, state_bits=bits)
    spread = ch.exp(2 * ch.randn((5, 30, 1, 1), generator=gen))  # (of another size in every channel)
    for _ in range(3):
        p.grad = (ch.randn(p.shape, generator=gen) * spread).to(dtype)
        opt.step()
    q = ch.nn.Parameter(p.detach().contiguous())
    other = AdamW([q], **HYPER, state_bits=bits)
    other.load_state_dict(opt.state_dict())
    for k, (name, own, most) in enumerate((('exp_avg', 2.0 ** -4, 2.0 ** -10), ('exp_avg_sq', 2.0 ** -3, 2.0 ** -17))):
        values = []
        for o, t in ((opt, p), (other, q)):
            v, shape = o.state[t][name], t.shape
            assert v.stride() == t.stride()
            if bits == 8:
                flat = ch.as_strided(v, (v.numel(),), (1,)).float() * o.state[t]['scales'][:, k].repeat_interleave(256)[:v.numel()]
                v = ch.as_strided(flat, shape, t.stride())
            values.append(v)
        was, now = values
        if bits == 32:
            assert ch.equal(was, now)
        else:
            assert bool(((now - was).abs() <= own * was.abs() + most * was.abs().max()).all())
    if dtype != ch.float32:
        assert ch.equal(opt.state[p]['master'], other.state[q]['master'])


def test_gradients_are_read_where_they_lie(monkeypatch):
    """Also where dimensions of one value have other strides, as those of a convolution of 1 x 1 in another memory format; only another
    order of values is copied, and sparse ones are refused."""
    AdamW, lib = on_the_host(monkeypatch)
    params = [ch.nn.Parameter(ch.randn(s)) for s in ((8, 4, 1, 1), (5, 1), (6, 7))]
    opt, want = AdamW(params, **HYPER), [Formula(p) for p in params]
    for step in range(3):
        for p, w in zip(params, want):
            p.grad = ch.randn(p.shape)
            w.step(p.grad)
        params[0].grad = params[0].grad.to(memory_format=ch.channels_last)
        params[1].grad = ch.as_strided(params[1].grad, (5, 1), (1, 9))
        if step == 2:
            params[2].grad = params[2].grad.t().contiguous().t()
        opt.step()
        same = [a == p.grad.data_ptr() for a, p in zip(lib.grads, params)]
        assert same == [True, True, step < 2] and (opt._grad_layouts is not None) == (step < 2)
    assert all(w.near(p.detach()) for w, p in zip(want, params))
    params[2].grad = ch.randn(6, 7).to_sparse()
    with pytest.raises(TypeError, match='dense'):
        opt.step()
    assert lib.steps == 3
