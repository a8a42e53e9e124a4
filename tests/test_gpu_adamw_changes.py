"""The optimizer among other things a program does: graphs, other memory, networks that are loaded, copies."""
import copy
import math
import pickle

import pytest
import torch as ch

from test_gpu_adamw import HYPER, Formula, params_of, set_grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('stepped', [False, True])
def test_a_step_is_not_captured(stepped):
    """A replay would make the same step again and again; the capture goes on without it, and so does the optimizer."""
    from ffcv_b200.training import AdamW
    params, gen = params_of([(300,), (20, 30)], ch.float32)
    opt = AdamW(params, **HYPER)
    want = [Formula(p, HYPER['lr'], HYPER['betas'], HYPER['eps'], HYPER['weight_decay']) for p in params]

    def step():
        set_grads(params, gen)
        opt.step()
        for p, w in zip(params, want):
            w.step(p.grad)

    if stepped:
        step()
    set_grads(params, gen)
    x, called = ch.ones(4, device='cuda'), []
    ch.cuda.synchronize()
    graph = ch.cuda.CUDAGraph()
    with ch.cuda.graph(graph):
        y = x * 2
        with pytest.raises(RuntimeError, match='captured'):
            opt.step(lambda: called.append(1))
    assert not called and opt._steps.tolist() == [int(stepped)] * 2
    x.fill_(3.0)
    graph.replay()
    assert y.tolist() == [6.0] * 4
    step()
    for p, w in zip(params, want):
        w.check(opt, p, 20)


def test_the_library_does_not_take_a_step_into_a_graph():
    from ffcv_b200.training import AdamW
    from ffcv_b200.training import _native as N
    params, gen = params_of([(300,)], ch.float32)
    opt = AdamW(params, **HYPER)
    set_grads(params, gen)
    opt.step()
    before = params[0].detach().clone()
    ch.cuda.synchronize()
    graph, capturing = ch.cuda.CUDAGraph(), N.capturing
    N.capturing = lambda: False
    try:
        with ch.cuda.graph(graph):
            ch.empty(1, device='cuda').fill_(0.0)
            with pytest.raises(RuntimeError, match='cannot be captured'):
                opt.step()
    finally:
        N.capturing = capturing
    assert opt._steps.tolist() == [1]
    graph.replay()
    assert ch.equal(params[0].detach(), before)


@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16, ch.float16], ids=str)
def test_another_order_in_memory(dtype):
    """Moments and masters stay with their values when the network's memory format changes between steps."""
    from ffcv_b200.training import AdamW
    net = ch.nn.Sequential(ch.nn.Conv2d(5, 7, 3), ch.nn.Conv2d(7, 40, 3)).cuda().to(dtype)
    params, gen = list(net.parameters()), ch.Generator('cuda').manual_seed(0)
    opt = AdamW(params, **HYPER)
    want = [Formula(p, HYPER['lr'], HYPER['betas'], HYPER['eps'], HYPER['weight_decay']) for p in params]
    for step in range(5):
        if step == 2:
            net.to(memory_format=ch.channels_last)
            assert opt._params[0] is net[0].weight and net[0].weight.stride(1) == 1
        if step == 4:
            net.to(memory_format=ch.contiguous_format)
        set_grads(params, gen)
        opt.step()
        for p, w in zip(params, want):
            w.step(p.grad)
    for p, w in zip(params, want):
        w.check(opt, p, 50)


@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_another_order_with_moments_of_8_bits(dtype):
    """What the state stands for is rounded once more (2^-4 and 2^-3 of a value, or 2^-10 and 2^-17 of its block's largest), and codes and
    scales are such as the kernel makes: the next step goes on from them."""
    from ffcv_b200.training import AdamW
    gen = ch.Generator('cuda').manual_seed(1)
    p = ch.nn.Parameter(ch.randn((9, 70, 3, 5), generator=gen, device='cuda').to(dtype))
    opt = AdamW([p], **HYPER, state_bits=8)
    spread = ch.exp(ch.randn((9, 70, 1, 1), generator=gen, device='cuda'))
    for _ in range(3):
        p.grad = (ch.randn(p.shape, generator=gen, device='cuda') * spread).to(dtype)
        opt.step()

    def moments():
        out = []
        for k, name in enumerate(('exp_avg', 'exp_avg_sq')):
            codes = opt.state[p][name]
            flat = ch.as_strided(codes, (codes.numel(),), (1,)).float() * opt.state[p]['scales'][:, k].repeat_interleave(256)[:codes.numel()]
            out.append(ch.as_strided(flat, codes.shape, codes.stride()).contiguous())
        return out

    before = moments()
    p.data = p.data.to(memory_format=ch.channels_last)
    p.grad = None
    opt.step()
    for was, now, own, most in zip(before, moments(), (2.0 ** -4, 2.0 ** -3), (2.0 ** -10, 2.0 ** -17)):
        assert bool(((now - was).abs() <= own * was.abs() + most * was.abs().max()).all()) and ch.equal(now > 0, was > 0)
    assert ch.equal(ch.frexp(opt.scales)[0], ch.full_like(opt.scales, 0.5))  # powers of two
    was, g = moments(), (ch.randn(p.shape, generator=gen, device='cuda') * spread).to(dtype)
    p.grad = g
    opt.step()
    b1, b2 = HYPER['betas']
    # (a code is off by one place at most)
    for now, want, own, most in zip(moments(), (b1 * was[0] + (1 - b1) * g.float(), b2 * was[1] + (1 - b2) * g.float() ** 2), (2.0 ** -3, 2.0 ** -2), (2.0 ** -9, 2.0 ** -16)):
        assert bool(((now - want).abs() <= own * want.abs() + most * want.abs().max()).all())


@pytest.mark.parametrize('bits', [8, 32])
def test_parameters_that_are_no_longer_what_they_were(bits):
    """Refused on the host; nothing is launched, and the step is made once they are again."""
    from ffcv_b200.training import AdamW
    whole = ch.randn(8, 6, device='cuda')
    for new, kind in ((whole.cpu(), TypeError), (whole.bfloat16(), TypeError), (whole[:4], ValueError), (whole.view(6, 8), ValueError),
                      (ch.randn(8, 12, device='cuda')[:, ::2], ValueError)):
        p, other = ch.nn.Parameter(whole.clone()), ch.nn.Parameter(ch.randn(5, device='cuda'))
        opt = AdamW([p, other], **HYPER, state_bits=bits)
        other.grad = ch.randn(5, device='cuda')
        opt.step()
        before = other.detach().clone()
        p.data = new
        with pytest.raises(kind):
            opt.step()
        assert ch.equal(other.detach(), before) and opt._steps.tolist() == [0, 1]
        p.data = whole.clone()
        p.grad = ch.randn(8, 6, device='cuda')
        opt.step()
        assert opt._steps.tolist() == [1, 2] and not ch.equal(p.detach(), whole)


@pytest.mark.parametrize('bits', [8, 32])
def test_a_network_that_is_loaded_between_steps(bits):
    """Its 16-bit weights are what the next step is made on."""
    from ffcv_b200.training import AdamW
    net, gen = ch.nn.Linear(40, 30).cuda().bfloat16(), ch.Generator('cuda').manual_seed(2)
    opt = AdamW(net.parameters(), **HYPER, state_bits=bits)
    params = list(net.parameters())
    for step in range(4):
        if step in (0, 2):
            new = {k: ch.randn(t.shape, generator=gen, device='cuda').bfloat16() for k, t in net.state_dict().items()}
            net.load_state_dict(new)
        set_grads(params, gen)
        before = [p.detach().float().clone() for p in params]
        opt.step()
        for p, was in zip(params, before):  # a step is lr * wd of a weight and lr / sqrt(1 - b2) at most
            assert float((opt.state[p]['master'] - was).abs().max()) <= HYPER['lr'] * (0.1 * 6 + 10.0) + 2.0 ** -8 * 6
            assert ch.equal(p.detach(), opt.state[p]['master'].bfloat16())


@pytest.mark.parametrize('how', ['deepcopy', 'pickle'])
@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_copies_go_on_by_themselves(bits, dtype, how):
    from ffcv_b200.training import AdamW
    params, gen = params_of([(300,), (20, 30), (7,)], dtype)
    opt = AdamW(params, **HYPER, state_bits=bits, seed=4, max_grad_norm=1e3)
    for _ in range(3):
        set_grads(params, gen)
        opt.step()
    both = params, opt
    others, other = copy.deepcopy(both) if how == 'deepcopy' else pickle.loads(pickle.dumps(both))
    for _ in range(2):
        set_grads(params, gen)
        for p, q in zip(params, others):
            q.grad = p.grad.clone()
        opt.step()
        other.step()
        assert all(p is not q and ch.equal(p, q) for p, q in zip(params, others))
        for a, b in ((opt.exp_avg, other.exp_avg), (opt.exp_avg_sq, other.exp_avg_sq), (opt.master, other.master), (opt.scales, other.scales)):
            assert a is b is None or (a.data_ptr() != b.data_ptr() and ch.equal(a.view(ch.uint8), b.view(ch.uint8)))
        assert math.isclose(float(opt.grad_norm), float(other.grad_norm))


@pytest.mark.parametrize('dtype', [ch.bfloat16, ch.float16], ids=str)
@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('more', [0, 70, 1100])
def test_masters_follow_parameters(dtype, bits, more):
    """Against the rule in plain operations: tensors of all sizes, some at odd places, in more than one launch, some of them written to, with
    infinities and what is no number; the others' masters are not touched."""
    from ffcv_b200.training import AdamW
    gen = ch.Generator('cuda').manual_seed(3)
    r = lambda *s: ch.randn(s, generator=gen, device='cuda')  # noqa: E731
    flat = r(40000).to(dtype)
    params = [ch.nn.Parameter(r(*s).to(dtype)) for s in ((1,), (255,), (257,), (8192,), (8193,), (70, 301), (0,), (300000,))]
    params += [ch.nn.Parameter(flat[1:20002]), ch.nn.Parameter(flat[20004:20007]), ch.nn.Parameter(r(9, 40).to(dtype).t())]
    params += [ch.nn.Parameter(r(3 + i % 5).to(dtype)) for i in range(more)]
    opt = AdamW(params, **HYPER, state_bits=bits)
    for p in params:
        p.grad = r(*p.shape).to(dtype)
    opt.step()
    want = [opt.state[p]['master'].clone() for p in params]
    for i, p in enumerate(params):
        if i % 3 == 0 or i == 8:  # (cut out of one tensor, the two odd ones share a version; what has not been written stays all the same)
            new = p.detach().clone()
            change = ch.rand(p.shape, generator=gen, device='cuda') < 0.3
            new[change] = (r(*p.shape) * 4).to(dtype)[change]
            if p.numel() > 50:
                new.view(-1)[5:8] = ch.tensor([math.inf, -0.0, math.nan], device='cuda', dtype=dtype) if new.is_contiguous() else new.view(-1)[5:8]
            want[i] = ch.where(new == p.detach(), want[i], new.float())
            with ch.no_grad():
                p.copy_(new)
    values = [p.detach().clone() for p in params]
    for group in opt.param_groups:
        group['lr'] = 0.0
    padding = opt.master.clone()
    opt.step()
    for p, w, v in zip(params, want, values):
        kept = ~ch.isnan(w)
        assert ch.equal(ch.isnan(opt.state[p]['master']), ~kept) and ch.equal(opt.state[p]['master'][kept], w[kept])
        assert ch.equal(p.detach()[kept], v[kept])
    starts = opt._start.tolist() + [opt.master.numel()]
    for i, p in enumerate(params):  # behind a tensor's last value there are zeros
        assert not opt.master[starts[i] + p.numel():starts[i + 1]].any() and not padding[starts[i] + p.numel():starts[i + 1]].any()
    for p in params:  # behind autograd's back, and asked for
        p.data.clamp_(-0.5, 0.5)
    opt.masters_from_parameters()
    for p in params:
        master, finite = opt.state[p]['master'], ~ch.isnan(p.detach())
        assert ch.equal(master.to(dtype)[finite], p.detach()[finite])
