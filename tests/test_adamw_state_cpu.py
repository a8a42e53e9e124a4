"""The optimizer's state as it is kept, saved, loaded and copied, on the host: a step is the formula in numpy."""
import copy
import pickle

import pytest
import torch as ch

from adamw_host import on_the_host

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def params_of(dtype, seed=0):
    gen = ch.Generator().manual_seed(seed)
    return [ch.nn.Parameter(ch.randn(s, generator=gen).to(dtype)) for s in ((300,), (20, 30), (7,))], gen


def set_grads(params, gen):
    for p in params:
        p.grad = ch.randn(p.shape, generator=gen).to(p.dtype)


def bytes_of(opt):
    return [t.contiguous().view(-1).view(ch.uint8).clone() for t in (opt.exp_avg, opt.exp_avg_sq, opt.scales, opt.master) if t is not None]


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_a_parameter_without_saved_state_begins_anew(monkeypatch, bits, dtype):
    """Loaded into an optimizer that has made steps of its own: as into a new one, whose masters are the parameters."""
    AdamW, lib = on_the_host(monkeypatch)
    a, gen = params_of(dtype)
    source = AdamW(a, **HYPER, state_bits=bits)
    set_grads(a, gen)
    source.step()
    saved = source.state_dict()
    for i, entry in ((1, {}), (2, None)):  # (as of parameters that had no gradient yet)
        if entry is None:
            del saved['state'][i]
        else:
            saved['state'][i] = entry
    used, fresh = [], []
    for into, steps in ((used, 3), (fresh, 0)):
        params, _ = params_of(dtype, 5)
        opt = AdamW(params, **HYPER, state_bits=bits)
        for _ in range(steps):
            set_grads(params, gen)
            opt.step()
        for p, q in zip(params, a):
            with ch.no_grad():
                p.copy_(q)
        opt.load_state_dict(saved)
        into.extend([opt, params])
    assert all(ch.equal(x, y) for x, y in zip(bytes_of(used[0]), bytes_of(fresh[0])))
    assert used[0]._steps.tolist() == fresh[0]._steps.tolist() == [1, 0, 0]
    set_grads(used[1], gen)
    for p, q in zip(used[1], fresh[1]):
        q.grad = p.grad.clone()
    for opt, _ in (used, fresh):
        opt.step()
    assert all(ch.equal(p, q) for p, q in zip(used[1], fresh[1]))


def test_what_does_not_fit_changes_nothing(monkeypatch):
    AdamW, lib = on_the_host(monkeypatch)
    params, gen = params_of(ch.bfloat16)
    opt = AdamW(params, **HYPER)
    set_grads(params, gen)
    opt.step()
    for spoil in (lambda s: s['state'][2].update(exp_avg=ch.zeros(8)), lambda s: s['state'][2].update(exp_avg_sq=ch.zeros(7).half()),
                  lambda s: s['param_groups'][0].update(lr=-1.0)):
        other, _ = params_of(ch.bfloat16, 9)
        saved = AdamW(other, lr=0.5).state_dict()
        spoil(saved)
        before = bytes_of(opt)
        with pytest.raises(ValueError):
            opt.load_state_dict(saved)
        assert all(ch.equal(x, y) for x, y in zip(before, bytes_of(opt)))
        assert opt.param_groups[0]['lr'] == HYPER['lr'] and opt._steps.tolist() == [1, 1, 1]


def write_in_place(p, new):
    with ch.no_grad():
        p.copy_(new)


def load_network(p, new):
    net = ch.nn.Module()
    net.p = p
    net.load_state_dict(dict(p=new))


def other_memory(p, new):
    p.data = new.clone()


def through_detach(p, new):
    p.detach().copy_(new)


@pytest.mark.parametrize('write', [write_in_place, load_network, other_memory, through_detach], ids=lambda f: f.__name__)
@pytest.mark.parametrize('dtype', [ch.bfloat16, ch.float16], ids=str)
@pytest.mark.parametrize('steps', [0, 2])
@pytest.mark.parametrize('bits', [8, 32])
def test_masters_follow_what_is_written(monkeypatch, write, dtype, steps, bits):
    """Before the first step and between steps: the next step is made on the new values.  Values that were not changed keep the digits that
    only their masters have."""
    AdamW, lib = on_the_host(monkeypatch)
    params, gen = params_of(dtype)
    opt = AdamW(params, **HYPER, state_bits=bits)
    for _ in range(steps):
        set_grads(params, gen)
        opt.step()
    new = params[1].detach().clone()
    new[3:9] = ch.randn((6, 30), generator=gen).to(dtype)
    new[4, 2], new[5, 3] = 0.0, float('inf')
    want = opt.state[params[1]]['master'].clone()
    want[3:9] = ch.where(new[3:9] == params[1].detach()[3:9], want[3:9], new[3:9].float())
    rest = [opt.state[p]['master'].clone() for p in (params[0], params[2])]
    write(params[1], new)
    for group in opt.param_groups:
        group['lr'] = 0.0  # a step of no size: the masters stay as they are when it begins
    set_grads(params, gen)
    opt.step()
    assert ch.equal(opt.state[params[1]]['master'], want) and ch.equal(params[1].detach(), new)
    assert all(ch.equal(opt.state[p]['master'], r) for p, r in zip((params[0], params[2]), rest))
    if steps:
        assert not ch.equal(want[:3], new[:3].float())


def test_masters_of_parameters_that_are_clamped_behind_autograds_back(monkeypatch):
    AdamW, lib = on_the_host(monkeypatch)
    params, gen = params_of(ch.bfloat16)
    opt = AdamW(params, **HYPER)
    set_grads(params, gen)
    opt.step()
    for p in params:
        p.data.clamp_(-0.5, 0.5)
    opt.masters_from_parameters()
    for p in params:
        master = opt.state[p]['master']
        assert ch.equal(master.to(p.dtype), p.detach()) and float(master.abs().max()) <= 0.5 + 2.0 ** -9
    plain, _ = params_of(ch.float32)
    AdamW(plain).masters_from_parameters()  # (there are none)


def test_loaded_masters_give_way_to_other_weights(monkeypatch):
    """A saved optimizer's masters belong to its weights; other weights that are there when it is loaded stay."""
    AdamW, lib = on_the_host(monkeypatch)
    a, gen = params_of(ch.bfloat16)
    opt = AdamW(a, **dict(HYPER, lr=0.0))
    set_grads(a, gen)
    opt.step()
    saved = opt.state_dict()
    b, _ = params_of(ch.bfloat16, 7)
    with ch.no_grad():
        b[0].copy_(a[0])
    before = [p.detach().clone() for p in b]
    other = AdamW(b, **HYPER)
    other.load_state_dict(saved)
    set_grads(b, gen)
    other.step()
    assert ch.equal(other.state[b[0]]['master'], saved['state'][0]['master'])
    assert all(ch.equal(p.detach(), w) for p, w in zip(b, before))


def test_a_parameter_without_a_gradient_keeps_its_version(monkeypatch):
    """A backward pass that needs it goes on; one that needs a parameter of the step does not."""
    AdamW, lib = on_the_host(monkeypatch)
    a, b = (ch.nn.Parameter(ch.ones(8)) for _ in range(2))
    opt = AdamW([a, b], **HYPER)
    x = ch.ones(8, requires_grad=True)
    needs_a, needs_b = (x * a).sum(), (x * b).sum()
    a.grad = ch.ones(8)
    versions = a._version, b._version
    opt.step()
    assert a._version > versions[0] and b._version == versions[1]
    needs_b.backward()
    assert ch.equal(x.grad, ch.ones(8))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        needs_a.backward()


def test_groups_without_parameters(monkeypatch):
    """A network without vectors, say, whose group comes first, in between, last, or alone."""
    AdamW, lib = on_the_host(monkeypatch)
    params, gen = params_of(ch.bfloat16)
    plain = [ch.nn.Parameter(p.detach().clone()) for p in params]
    opt = AdamW([dict(params=[]), dict(params=params[:2]), dict(params=[], lr=1.0), dict(params=params[2:]), dict(params=[])], **HYPER)
    want = AdamW(plain, **HYPER)
    for _ in range(2):
        set_grads(params, gen)
        for p, q in zip(params, plain):
            q.grad = p.grad.clone()
        opt.step()
        want.step()
    assert all(ch.equal(p, q) for p, q in zip(params, plain))
    opt.load_state_dict(opt.state_dict())
    empty = AdamW([dict(params=[])], **HYPER)
    assert empty.step(lambda: 3) == 3
    empty.load_state_dict(empty.state_dict())
    empty.masters_from_parameters()
    empty.add_param_group(dict(params=params))
    set_grads(params, gen)
    empty.step()
    assert empty._steps.tolist() == [1, 1, 1]


@pytest.mark.parametrize('how', ['deepcopy', 'pickle', 'copy.copy'])
@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
def test_copies_go_on_by_themselves(monkeypatch, bits, dtype, how):
    """A copy of a network and its optimizer makes the steps that they would, on state of its own."""
    AdamW, lib = on_the_host(monkeypatch)
    params, gen = params_of(dtype)
    opt = AdamW([dict(params=params[:2]), dict(params=params[2:], lr=1e-2)], **HYPER, state_bits=bits, seed=4)
    for step in range(3):
        set_grads(params, gen)
        params[1].grad = None if step == 1 else params[1].grad
        opt.step()
    if how == 'copy.copy':  # (of the optimizer alone: the same parameters)
        other = copy.copy(opt)
        before = bytes_of(opt)
        other.step()
        assert other.param_groups[0]['params'][0] is params[0] and all(ch.equal(x, y) for x, y in zip(before, bytes_of(opt)))
        assert opt._steps.tolist() == [3, 2, 3] and opt.state[params[0]]['exp_avg'].data_ptr() == opt.exp_avg.data_ptr()
        return
    both = params, opt
    others, other = copy.deepcopy(both) if how == 'deepcopy' else pickle.loads(pickle.dumps(both))
    assert type(other) is AdamW and (other.state_bits, other.seed, other._steps.tolist()) == (bits, 4, [3, 2, 3])
    assert all(p is not q and p is r for p, q, r in zip(others, params, other._params))
    assert all(ch.equal(x, y) for x, y in zip(bytes_of(opt), bytes_of(other)))
    for _ in range(2):
        set_grads(params, gen)
        for p, q in zip(params, others):
            q.grad = p.grad.clone()
        before = bytes_of(other)
        opt.step()
        assert all(ch.equal(x, y) for x, y in zip(before, bytes_of(other)))
        other.step()
        assert all(ch.equal(p, q) for p, q in zip(params, others)) and all(ch.equal(x, y) for x, y in zip(bytes_of(opt), bytes_of(other)))
    other.load_state_dict(opt.state_dict())
    other.add_param_group(dict(params=[ch.nn.Parameter(ch.ones(5, dtype=dtype))]))
    assert opt.state_dict()['state'][1]['step'] == 4
