"""The optimizer's state as it is kept, saved, loaded and copied, on the host: a step is the formula in numpy."""
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
