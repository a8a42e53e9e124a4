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
