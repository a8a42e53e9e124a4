"""Calls from several threads of a program on one GPU."""
import threading

import pytest
import torch as ch

pytestmark = pytest.mark.gpu


def side_by_side(calls, times):
    """Every call `times` times in a thread of its own, all at once; what they raised."""
    raised, start = [], threading.Barrier(len(calls))

    def work(call):
        start.wait()
        try:
            for _ in range(times):
                call()
        except Exception as e:  # noqa: BLE001
            raised.append(e)

    threads = [threading.Thread(target=work, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ch.cuda.synchronize()
    return raised


def test_rows_of_different_widths():
    """One kernel has rows of many widths, each of which needs another amount of shared memory; what a call may have is not lowered by
    one beside it."""
    from ffcv_b200.training import norm_residual_backward, norm_residual_forward
    calls, checks = [], []
    for width in (4096, 2048, 1024, 3136):
        x, h, dy, dz = (ch.randn(2, 4, width, device='cuda') for _ in range(4))
        y, z, stats = norm_residual_forward(x, h)
        want = norm_residual_backward(dy, dz, x, h, stats)
        calls.append(lambda x=x, h=h, dy=dy, dz=dz, stats=stats: (norm_residual_forward(x, h), norm_residual_backward(dy, dz, x, h, stats)))
        checks.append((calls[-1], want))
    assert not side_by_side(calls, 3000)
    assert all(ch.equal(call()[1][k], want[k]) for call, want in checks for k in want)


def test_losses_of_different_classes():
    from ffcv_b200.training import cross_entropy_with_grad
    calls = []
    for classes in (18000, 11000, 14000, 12500):
        x, y = ch.randn(300, classes, device='cuda'), ch.randint(classes, (300,), device='cuda')
        calls.append(lambda x=x, y=y: cross_entropy_with_grad(x, y))
    assert not side_by_side(calls, 3000)
