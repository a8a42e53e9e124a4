"""Group norm: statistics of samples without positions."""
import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('samples,channels,groups,sides', [(3, 8, 2, (0,)), (2, 32, 4, (0, 5)), (1, 6, 6, (4, 0))])
def test_statistics_of_nothing_are_no_numbers(samples, channels, groups, sides):
    from ffcv_b200.training import group_norm_act_backward, group_norm_act_forward
    x = torch.empty(samples, channels, *sides, device='cuda')
    w = torch.ones(channels, device='cuda')
    for _ in range(3):
        torch.full((1 << 20,), 7.0, device='cuda')  # (what was in the memory before)
        y, stats = group_norm_act_forward(x, groups, weight=w)
        assert y.shape == x.shape and stats.shape == (samples, groups, 2) and bool(stats.isnan().all())
        grads = group_norm_act_backward(y, x, stats, groups, weight=w)
        assert grads['x'].shape == x.shape and not grads['weight'].any()
