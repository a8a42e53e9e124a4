"""Group norm: statistics of samples without positions, and those that were kept elsewhere."""
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


@pytest.mark.parametrize('sides', [(6, 7), (170, 171)])
@pytest.mark.parametrize('offset', [0, 1, 2, 3])
def test_statistics_kept_in_another_tensor(sides, offset):
    from ffcv_b200.training import group_norm_act_backward, group_norm_act_forward
    x, dy = (torch.randn(2, *sides, 32, device='cuda').movedim(-1, 1) for _ in range(2))
    _, stats = group_norm_act_forward(x, 4, activation='silu')
    kept = torch.zeros(stats.numel() + offset, device='cuda')[offset:].view(stats.shape)
    kept.copy_(stats)
    assert kept.data_ptr() % 8 == offset % 2 * 4
    want, got = (group_norm_act_backward(dy, x, s, 4, activation='silu')['x'] for s in (stats, kept))
    assert torch.equal(got, want)
