"""Statistics that the norm's backward pass is given: kept in the middle of another tensor, or not those of the call."""
import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu


def made(rows=70, width=96):
    from ffcv_b200.training import norm_residual_forward
    x, h, dz = (torch.randn(rows, width, device='cuda') for _ in range(3))
    return x, h, dz, norm_residual_forward(x, h)[2]


@pytest.mark.parametrize('offset', range(5))
def test_kept_in_another_tensor(offset):
    from ffcv_b200.training import norm_residual_backward
    x, h, dz, stats = made()
    kept = torch.zeros(stats.numel() + offset, device='cuda')[offset:]
    kept.copy_(stats)
    assert kept.data_ptr() % 16 == offset % 4 * 4
    assert torch.equal(norm_residual_backward(None, dz, x, h, kept)['x'], norm_residual_backward(None, dz, x, h, stats)['x'])


def test_others_are_refused():
    from ffcv_b200.training import norm_residual_backward
    x, h, dz, stats = made()
    for bad in (stats[:-4], stats.double(), stats.cpu(), stats.view(-1, 4), torch.stack([stats, stats], 1)[:, 0], None):
        with pytest.raises(ValueError, match='stats'):
            norm_residual_backward(None, dz, x, h, bad)
