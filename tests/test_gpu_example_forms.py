"""The example's other forms run: a convolutional stem, a head that makes its loss itself, a teacher's logits out of the data set; and their gradients."""
import importlib.util
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples', 'train_image_transformer.py')


@pytest.mark.parametrize('form', [['--stem', 'convolutions', '--head', 'whole'], ['--teacher', '4'], ['--stem', 'convolutions', '--teacher', '3']])
def test_forms_run(form):
    run = subprocess.run([sys.executable, EXAMPLE, '--epochs', '1', '--count', '256', '--batch', '64', '--layers', '2', *form], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    losses = json.loads(run.stdout.strip().splitlines()[-1])['losses']
    assert len(losses) == 1 and 0 < losses[0] < 20


def test_gradients_of_the_two_heads():
    """A whole head's loss and gradients are those of logits and the loss behind them, but for roundings: logits of 16 bits are off by 2^-9 of their size,
    gradients by a few of these."""
    import torch
    from ffcv_b200.training import MixupCrossEntropy
    spec = importlib.util.spec_from_file_location('example', EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    whole = example.ImageTransformer(50, 16, 64, 1, 2, 'convolutions', 'whole').cuda().bfloat16()
    parts = example.ImageTransformer(50, 16, 64, 1, 2, 'convolutions', 'logits').cuda().bfloat16()
    parts.load_state_dict(whole.state_dict())
    images = torch.randn(32, 3, 64, 64, device='cuda', dtype=torch.bfloat16)
    labels = torch.randint(50, (32,), device='cuda').float()
    mixed = torch.stack([labels, labels.roll(1), torch.rand(32, device='cuda')], 1)
    one, other = whole.head(whole.hidden(images), mixed), MixupCrossEntropy(label_smoothing=0.1)(parts(images), mixed)
    one.backward(), other.backward()
    assert abs(float(one.detach()) - float(other.detach())) < 0.02
    for (name, p), (_, q) in zip(whole.named_parameters(), parts.named_parameters()):
        assert (p.grad.float() - q.grad.float()).norm() <= 0.05 * q.grad.float().norm() + 1e-3, name
