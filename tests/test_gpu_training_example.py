"""The loader and the training operators together, as the example runs them: the loss of a set whose classes differ by colour
falls to what mixing and smoothing of labels leave of it, with either state."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize('bits', [8, 32])
def test_image_transformer_learns(bits):
    run = subprocess.run([sys.executable, os.path.join(ROOT, 'examples', 'train_image_transformer.py'), '--epochs', '4', '--count', '1024',
                          '--batch', '64', '--layers', '2', '--state-bits', str(bits)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    losses = json.loads(run.stdout.strip().splitlines()[-1])['losses']
    # ten classes: 2.30 at the start; smoothing by 0.1 and mixing with Beta(0.2, 0.2) leave about 0.8
    assert losses[0] < 2.6 and losses[-1] < 1.6 and losses[-1] < losses[0] - 0.3, losses
