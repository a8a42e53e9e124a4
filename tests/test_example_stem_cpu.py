"""The example's convolutional stem gives a token for each patch."""
import importlib.util
import os

import pytest
import torch

EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples', 'train_image_transformer.py')


@pytest.mark.parametrize('patch', [1, 2, 3, 4, 6, 7, 8, 10, 12, 14, 16, 24, 32])
def test_a_token_for_each_patch(patch, monkeypatch):
    from ffcv_b200 import training
    spec = importlib.util.spec_from_file_location('example', EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    monkeypatch.setattr(training, 'GroupNormAct', lambda *how: torch.nn.Identity())  # (no sizes change there)
    tokens = example.Stem(patch, 16)(torch.zeros(1, 3, 3 * patch, 5 * patch))
    assert tokens.shape == (1, 15, 16)
