"""What the training kernels' sources have to hold to, whatever they compute."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'ffcv_b200', 'csrc')
SOURCES = ('cross_entropy.cu', 'norm_residual.cu', 'norm_forward.cu', 'norm_backward.cu', 'rotary.cu', 'adamw.cu')


def kernels(source):
    """Names and bodies of a file's kernels."""
    text = open(os.path.join(CSRC, source)).read()
    for found in re.finditer(r'__global__[^;{]*?(\w+)\([^;{]*\)\s*\{', text):
        depth, at = 1, found.end()
        while depth:
            depth += {'{': 1, '}': -1}.get(text[at], 0)
            at += 1
        yield found.group(1), text[found.end():at - 1]


@pytest.mark.parametrize('source', SOURCES)
def test_every_kernel_waits_itself_for_the_one_before(source):
    """Launched early, a kernel is promised to see what earlier kernels wrote only once it has waited itself: on every path, before it lets
    the next one begin, and before it uses an address that it was given."""
    found = list(kernels(source))
    assert found
    for name, body in found:
        lines = [line for line in body.split('\n') if line.strip()]
        waits = [k for k, line in enumerate(lines) if line == '    wait_for_previous();']
        assert len(waits) == 1 and body.count('wait_for_previous') == 1, name
        before = '\n'.join(lines[:waits[0]])
        assert 'let_next_begin' not in before and 'return' not in before and 'static_cast<const' not in before and 'reinterpret_cast' not in before, name
