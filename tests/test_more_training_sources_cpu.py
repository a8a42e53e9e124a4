"""What the sources of the losses and the group norm have to hold to, as those of the other training kernels."""
import pytest
from test_training_sources_cpu import kernels, test_every_kernel_waits_itself_for_the_one_before as waits

SOURCES = ('linear_cross_entropy.cu', 'distillation.cu', 'group_norm.cu')


@pytest.mark.parametrize('source', SOURCES)
def test_every_kernel_waits_itself(source):
    waits(source)
    assert len(list(kernels(source))) >= {'distillation.cu': 1}.get(source, 6)


def test_symbols():
    import ctypes
    from ffcv_b200 import libffcv
    for name in ('ffcvb_linear_cross_entropy', 'ffcvb_linear_cross_entropy_workspace', 'ffcvb_distillation', 'ffcvb_group_norm', 'ffcvb_group_norm_backward',
                 'ffcvb_group_norm_workspace'):
        assert isinstance(getattr(libffcv.lib, name), ctypes._CFuncPtr)
