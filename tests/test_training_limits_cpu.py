"""What the training calls refuse by their sizes, without a GPU: nothing is launched, whatever the addresses."""


def test_classes_that_32_bits_cannot_count():
    """A row's classes are counted in steps of up to 8192 behind the last one, in 32 bits; there are no rows here, so that nothing is read."""
    from ffcv_b200.training import _native as N

    def call(rows, classes):
        return N.lib.ffcvb_cross_entropy(N.CROSS_ENTROPY.pack(
            0, 0, 0, 0, 0, 0, 0, 0, rows, classes, classes, 1, classes, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0.0, 1.0), None)

    for classes in (0x7fff0000 + 1, 0x7fffff00, 0x7fffffff, 1 << 31, 1 << 40):
        assert call(0, classes) == -2 and b'bad size' in N.lib.ffcvb_training_error()
    assert call(0, 0x7fff0000) != -2 and call(1 << 28, 5) == -2


def test_masters_are_asked_for_with_whole_arguments():
    import numpy as np
    from ffcv_b200.training import _native as N
    numel, which = np.array([3], np.int64), b'\1' + b'\0' * 7

    def call(table=16, master=16, kind=2, n=1, numel_at=numel.ctypes.data, which=which):
        return N.lib.ffcvb_adamw_masters(N.ADAMW.pack(table, 16, 16, 0, master, 0, 0, 0, 0, kind, 32, n, 0.0), numel_at, which, None)

    assert N.lib.ffcvb_adamw_masters(None, None, None, None) == -2 and b'no arguments' in N.lib.ffcvb_training_error()
    for bad in (dict(table=0), dict(master=0), dict(kind=0), dict(kind=3), dict(n=-1), dict(numel_at=None), dict(which=None)):
        assert call(**bad) == -2
    assert call(n=0) == 0
