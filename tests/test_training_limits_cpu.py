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
