"""More refusals of the row operators and 8-bit products, and what their modules do without a kernel (no GPU)."""


def test_wait_test_arguments():
    import flb_native as nat
    assert nat.lib.flb_selftest_late_copy(16, 16, 8, 0, None) == 1 and nat.lib.flb_selftest_late_copy(16, 16, 16, 100001, None) == 1
    assert nat.lib.flb_selftest_late_copy(16, 24, 16, 0, None) == 3
    assert nat.lib.flb_int8_linear_wait_test(16, 64, None, 0, None, 16, 64, 16, None, 0, 16, 4, 8, 64, 2, 256, 1 << 30, 1, -2, 1, None) == 1
    assert nat.lib.flb_int8_linear_wait_test(16, 64, None, 0, None, 16, 64, 16, None, 0, 16, 4, 8, 64, 2, 256, 1 << 30, 1, 0, 0, None) == 1
