"""gated_scan and gated_scan_step on sizes beyond one launch: a grid has less than 2^32 threads along an axis."""
import ctypes

import pytest
import torch


def test_grids_that_do_not_fit_are_refused_before_anything_is_launched():
    from t2fw_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 64)
    for B, T, D, dtype in ((1, 1 << 31, 64, 0), (1 << 24, 2000, 4, 1), (1 << 20, 4096, 64, 2), (3, 1 << 31, 64, 3)):
        assert lib.t2fw_gated_scan_forward(*(p,) * 7, B, T, D, None, dtype, 0, p, 1 << 62, None) == 3
        assert b"too many workgroups" in lib.t2fw_last_error()
        assert lib.t2fw_gated_scan_backward(*(p,) * 9, B, T, D, None, dtype, 0, p, 1 << 62, None) == 3
    for B, D, dtype in ((1 << 24, 2048, 1), (1 << 24, 1024, 0), (1 << 24, 512, 3)):
        assert lib.t2fw_gated_scan_step(*(p,) * 5, B, D, dtype, 0, None) == 3
        assert b"too many channels" in lib.t2fw_last_error()


@pytest.mark.gpu
def test_no_steps_of_more_channels_than_threads_of_a_launch():
    import t2fw_amd as t2
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    B, D = (1 << 16) + 3, 1 << 16
    state = torch.full((B, D), 3.0, device="cuda")
    none = torch.zeros(B, 0, D, device="cuda")
    with torch.no_grad():
        h, last = t2.gated_scan(none, none, state)
    assert h.shape == (B, 0, D) and torch.equal(last, state)
