"""Refusals of the RMS norm that need no GPU."""
import ctypes

import pytest
import torch


def test_cpu_tensors_and_mismatched_arguments_are_refused():
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    x, w = torch.zeros(4, 8), torch.ones(8)
    for bad in (lambda: hip_ops.rms_norm_forward(x, w), lambda: hip_ops.rms_norm_e4m3(x, w), lambda: autograd.rms_norm(x, w),
                lambda: hip_ops.rms_norm_backward(x, x, torch.ones(4), w), lambda: autograd.RMSNorm(8)(x)):
        with pytest.raises(ValueError, match="CUDA"):
            bad()


def test_the_native_side_refuses_bad_blocks():
    from distributed_tensorflow_amd import native
    lib = native.hip()
    empty = ctypes.create_string_buffer(256)  # an argument block of zeros
    for fn in (lib.dtf_rms_norm_fwd, lib.dtf_rms_norm_bwd):
        fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
        assert fn(empty, None) == -22 and fn(None, None) == -22
    lib.dtf_rms_norm_bwd_blocks.argtypes = [ctypes.c_long, ctypes.c_int]
    assert lib.dtf_rms_norm_bwd_blocks(0, 8) == -22 and lib.dtf_rms_norm_bwd_blocks(3, 5000) == 3
