"""Refusals of the RMS norm that need no GPU, and the mirror of its argument block."""
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
    from distributed_tensorflow_amd.ops import hip_ops
    lib = native.hip()
    assert lib.dtf_sizeof_rms_norm_args() == ctypes.sizeof(hip_ops.RmsNormArgs)
    a = hip_ops.RmsNormArgs()
    assert lib.dtf_rms_norm_fwd(ctypes.byref(a), None) == -22 and lib.dtf_rms_norm_fwd(None, None) == -22
    assert lib.dtf_rms_norm_bwd(ctypes.byref(a), None) == -22
    a.x = a.w = a.y = 64
    a.dim = 8
    for rows in (0, -1, 1 << 31):
        a.rows = rows
        assert lib.dtf_rms_norm_fwd(ctypes.byref(a), None) == -22
    a.rows, a.res = 1, 64  # a residual, and nowhere to write the sum
    assert lib.dtf_rms_norm_fwd(ctypes.byref(a), None) == -22
    assert lib.dtf_rms_norm_bwd_blocks(0, 8) == -22 and lib.dtf_rms_norm_bwd_blocks(3, 8) == 3
