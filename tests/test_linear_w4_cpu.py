"""The 4-bit weights' format (on the CPU), and refusals of the product that need no GPU."""
import ctypes

import pytest
import torch

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


@pytest.mark.parametrize("K,N", [(1, 1), (128, 16), (129, 17), (300, 40), (32, 100)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantized_weights_are_the_nearest_values(K, N, group, dtype):
    from distributed_tensorflow_amd.ops import hip_ops
    w = torch.randn(K, N, generator=torch.Generator().manual_seed(K + N)).to(dtype)
    wq, scales = hip_ops.quantize_w4(w, group)
    assert wq.shape == (-(-N // 16), -(-K // 128), 64, 16) and scales.shape == (-(-N // 16), -(-K // 128) * 128 // group, 16)
    back = hip_ops.dequantize_w4(wq, scales, K, N)
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64)
    for k in range(0, K, max(1, K // 40)):  # straight from the documented layout
        for n in range(N):
            byte = int(wq[n // 16, k // 128, 16 * (k % 32 // 8) + n % 16, 4 * (k % 128 // 32) + k % 8 // 2])
            s = float(scales[n // 16, k // group, n % 16])
            top = float(w[k // group * group:(k // group + 1) * group, n].abs().max())
            assert abs(s - top / 6) <= top / 6 * 2.0 ** -8
            value = float(table[byte >> 4 if k % 2 else byte & 15]) * s
            assert value == float(back[k, n])
            # no other value of the scaled table is nearer, up to the rounding of w / s
            assert abs(float(w[k, n]) - value) <= float((table * s - float(w[k, n])).abs().min()) + 1e-6 * top
    full = hip_ops.dequantize_w4(wq, scales, -(-K // 128) * 128, -(-N // 16) * 16)
    assert not full[K:].any() and not full[:, N:].any()


def test_ties_go_to_the_even_code_and_zeros_stay():
    from distributed_tensorflow_amd.ops import hip_ops
    w = torch.zeros(32, 2)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    w[:7, 0], w[7, 0], w[8:15, 0] = torch.tensor(ties), 6.0, -torch.tensor(ties)
    wq, scales = hip_ops.quantize_w4(w, 32)
    back = hip_ops.dequantize_w4(wq, scales, 32, 2)
    assert back[:7, 0].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0] and back[8:15, 0].tolist() == [-0.0, -1.0, -1.0, -2.0, -2.0, -4.0, -4.0]
    assert not back[:, 1].any() and float(scales[0, 0, 1]) == 0
    tiny = hip_ops.dequantize_w4(*hip_ops.quantize_w4(torch.full((32, 1), 1e-45), 32), 32, 1)
    assert not tiny.any()


def test_refusals():
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    w = torch.randn(64, 32)
    for bad in (lambda: hip_ops.quantize_w4(w, 16), lambda: hip_ops.quantize_w4(w.double()), lambda: hip_ops.quantize_w4(w[0]),
                lambda: hip_ops.quantize_w4(w[:0]), lambda: hip_ops.quantize_w4(torch.full((4, 4), float("inf")))):
        with pytest.raises(ValueError):
            bad()
    wq, scales = hip_ops.quantize_w4(w)
    for bad in (lambda: hip_ops.dequantize_w4(wq, scales, 64, 33), lambda: hip_ops.dequantize_w4(wq, scales, 129, 32),
                lambda: hip_ops.dequantize_w4(wq, scales.float(), 64, 32), lambda: hip_ops.dequantize_w4(wq, scales[:1], 64, 32),
                lambda: hip_ops.dequantize_w4(wq[:, :, :32], scales, 64, 32), lambda: hip_ops.linear_w4(torch.zeros(1, 64), wq, scales, 32)):
        with pytest.raises(ValueError):
            bad()
    layer = autograd.LinearW4.from_linear(autograd.Linear(64, 32))
    with pytest.raises(ValueError, match="CUDA"):
        layer(torch.zeros(1, 64))
    with pytest.raises(ValueError, match="group"):
        autograd.LinearW4(64, 32, group=48)
    again = autograd.LinearW4(64, 32)
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again.wq, layer.wq) and torch.equal(again.scales.view(torch.int16), layer.scales.view(torch.int16))


def test_the_native_side_refuses_bad_blocks():
    from distributed_tensorflow_amd import native
    fn = native.hip().dtf_linear_w4
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert fn(None, None) == -22 and fn(ctypes.create_string_buffer(256), None) == -22  # nothing, and an argument block of zeros


def test_no_tile_of_columns_that_holds_no_row_is_chosen():
    """16 columns hold 16 rows, of float32 (three columns a row) 5; a further tile of them only for rows that the ones before do not hold.
    262144 outputs and their neighbours took a second one for a single row."""
    from distributed_tensorflow_amd import native
    fn = native.hip().dtf_linear_w4_tiles
    fn.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    assert fn(0, 1, 1, 0) == -22 and fn(1, 1, 1, 3) == -22 and fn(1, 0, 1, 0) == -22 and fn(1, 1, 0, 0) == -22
    widths = {1, 16, 17, 209000, 262144, 524288, (1 << 31) - 17} | {int(16 * 1.11 ** i) + i % 3 for i in range(150)}
    several = 0
    for xtype, parts in ((0, 3), (1, 1), (2, 1)):
        for rows in list(range(1, 36)) + [64, 1000, 327675]:
            for k in (1, 4096, 8192, 16384):
                for n in widths:
                    c, r = divmod(fn(rows, n, k, xtype), 16)
                    assert 1 <= c <= (3 if xtype == 0 else 2) and (1 if c == 1 else 2) <= r <= 4
                    assert c == 1 or rows > (c - 1) * 16 // parts, (rows, n, k, xtype, c, r)
                    several += c > 1
    assert several > 1000


def test_a_launch_stays_below_two_to_the_32_threads():
    """More are cut off without an error: 800 M outputs of 512 k (206 GB of weights) took 2^32 and more."""
    from distributed_tensorflow_amd import native
    tiles, waves = native.hip().dtf_linear_w4_tiles, native.hip().dtf_linear_w4_waves
    for fn in (tiles, waves):
        fn.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    assert waves(0, 1, 1, 0) == -22 and waves(1, 1, 1, 3) == -22
    for xtype in (0, 1, 2):
        for rows in (1, 2, 5, 6, 16, 17, 33, 327675):
            for k in (1, 128, 129, 512, 2048, 16384):
                for n in (1, 2048, 1 << 20, 805306368, 805306369, 900000000, 1 << 30, (1 << 31) - 18):
                    r = tiles(rows, n, k, xtype) % 16
                    groups, w = -(-(-(-n // 16)) // r), waves(rows, n, k, xtype)
                    assert 1 <= w <= min(12, -(-k // 128)) and groups * 64 * w < 1 << 32, (xtype, rows, k, n, r, w)
    # where the limit is far, as many as the sizes ask for
    assert waves(1, 2048, 16384, 1) == 12 and waves(1, 8192, 8192, 1) == 8 and waves(16, 16384, 16384, 0) == 4 and waves(3, 100, 300, 1) == 3


def test_a_layers_buffers_keep_their_types_through_casts_of_the_model():
    """wq, scales and bias are a format: a model's float(), half() or to(bfloat16) turned scales and bias into types that the kernel refuses."""
    from distributed_tensorflow_amd.ops import autograd
    layer = autograd.LinearW4.from_linear(autograd.Linear(130, 20), 32)
    want = {k: t.clone() for k, t in layer.state_dict().items()}
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), layer)
    for cast in (lambda m: m.float(), lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu"),
                 lambda m: m.float()):
        cast(model)
        assert list(layer.state_dict()) == list(want)
        for k, t in layer.state_dict().items():
            assert t.dtype == want[k].dtype and torch.equal(t.view(torch.uint8), want[k].view(torch.uint8)), k
    assert model[0].weight.dtype == torch.float32  # the last cast
    meta = model.to("meta")[1]
    assert all(t.is_meta and t.dtype == want[k].dtype for k, t in meta.state_dict().items())
