"""csrc/hip/linear_w4.hip through ops.hip_ops, against float64 products with the weights that the codes stand for."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F, B, E = torch.float32, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24


def _weights(K, N, group, seed=0):
    from distributed_tensorflow_amd.ops import hip_ops
    gen = torch.Generator("cuda").manual_seed(seed)
    w = torch.randn(K, N, generator=gen, device="cuda") * torch.exp(torch.randn(1, N, generator=gen, device="cuda"))
    wq, scales = hip_ops.quantize_w4(w, group)
    return wq, scales, hip_ops.dequantize_w4(wq, scales, K, N).double()


def _rows(M, K, dtype, seed=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=gen, device="cuda") * torch.exp(2 * torch.randn(M, 1, generator=gen, device="cuda"))
    if dtype != E:
        return x.to(dtype), None
    scale = x.abs().amax(1) / 448
    return (x / scale[:, None]).to(E), scale


def check(y, x, scale, w, bias, relu):
    """Products of bf16 parts are exact in fp32.  A sum of K of them, its groups' and waves' partial sums: no more than K + 100 additions of
    U each on the magnitudes (three parts of an fp32 row: within 1.01 of its own), then scale, bias and the result's type."""
    x = x.double() if scale is None else x.double() * scale.double()[:, None]
    want, size = x @ w, x.abs() @ w.abs()
    K = x.shape[1]
    off = size * (3 * K + 100) * U
    if bias is not None:
        want, off = want + bias.double(), off + U * (want.abs() + bias.double().abs()) * 2
    if relu:
        want = want.clamp(min=0)
    off = off + want.abs() * (2.0 ** -8 if y.dtype == B else U) + 1e-37
    worst = ((y.double() - want).abs() / off).max()
    assert bool(worst <= 1), float(worst)


# (rows, K, N): one element; tails of k and of outputs; one k tile and many; one, two and four tiles of columns; rows behind the last chunk
SHAPES = [(1, 1, 1), (1, 128, 16), (1, 2048, 1008), (2, 130, 33), (3, 127, 5), (5, 3136, 1025), (6, 96, 40), (10, 256, 48), (11, 264, 16), (16, 512, 64),
          (17, 1000, 31), (32, 1024, 16), (33, 72, 100), (64, 640, 200), (65, 256, 17), (150, 136, 20), (3, 2, 20), (4, 9, 17), (2, 15, 3), (16, 141, 16), (5, 2047, 40), (1, 16384, 8200), (16, 4096, 8208)]


@pytest.mark.parametrize("dtype", [F, B, E])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_products(M, K, N, group, dtype):
    from distributed_tensorflow_amd.ops import hip_ops
    wq, scales, w = _weights(K, N, group)
    x, scale = _rows(M, K, dtype)
    bias = torch.randn(N, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    y = hip_ops.linear_w4(x, wq, scales, N, bias=bias, x_scale=scale)
    check(y, x, scale, w, bias, False)
    assert torch.equal(y, hip_ops.linear_w4(x, wq, scales, N, bias=bias, x_scale=scale))  # a fixed order of the sums
    check(hip_ops.linear_w4(x, wq, scales, N, relu=True, x_scale=scale, out_dtype=B), x, scale, w, None, True)


# two and three tiles of columns a wave (more rows than one tile holds, outputs or rows enough to fill the chip), each with one to four tiles of
# outputs; twelve waves for a long k: fewer k than a tile, fewer tiles of k than waves, a tail; all columns taken, a last pass of one row, an odd number of output tiles
@pytest.mark.parametrize("dtype", [F, B, E])
@pytest.mark.parametrize("M,K,N,group", [(16, 100, 8200, 32), (12, 300, 16390, 64), (6, 515, 16400, 128), (10, 1000, 16384, 32), (17, 64, 16385, 64),
                                         (32, 777, 16390, 32), (1025, 129, 520, 32), (1030, 512, 500, 128), (257, 1001, 514, 64), (353, 260, 1030, 128), (12300, 130, 9, 32),
                                         (16, 140, 11000, 64), (32, 8300, 11000, 32), (7, 200, 9700, 32), (40, 100, 4700, 64), (5000, 70, 20, 64),
                                         (17, 128, 12352, 64), (17, 130, 18490, 32), (33, 100, 13700, 128), (11, 200, 8190, 64), (21, 390, 13700, 32), (3000, 128, 32, 128),
                                         (3, 8100, 100, 64), (16, 9001, 40, 128), (37, 16384, 17, 32)])
def test_several_tiles_of_columns(M, K, N, group, dtype):
    test_products(M, K, N, group, dtype)


# fp32 rows are cut into three parts: a NaN or an infinity reaches its own row alone, in a whole tile of k and in the last one, and a NaN whose
# bits all lie in the lower half stays one; the largest and the smallest finite values are summed exactly
@pytest.mark.parametrize("M,K,N", [(3, 300, 40), (16, 300, 8200), (6, 300, 16400)])
def test_fp32_values_at_the_ends_of_the_range(M, K, N):
    from distributed_tensorflow_amd.ops import hip_ops
    wq, scales, w = _weights(K, N, 32)
    x, _ = _rows(M, K, F)
    clean = hip_ops.linear_w4(x, wq, scales, N)
    used = w.abs().sum(1) != 0
    assert bool(used[7]) and bool(used[290])
    for k in (7, 290):
        for bits in (0x7f800000, 0xff800000, 0x7f800001, 0x7fc00000):
            z = x.clone()
            z.view(torch.int32)[1, k] = bits - (1 << 32) if bits >> 31 else bits
            y = hip_ops.linear_w4(z, wq, scales, N)
            hit = w[k] != 0
            assert bool(y[1, hit].isfinite().logical_not().all())
            assert torch.equal(y[1].isnan()[hit], torch.full_like(hit, bits & 0x7fffff != 0)[hit])
            rest = torch.arange(M, device="cuda") != 1
            assert torch.equal(y[rest], clean[rest])
    for v in (torch.finfo(F).max / 2 ** 20, 2.0 ** -100):
        z = torch.zeros_like(x)
        z[:, 7] = v
        y = hip_ops.linear_w4(z, wq, scales, N).double()
        want = z.double() @ w
        assert bool(((y - want).abs() <= 8 * U * want.abs()).all())


@pytest.mark.parametrize("dtype", [F, B, E])
@pytest.mark.parametrize("K", [256, 257, 264])
def test_strides_alignment_and_leading_dimensions(K, dtype):
    from distributed_tensorflow_amd.ops import hip_ops
    wq, scales, w = _weights(K, 40, 32)
    wide, scale = _rows(7, K + 50, dtype)
    for lo in (0, 1, 2, 8, 16):
        x = wide[:, lo:lo + K]
        check(hip_ops.linear_w4(x, wq, scales, 40, x_scale=scale), x, scale, w, None, False)
    t = wide[:, :K].t().contiguous().t()  # elements of a row apart from one another
    check(hip_ops.linear_w4(t, wq, scales, 40, x_scale=scale), t, scale, w, None, False)
    y = hip_ops.linear_w4(wide[:6, :K].reshape(2, 3, K), wq, scales, 40, x_scale=None if scale is None else scale[:6])
    assert y.shape == (2, 3, 40)
    check(y.reshape(6, 40), wide[:6, :K], None if scale is None else scale[:6], w, None, False)
    one = hip_ops.linear_w4(wide[0, :K].contiguous(), wq, scales, 40, x_scale=None if scale is None else scale[:1])
    assert one.shape == (40,) and torch.equal(one, hip_ops.linear_w4(wide[:1, :K], wq, scales, 40, x_scale=None if scale is None else scale[:1])[0])
    if dtype != E:  # one row for all, and a scale that other types may have
        e = wide[:1, :K].expand(5, K)
        s = torch.rand(5, device="cuda")
        check(hip_ops.linear_w4(e, wq, scales, 40, x_scale=s), e, s, w, None, False)


def test_float32_rows_lose_nothing_to_the_matrix_instructions_type():
    """A single weight of 1: the output is x itself, all 24 bits of it, far down the range of exponents."""
    from distributed_tensorflow_amd.ops import hip_ops
    w = torch.zeros(64, 16)
    w[5, 3] = 6.0
    wq, scales = (t.cuda() for t in hip_ops.quantize_w4(w, 32))
    gen = torch.Generator("cuda").manual_seed(0)
    for e in (0, 100, -60, -90):
        x = torch.zeros(5, 64, device="cuda")
        x[:, 5] = torch.randn(5, generator=gen, device="cuda") * 2.0 ** e
        y = hip_ops.linear_w4(x, wq, scales, 16)
        assert torch.equal(y[:, 3].double(), (x[:, 5].double() * 6).float().double())


@pytest.mark.parametrize("dtype", [F, B])
def test_infinities_and_nan_stay_in_their_rows(dtype):
    from distributed_tensorflow_amd.ops import hip_ops
    wq, scales, w = _weights(200, 20, 64)
    w4 = w.float()
    assert bool((w4 != 0).any())
    x, _ = _rows(5, 200, dtype)
    x[1, 7], x[2, 199], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[4] = 0
    y = hip_ops.linear_w4(x, wq, scales, 20)
    check(y[:1], x[:1], None, w, None, False)
    assert bool(torch.isnan(y[2]).all()) and not y[4].any()
    for row, k, sign in ((1, 7, 1), (3, 0, -1)):
        want = w4[k] * sign * float("inf")  # a weight of zero gives NaN
        assert torch.equal(torch.isnan(want), torch.isnan(y[row])) and torch.equal(want[w4[k] != 0], y[row][w4[k] != 0])
    relu = hip_ops.linear_w4(x, wq, scales, 20, relu=True)
    assert bool(torch.isnan(relu[2]).all())
    if dtype == F:  # a NaN whose payload lies in the low bits alone
        z = torch.zeros(1, 200, device="cuda")
        z.view(torch.int32)[0, 3] = 0x7F800001
        assert bool(torch.isnan(hip_ops.linear_w4(z, wq, scales, 20)).all())


def test_layers_capture_and_another_stream():
    from distributed_tensorflow_amd.ops import autograd
    layer = autograd.Linear(256, 100, relu=True).cuda()
    q = autograd.LinearW4.from_linear(layer, 32)
    from distributed_tensorflow_amd.ops import hip_ops
    w = hip_ops.dequantize_w4(q.wq, q.scales, 256, 100).double()
    x = _rows(3, 256, F)[0]
    check(q(x), x, None, w, layer.bias.detach(), True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = q(x)
    for i in range(4):
        x.copy_(_rows(3, 256, F, seed=i + 5)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, q(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = q(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)


def test_weights_behind_two_to_the_32_bytes():
    from distributed_tensorflow_amd.ops import hip_ops
    K, N = 65600, 140001
    kt, nt = -(-K // 128), -(-N // 16)
    gen = torch.Generator("cuda").manual_seed(0)
    wq = torch.randint(0, 256, (nt, kt, 64, 16), generator=gen, device="cuda", dtype=torch.uint8)
    scales = torch.rand(nt, kt * 4, 16, generator=gen, device="cuda").to(B)
    assert wq.numel() > 1 << 32
    x, _ = _rows(2, K, B)
    y = hip_ops.linear_w4(x, wq, scales, N)
    for lo, hi in ((0, 2), (nt - 2, nt)):  # the first and the last outputs
        w = hip_ops.dequantize_w4(wq[lo:hi], scales[lo:hi], K, 32).double()[:, :min(N, hi * 16) - lo * 16]
        check(y[:, lo * 16:hi * 16], x, None, w, None, False)


def test_e4m3_nan_and_gradients_that_are_not_taken():
    from distributed_tensorflow_amd.ops import hip_ops
    w = torch.randn(64, 32, device="cuda", requires_grad=True)
    wq, scales = hip_ops.quantize_w4(w)
    assert not scales.requires_grad and not hip_ops.dequantize_w4(wq, scales, 64, 32).requires_grad
    x = torch.ones(2, 64, device="cuda")
    x[1, 3] = float("nan")
    y = hip_ops.linear_w4(x.to(E), wq, scales, 32, x_scale=torch.ones(2, device="cuda"))
    assert bool(torch.isfinite(y[0]).all()) and bool(torch.isnan(y[1]).all())
    y = hip_ops.linear_w4(x[:1].to(E), wq, scales, 32, x_scale=torch.zeros(1, device="cuda"), bias=torch.ones(32, device="cuda"))
    assert bool((y == 1).all())


def test_empty_batches_and_refusals():
    from distributed_tensorflow_amd.ops import hip_ops
    wq, scales, _ = _weights(64, 32, 64)
    x = torch.zeros(2, 64, device="cuda")
    assert hip_ops.linear_w4(x[:0], wq, scales, 32).shape == (0, 32)
    for bad in (lambda: hip_ops.linear_w4(x.half(), wq, scales, 32), lambda: hip_ops.linear_w4(x.to(E), wq, scales, 32),
                lambda: hip_ops.linear_w4(torch.zeros(2, 129, device="cuda"), wq, scales, 32), lambda: hip_ops.linear_w4(x, wq, scales, 33),
                lambda: hip_ops.linear_w4(x, wq, scales, 16), lambda: hip_ops.linear_w4(x, wq.cpu(), scales.cpu(), 32),
                lambda: hip_ops.linear_w4(x, wq, scales, 32, bias=torch.zeros(31, device="cuda")),
                lambda: hip_ops.linear_w4(x, wq, scales, 32, bias=torch.zeros(32, device="cuda", dtype=B)),
                lambda: hip_ops.linear_w4(x, wq, scales, 32, x_scale=torch.zeros(1, device="cuda")),
                lambda: hip_ops.linear_w4(x, wq, scales, 32, out_dtype=torch.float16),
                lambda: hip_ops.linear_w4(x[:, :0], wq, scales, 32),
                lambda: hip_ops.linear_w4(x[:1].expand(65535 * 5 + 1, 64), wq, scales, 32)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("which", ["x", "bias", "x_scale"])
def test_operands_that_require_a_gradient_make_the_backward_pass_raise(which):
    """The values are those of any call; a loss that goes through the layer is refused instead of losing this branch's gradient."""
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    wq, scales, w = _weights(200, 40, 64)
    x, _ = _rows(3, 200, F)
    ops = {"x": x, "bias": torch.ones(40, device="cuda"), "x_scale": torch.ones(3, device="cuda")}
    want = hip_ops.linear_w4(ops["x"], wq, scales, 40, bias=ops["bias"], x_scale=ops["x_scale"])
    leaf = ops[which].requires_grad_()
    run = lambda: hip_ops.linear_w4(ops["x"], wq, scales, 40, bias=ops["bias"], x_scale=ops["x_scale"])  # noqa: E731
    y = run()
    assert torch.equal(y.detach(), want) and y.requires_grad
    with pytest.raises(RuntimeError, match="no backward pass"):
        (y.sum() + leaf.sum()).backward()
    assert leaf.grad is None
    with torch.no_grad():
        assert not run().requires_grad
    # a gradient that does not go through the layer is taken as ever
    other = torch.ones(3, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((run().sum(1) * other).sum(), other)
    assert torch.equal(g, want.sum(1))
    if which == "x":  # the layer in the middle of a model that is trained
        first, last = autograd.Linear(200, 200).cuda(), autograd.LinearW4.from_linear(autograd.Linear(200, 40).cuda())
        hidden = first(x.detach())
        with pytest.raises(RuntimeError, match="no backward pass"):
            (last(hidden).sum() + hidden.sum()).backward()


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_large_values_up_to_where_a_groups_products_overflow(group, dtype):
    """A group's products are summed in fp32 before its scale: they have to be finite there, as 6 * group * |x| is for the values here.  (The largest
    values of the type itself, times a code of up to 6, are not.)"""
    from distributed_tensorflow_amd.ops import hip_ops
    wq, scales = hip_ops.quantize_w4(0.02 * torch.randn(300, 40, generator=torch.Generator("cuda").manual_seed(0), device="cuda"), group)
    w = hip_ops.dequantize_w4(wq, scales, 300, 40).double()
    top = torch.finfo(F).max
    sign = torch.where(torch.rand(5, 300, generator=torch.Generator("cuda").manual_seed(1), device="cuda") < 0.5, -1.0, 1.0)
    x = (sign * (top / (8 * group))).to(dtype)
    assert float(w.abs().amax()) < 0.2  # (300 / 256 of that: the sum over the groups stays finite too)
    check(hip_ops.linear_w4(x, wq, scales, 40), x, None, w, None, False)
    z = torch.zeros(3, 300, device="cuda").to(dtype)
    z[:, 7] = top / 8  # alone in its group
    check(hip_ops.linear_w4(z, wq, scales, 40), z, None, w, None, False)
