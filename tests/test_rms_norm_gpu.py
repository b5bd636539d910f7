"""csrc/hip/rms_norm.hip through ops.hip_ops and ops.autograd, against the definition in float64."""
import pytest
import torch

from rms_norm_oracle import check_backward, check_e4m3, check_forward

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
# (rows, dim): one element; a wave a row with 1, 2, 4 pieces; odd widths; 256 and 1024 threads; rows longer than a workgroup's registers
SHAPES = [(1, 1), (3, 7), (1, 2048), (5, 256), (1500, 512), (1030, 1024), (1027, 2048), (33, 1000), (6, 1001), (2, 3137), (700, 4096), (4, 4100),
          (3, 8192), (2, 8199), (2, 16384), (2, 20000), (1025, 129), (1100, 250), (512, 2048), (513, 2048),
          (511, 1000), (300, 4097)]


def _rand(gen, *shape, dtype=F):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _inputs(rows, dim, dtype, residual, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    x = _rand(gen, rows, dim, dtype=dtype)
    res = (3 * _rand(gen, rows, dim)).to(dtype) if residual else None
    return gen, x, res, 1 + 0.3 * _rand(gen, dim)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_forward_backward_and_e4m3(rows, dim, dtype, residual):
    from distributed_tensorflow_amd.ops import hip_ops
    gen, x, res, w = _inputs(rows, dim, dtype, residual)
    y, h, rstd = hip_ops.rms_norm_forward(x, w, res, eps=1e-5)
    check_forward(y, h, rstd, x, w, res, 1e-5)
    assert residual or h is x
    q, scale, h2 = hip_ops.rms_norm_e4m3(x, w, res, eps=1e-5)
    check_e4m3(q, scale, x, w, res, 1e-5)
    assert torch.equal(h, h2)
    dy = _rand(gen, rows, dim, dtype=dtype)
    dh = _rand(gen, rows, dim, dtype=dtype) if residual else None
    dx, dw = hip_ops.rms_norm_backward(dy, x, rstd, w, res, dh)
    check_backward(dx, dw, dy, x, rstd, w, res, dh)
    dx2, none = hip_ops.rms_norm_backward(dy, x, rstd, w, res, dh, need_dw=False)
    assert torch.equal(dx, dx2) and none is None
    again = hip_ops.rms_norm_backward(dy, x, rstd, w, res, dh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])  # no atomics: the same bits


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("dim", [64, 72, 1000, 16388, 16400])
def test_strided_and_unaligned_rows(dtype, dim):
    from distributed_tensorflow_amd.ops import hip_ops
    gen = torch.Generator("cuda").manual_seed(1)
    room = lambda: _rand(gen, 9, dim + 40, dtype=dtype)  # noqa: E731
    for lo in (0, 1, 8):
        x, res, dy, dh = (room()[:, lo:lo + dim] for _ in range(4))
        w = 1 + 0.3 * _rand(gen, dim + 1)[1:].clone()
        y, h, rstd = hip_ops.rms_norm_forward(x, w, res)
        check_forward(y, h, rstd, x, w, res, 1e-6)
        dx, dw = hip_ops.rms_norm_backward(dy, x, rstd, w, res, dh)
        check_backward(dx, dw, dy, x, rstd, w, res, dh)
        y1, h1, r1 = hip_ops.rms_norm_forward(x, w)
        dx1, dw1 = hip_ops.rms_norm_backward(dy, x, r1, w, dh=dh)
        check_backward(dx1, dw1, dy, x, r1, w, None, dh)
        dx2, dw2 = hip_ops.rms_norm_backward(dy, x, rstd, w, res)
        check_backward(dx2, dw2, dy, x, rstd, w, res, None)
        q, scale, _ = hip_ops.rms_norm_e4m3(x, w, res)
        check_e4m3(q, scale, x, w, res, 1e-6)
    t = _rand(gen, dim, 5, dtype=dtype).t()  # elements of a row apart from one another
    y, h, rstd = hip_ops.rms_norm_forward(t, w)
    check_forward(y, h, rstd, t, w, None, 1e-6)
    e = _rand(gen, 1, dim, dtype=dtype).expand(6, dim)  # one row for all
    y, h, rstd = hip_ops.rms_norm_forward(e, w)
    check_forward(y, h, rstd, e, w, None, 1e-6)
    n = _rand(gen, 2, 3, dim, dtype=dtype)
    y, h, rstd = hip_ops.rms_norm_forward(n, w, n)
    assert y.shape == n.shape and rstd.shape == (2, 3)
    check_forward(y, h, rstd, n, w, n, 1e-6)


def test_rows_of_zeros_nan_inf_and_tiny_values():
    from distributed_tensorflow_amd.ops import hip_ops
    x = torch.ones(6, 300, device="cuda")
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    x[4] *= 1e-30
    w = torch.ones(300, device="cuda")
    y, _, rstd = hip_ops.rms_norm_forward(x, w, eps=0.0)
    assert bool(torch.isnan(y[0]).all()) and bool(torch.isinf(rstd[0]))  # 0 / 0, as the formula says without eps
    assert bool(torch.isnan(y[1]).all()) and float(rstd[2]) == 0 and bool(torch.isnan(y[2, 7])) and float(y[2, 8]) == 0
    assert bool((y[3] == 1).all())
    q, scale, _ = hip_ops.rms_norm_e4m3(x, w)
    assert float(scale[0]) == 0 and not q[0].float().any()
    assert bool(torch.isnan(scale[1])) and bool(torch.isnan(scale[2])) and bool((q[3].float() == 448).all())
    assert float(scale[4]) > 0 and bool((q[4].float() == 448).all())  # 1e-27, far above 2^-100
    q, scale, _ = hip_ops.rms_norm_e4m3(x[3:4], w * 1e-33)
    assert bool(torch.isfinite(q.float()).all())
    # 1e-33 is below 2^-100: in units of 2^-100 / 448 it is 0.57, where e4m3's grid is 2^-4
    assert abs(float(q[0, 0]) * float(scale[0]) - 1e-33) <= 2.0 ** -100 / 448 * 2.0 ** -5 * 1.001


def test_empty_rows():
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    y = autograd.rms_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 16) and not w.grad.any() and x.grad.shape == (0, 16)
    q, scale, h = hip_ops.rms_norm_e4m3(x.detach(), w.detach(), x.detach())
    assert q.shape == (0, 16) and scale.shape == (0,) and h.shape == (0, 16)


@pytest.mark.parametrize("rows,dim", [(5, 40), (64, 515)])
def test_gradients_against_autograd_in_float64_and_differences(rows, dim):
    from distributed_tensorflow_amd.ops import autograd
    gen, x, res, w = _inputs(rows, dim, F, True, seed=3)
    a, b = _rand(gen, rows, dim), _rand(gen, rows, dim)
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    y, h = autograd.rms_norm(*leaves, eps=1e-5)
    grads = torch.autograd.grad((y * a).sum() + (h * b).sum(), leaves)
    l64 = [t.double().requires_grad_() for t in (x, w, res)]

    def loss64(x, w, res):
        h = x + res
        return (h / (h.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w * a.double()).sum() + (h * b.double()).sum()

    want = torch.autograd.grad(loss64(*l64), l64)
    for g, t in zip(grads, want):  # 64 U of terms no larger than 10 times the gradient's own norm over its elements
        assert float((g.double() - t).norm() / t.norm()) < 64 * 2.0 ** -24 * 10
    for i in range(3):  # a central difference along a random direction, float64: h^2 / 6 of the third derivative, ~1e-9 relative at 1e-4
        v = torch.randn(l64[i].shape, generator=torch.Generator().manual_seed(i)).double().cuda()
        at = lambda s: loss64(*[t.detach() + (s * v if j == i else 0) for j, t in enumerate(l64)])  # noqa: E731
        diff = float(at(1e-4) - at(-1e-4)) / 2e-4
        mine = float((grads[i].double() * v).sum())
        assert abs(diff - mine) <= 1e-5 * float((grads[i].double() * v).abs().sum())


def test_which_gradients_are_asked_for():
    from distributed_tensorflow_amd.ops import autograd
    gen, x, res, w = _inputs(7, 64, F, True)
    layer = autograd.RMSNorm(64).cuda()
    x.requires_grad_()
    y, h = layer(x, res)
    h.sum().backward()  # only the residual stream's
    assert torch.equal(x.grad, torch.ones_like(x)) and not layer.weight.grad.any()
    layer.weight.requires_grad_(False)
    x.grad = None
    layer(x).sum().backward()
    assert x.grad is not None
    layer.weight.requires_grad_(True)
    layer.weight.grad = None
    layer(x.detach()).sum().backward()
    assert layer.weight.grad is not None
    with pytest.raises(RuntimeError):  # once differentiable
        g, = torch.autograd.grad(layer(x).pow(2).sum(), x, create_graph=True)
        g.sum().backward()


def test_captured_forward_and_backward_replay_like_eager():
    from distributed_tensorflow_amd.ops import autograd
    gen, x, res, w = _inputs(40, 1024, B, True)
    x.requires_grad_(), w.requires_grad_()
    dy, dh = _rand(gen, 40, 1024, dtype=B), _rand(gen, 40, 1024, dtype=B)

    def step():
        y, h = autograd.rms_norm(x, w, res)
        return (y, h) + torch.autograd.grad((y, h), (x, w), (dy, dh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(_rand(gen, 40, 1024, dtype=B))
            dy.copy_(_rand(gen, 40, 1024, dtype=B))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_another_stream_than_the_tensors_own():
    from distributed_tensorflow_amd.ops import hip_ops
    gen, x, res, w = _inputs(2000, 2048, B, True)
    want = hip_ops.rms_norm_forward(x, w, res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hip_ops.rms_norm_forward(x, w, res)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_rows_behind_two_to_the_31_elements():
    from distributed_tensorflow_amd.ops import hip_ops
    rows, dim = (1 << 20) + 3, 2056
    x = torch.zeros(rows, dim, dtype=B, device="cuda")
    x[-5:] = torch.randn(5, dim, generator=torch.Generator("cuda").manual_seed(0), device="cuda").to(B)
    w = torch.ones(dim, device="cuda")
    y, h, rstd = hip_ops.rms_norm_forward(x, w, x)
    check_forward(y[-5:], h[-5:], rstd[-5:], x[-5:], w, x[-5:], 1e-6)
    dx, dw = hip_ops.rms_norm_backward(x, x, rstd, w, x)
    check_backward(dx[-5:], None, x[-5:], x[-5:], rstd[-5:], w, x[-5:], None)
    assert not dx[:-5].any()
    q, scale, _ = hip_ops.rms_norm_e4m3(x, w)
    check_e4m3(q[-5:], scale[-5:], x[-5:], w, None, 1e-6)


def test_more_rows_than_a_launch_takes():
    from distributed_tensorflow_amd.ops import hip_ops
    rows = (1 << 21) + 1000
    x = torch.randn(rows, 24, generator=torch.Generator("cuda").manual_seed(0), device="cuda")
    w = torch.ones(24, device="cuda")
    y, h, rstd = hip_ops.rms_norm_forward(x, w, x)
    check_forward(y, h, rstd, x, w, x, 1e-6)
    q, scale, h2 = hip_ops.rms_norm_e4m3(x.to(B), w, x.to(B))
    check_e4m3(q, scale, x.to(B), w, x.to(B), 1e-6)
    dx, dw = hip_ops.rms_norm_backward(x, x, rstd, w, x)
    check_backward(dx, dw, x, x, rstd, w, x, None)


def test_a_single_row_without_a_batch_and_inference_mode():
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    x = torch.randn(300, device="cuda")
    w = torch.rand(300, device="cuda", requires_grad=True)
    y, h, rstd = hip_ops.rms_norm_forward(x, w)
    assert y.shape == (300,) and rstd.shape == () and not y.requires_grad
    check_forward(y, h, rstd, x, w.detach(), None, 1e-6)
    dx, dw = hip_ops.rms_norm_backward(y, x, rstd, w)
    check_backward(dx, dw, y, x, rstd, w.detach(), None, None)
    q, scale, _ = hip_ops.rms_norm_e4m3(x, w)
    assert q.shape == (300,) and scale.shape == ()
    with torch.inference_mode():
        a, b = autograd.rms_norm(x, w, x)
        assert torch.equal(b, x + x) and not a.requires_grad


def test_refusals():
    from distributed_tensorflow_amd.ops import hip_ops
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: hip_ops.rms_norm_forward(x.double(), w), lambda: hip_ops.rms_norm_forward(x.half(), w),
                lambda: hip_ops.rms_norm_forward(x, w.to(B)), lambda: hip_ops.rms_norm_forward(x, torch.ones(7, device="cuda")),
                lambda: hip_ops.rms_norm_forward(x, w, x[:3]), lambda: hip_ops.rms_norm_forward(x, w, x.to(B)),
                lambda: hip_ops.rms_norm_forward(x, w, x[:1]), lambda: hip_ops.rms_norm_forward(x, w, eps=-1.0),
                lambda: hip_ops.rms_norm_forward(x, w, eps=float("nan")), lambda: hip_ops.rms_norm_forward(x, w.cpu()),
                lambda: hip_ops.rms_norm_forward(torch.zeros((), device="cuda"), w),
                lambda: hip_ops.rms_norm_forward(torch.zeros(3, 0, device="cuda"), torch.ones(0, device="cuda")),
                lambda: hip_ops.rms_norm_backward(x, x, torch.ones(3, device="cuda"), w),
                lambda: hip_ops.rms_norm_backward(x[:3], x, torch.ones(4, device="cuda"), w),
                lambda: hip_ops.rms_norm_backward(x, x, torch.ones(4, device="cuda"), w, dh=x.to(B))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("residual", [False, True])
def test_second_derivatives_are_refused_for_constant_incoming_gradients_too(residual):
    """dx and dw depend on x, w and the residual also where dy does not require a gradient: y.sum(), or fixed grad_outputs."""
    from distributed_tensorflow_amd.ops import autograd
    gen, x, res, w = _inputs(7, 64, F, residual)
    leaves = [t.requires_grad_() for t in (x, w, res) if t is not None]
    dy = _rand(gen, 7, 64)

    def grads(inputs):
        y = autograd.rms_norm(x, w, res)
        return torch.autograd.grad(y[0] if residual else y, inputs, dy, create_graph=True)

    for leaf in leaves:
        g, = grads([leaf])
        with pytest.raises(RuntimeError, match="differentiable once"):
            (g.sum() + leaf.sum()).backward()
    for g in grads(leaves):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum(), leaves, allow_unused=True)
    y = autograd.rms_norm(x, w, res)
    g, = torch.autograd.grad((y[0] if residual else y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g * g).sum().backward()


def test_what_has_a_second_derivative_or_none_is_not_refused():
    from distributed_tensorflow_amd.ops import autograd
    gen, x, res, w = _inputs(7, 64, F, True)
    a = _rand(gen, 7, 64)
    # dw of constant rows and a constant dy depends on nothing that requires a gradient
    w.requires_grad_()
    dw, = torch.autograd.grad(autograd.rms_norm(x, w), w, a, create_graph=True)
    assert not dw.requires_grad and torch.equal(dw, torch.autograd.grad(autograd.rms_norm(x, w), w, a)[0])
    # h = x + residual is linear: its gradient is dh itself, and dh's own graph goes on
    x.requires_grad_()
    a.requires_grad_()
    _, h = autograd.rms_norm(x, w, res)
    g, = torch.autograd.grad((h * a * a).sum(), x, create_graph=True)
    assert torch.equal(g, a * a)
    g.sum().backward()
    assert torch.equal(a.grad, 2 * a.detach())


def test_the_forms_without_a_backward_pass_refuse_one():
    """x or the residual requires a gradient: the values are those of any call, the backward pass raises instead of dropping it."""
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    gen, x, res, w = _inputs(5, 200, B, True)
    want8, want = hip_ops.rms_norm_e4m3(x, w, res), hip_ops.rms_norm_forward(x, w, res)
    for name in ("x", "res"):
        z, r = (x.clone().requires_grad_(), res) if name == "x" else (x, res.clone().requires_grad_())
        for got, ref in ((hip_ops.rms_norm_e4m3(z, w, r), want8), (hip_ops.rms_norm_forward(z, w, r), want)):
            for a, b in zip(got, ref):
                assert torch.equal(a.detach().view(torch.uint8), b.view(torch.uint8))
                with pytest.raises(RuntimeError, match="no backward pass"):
                    a.float().sum().backward()
        with torch.no_grad():
            assert not any(t.requires_grad for t in hip_ops.rms_norm_e4m3(z, w, r) + hip_ops.rms_norm_forward(z, w, r))
    z = x.clone().requires_grad_()
    q, scale, h = hip_ops.rms_norm_e4m3(z, w)
    assert h is z and q.requires_grad  # (without a residual h is x, whose gradient is its own)
    layer = autograd.RMSNorm(200).cuda()
    assert hip_ops.rms_norm_e4m3(x, layer.weight)[0].requires_grad  # (its weight has no gradient here either)


def test_backward_of_more_long_rows_than_a_launch_takes():
    """2^22 workgroups of 1024 threads are 2^32 threads (x and dy are one row for all, dx is 137 GB)."""
    from distributed_tensorflow_amd.ops import hip_ops
    rows, dim = (1 << 22) + 3, 8196
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GB of free memory")
    gen, one, _, w = _inputs(1, dim, F, False)
    dy = _rand(gen, 1, dim)
    rstd = 0.5 + torch.rand(rows, generator=gen, device="cuda")
    dx, _ = hip_ops.rms_norm_backward(dy.expand(rows, dim), one.expand(rows, dim), rstd, w, need_dw=False)
    for at in list(range(0, rows, 262139)) + [rows - 5]:
        r = rstd[at:at + 3]
        check_backward(dx[at:at + 3], None, dy.expand(3, dim), one.expand(3, dim), r, w, None, None)
    del dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 2])
def test_dw_of_more_columns_than_a_launch_takes(rows):
    """2^28 columns, 64 a workgroup of 1024 threads, are 2^32 threads."""
    from distributed_tensorflow_amd.ops import hip_ops
    dim = (1 << 28) + 70
    gen = torch.Generator("cuda").manual_seed(0)
    x, dy, w = _rand(gen, rows, dim, dtype=B), _rand(gen, rows, dim, dtype=B), torch.ones(dim, device="cuda")
    rstd = torch.full((rows,), 0.75, device="cuda")
    dw = hip_ops.rms_norm_backward(dy, x, rstd, w)[1]
    for at in list(range(0, dim, (1 << 22) - 3)) + [dim - 80]:  # a product and its sum of two rows, one rounding each
        h, d = x[:, at:at + 80].double() * 0.75, dy[:, at:at + 80].double()
        assert bool(((dw[at:at + 80].double() - (h * d).sum(0)).abs() <= (h * d).abs().sum(0) * 4 * 2.0 ** -24).all()), at
