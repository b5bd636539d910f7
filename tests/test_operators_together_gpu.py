"""The RMS norm, AdamW and the 4-bit dense layer as they are used together: a residual block with a class layer is trained, its class
layer is brought to 4 bits, and single rows go through norm (8 bits) and layer (4 bits)."""
import pytest
import torch

import adamw_oracle
from rms_norm_oracle import check_backward, check_e4m3, check_forward

pytestmark = pytest.mark.gpu
HYPER = dict(lr=2e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01)


class Block(torch.nn.Module):
    def __init__(self, dim, classes):
        super().__init__()
        from distributed_tensorflow_amd.ops import autograd as ag
        self.inner = ag.Linear(dim, dim, relu=True, std=0.05, bias_init=0.0)
        self.norm = ag.RMSNorm(dim)
        self.head = ag.Linear(dim, classes, std=0.05, bias_init=0.0)

    def forward(self, x):
        self.a = self.inner(x)
        self.y, self.h = self.norm(self.a, x)
        return self.head(self.y)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dim,classes", [(264, 10), (2048, 101)])
def test_train_quantise_and_serve(dim, classes, bits):
    from distributed_tensorflow_amd.ops import autograd as ag, hip_ops
    from distributed_tensorflow_amd.optim.adamw import AdamW
    torch.manual_seed(0)
    net = Block(dim, classes).cuda()
    opt = AdamW(net.parameters(), lr=HYPER["lr"], eps=HYPER["eps"], weight_decay=HYPER["wd"], state_bits=bits)
    x = torch.randn(64, dim, device="cuda", requires_grad=True)
    target = torch.randint(0, classes, (64,), device="cuda")
    for t in range(1, 4):
        opt.zero_grad()
        loss = torch.nn.functional.cross_entropy(net(x), target) + 1e-3 * net.h.pow(2).mean()  # (h has a gradient of its own)
        for v in (net.a, net.y, net.h):
            v.retain_grad()
        loss.backward()
        w = net.norm.weight
        rstd = hip_ops.rms_norm_forward(net.a.detach(), w.detach(), x.detach())[2]
        check_forward(net.y.detach(), net.h.detach(), rstd, net.a.detach(), w.detach(), x.detach(), net.norm.eps)
        check_backward(net.a.grad, w.grad, net.y.grad, net.a.detach(), rstd, w.detach(), x.detach(), net.h.grad)
        params = list(net.parameters())
        before = [({k: s.clone() for k, s in opt.state[p].items()}, p.detach().clone()) for p in params]
        opt.step()
        for p, (state, old) in zip(params, before):
            adamw_oracle.check(state, opt.state[p], old, p.detach(), p.grad, t, HYPER)
    # serving: one row after the other, then the whole chain from a graph
    q4 = ag.LinearW4.from_linear(net.head, 64)
    w4 = hip_ops.dequantize_w4(q4.wq, q4.scales, dim, classes).double()
    step = w4.new_tensor(1.0) * q4.scales.float().permute(1, 0, 2).reshape(q4.scales.shape[1], -1).repeat_interleave(64, 0)[:dim, :classes].double()
    with torch.no_grad():
        a = net.inner(x)

    def serve(a, x):
        q, scale, h = hip_ops.rms_norm_e4m3(a, net.norm.weight.detach(), x, eps=net.norm.eps)
        return q, scale, h, q4(q, scale)

    for i in (0, 17, 63):
        q, scale, h, logits = serve(a[i:i + 1], x.detach()[i:i + 1])
        check_e4m3(q, scale, a[i:i + 1], net.norm.weight.detach(), x.detach()[i:i + 1], net.norm.eps)
        rows = q.double() * scale.double()[:, None]
        want = rows @ w4 + q4.bias.double()
        assert bool(((logits.double() - want).abs() <= (rows.abs() @ w4.abs()) * (3 * dim + 100) * 2.0 ** -24 + want.abs() * 2.0 ** -22).all())
        # against the layer as it was trained: the rows' rounding to e4m3 (half a step, 2^-4, or 2^-10 of the row's scale) on the 4-bit
        # weights, and the weights' rounding (half the widest gap of the values, 1, times the group's scale, which is itself rounded by
        # 2^-8 of 6) on the exact rows
        with torch.no_grad():
            exact = net.norm(a[i:i + 1], x[i:i + 1])[0].double()
        full = exact @ net.head.weight.detach().double() + net.head.bias.detach().double()
        rounding = torch.maximum(exact.abs() * 2.0 ** -4, scale.double()[:, None] * 2.0 ** -10) * 1.001
        bound = rounding @ w4.abs() + exact.abs() @ (step * (1 + 6 * 2.0 ** -8)) + 1e-4 * (exact.abs() @ w4.abs())
        assert bool(((logits.double() - full).abs() <= bound).all())
    row, res = a[:1].clone(), x.detach()[:1].clone()
    serve(row, res)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serve(row, res)
    for i in (5, 6, 7, 8):
        row.copy_(a[i:i + 1])
        res.copy_(x.detach()[i:i + 1])
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, serve(a[i:i + 1], x.detach()[i:i + 1])):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_a_captured_training_step_replays_like_eager():
    """Forward, backward and AdamW in one graph; the eager graph of the leaves is gone before the capture begins."""
    from distributed_tensorflow_amd.ops import autograd as ag
    from distributed_tensorflow_amd.optim.adamw import AdamW

    def make():
        torch.manual_seed(3)
        w = torch.nn.Parameter(1 + 0.1 * torch.randn(512, device="cuda"))
        return w, AdamW([w], state_bits=8, seed=4)

    x = torch.randn(600, 512, device="cuda").to(torch.bfloat16)
    res, dy = torch.randn(600, 512, device="cuda").to(torch.bfloat16), torch.randn(600, 512, device="cuda").to(torch.bfloat16)
    (w1, o1), (w2, o2) = make(), make()
    g1 = torch.zeros(512, device="cuda")

    def step(w, opt, into):
        y, h = ag.rms_norm(x, w, res)
        g, = torch.autograd.grad((y,), (w,), (dy,))
        into.copy_(g)
        opt.step(grads=[into])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*make(), torch.zeros(512, device="cuda"))  # warm up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(w1, o1, g1)
    for i in range(4):
        x.copy_(torch.randn(600, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        step(w2, o2, torch.zeros(512, device="cuda"))
        assert torch.equal(w1, w2)
        for k, t in o1.arenas().items():
            assert torch.equal(t.view(torch.uint8), o2.arenas()[k].view(torch.uint8))


def test_forward_mode_derivatives_are_refused():
    """Tangents were dropped without a word where there is no rule for them; autograd.rms_norm's node refuses them itself."""
    import torch.autograd.forward_ad as fwd
    from distributed_tensorflow_amd.ops import autograd as ag, hip_ops
    x, w, t = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda"), torch.randn(4, 64, device="cuda")
    wq, scales = hip_ops.quantize_w4(torch.randn(64, 32, device="cuda"))
    with fwd.dual_level():
        d = fwd.make_dual(x, t)
        for f in (lambda: ag.rms_norm(d, w), lambda: hip_ops.rms_norm_forward(d, w), lambda: hip_ops.rms_norm_forward(x, w, d),
                  lambda: hip_ops.rms_norm_e4m3(d, w), lambda: hip_ops.rms_norm_e4m3(x, fwd.make_dual(w, w)),
                  lambda: hip_ops.linear_w4(d, wq, scales, 32), lambda: hip_ops.linear_w4(x, wq, scales, 32, bias=fwd.make_dual(w[:32], w[:32]))):
            with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                f()
        assert hip_ops.linear_w4(x, wq, scales, 32).shape == (4, 32)


def test_lazily_negated_views():
    """The imaginary part of a conjugate is a view whose memory holds the other sign; with one element a row it passes for contiguous."""
    from distributed_tensorflow_amd.ops import hip_ops
    from distributed_tensorflow_amd.optim.adamw import AdamW
    z = torch.randn(3, 1, dtype=torch.complex64, device="cuda")
    x, plain = z.conj().imag, -z.imag.clone()
    assert x.is_neg() and not plain.is_neg()
    one = torch.ones(1, device="cuda")
    y, h, rstd = hip_ops.rms_norm_forward(x, one, x)
    check_forward(y, h, rstd, plain, one, plain, 1e-6)
    check_e4m3(*hip_ops.rms_norm_e4m3(x, one)[:2], plain, one, None, 1e-6)
    check_backward(*hip_ops.rms_norm_backward(x, x, rstd, one, x, x), plain, plain, rstd, one, plain, plain)
    wq, scales = hip_ops.quantize_w4(torch.ones(1, 20, device="cuda"), 32)
    assert torch.equal(hip_ops.linear_w4(x, wq, scales, 20), hip_ops.linear_w4(plain, wq, scales, 20))
    ps = [torch.zeros(1, 1, device="cuda", requires_grad=True) for _ in range(2)]
    for p, g in zip(ps, (x[:1], plain[:1])):
        AdamW([p], lr=0.1).step(grads=[g])
    assert torch.equal(ps[0], ps[1]) and float(ps[0].detach()) != 0
    neg = z.conj().imag[0]
    for bad in (lambda: hip_ops.rms_norm_forward(plain, neg), lambda: hip_ops.rms_norm_backward(plain[:1], plain[:1], neg, one),
                lambda: hip_ops.linear_w4(plain[:1], wq, scales, 20, x_scale=neg), lambda: AdamW([neg.detach().requires_grad_()])):
        with pytest.raises(ValueError):
            bad()
