"""csrc/hip/adamw.hip through optim.adamw: against the definition in float64 and, bit for bit, the CPU's eager form."""
import pytest
import torch

from adamw_oracle import check
from distributed_tensorflow_amd.optim.adamw import AdamW

pytestmark = pytest.mark.gpu
HYPER = dict(lr=3e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.02)
KW = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.02)
F, B = torch.float32, torch.bfloat16


def _same(a, b):
    return torch.equal(a.detach().cpu().contiguous().view(torch.uint8), b.detach().cpu().contiguous().view(torch.uint8))


def _pair(sizes, dtypes, bits, offset=0, seed=0):
    """The same parameters on the GPU (views that start `offset` elements behind an aligned address) and on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    gpu, cpu = [], []
    for i, n in enumerate(sizes):
        x = (0.3 * torch.randn(n, generator=gen)).to(dtypes[i % len(dtypes)])
        room = torch.zeros(n + offset + 8, dtype=x.dtype, device="cuda")
        room[offset:offset + n] = x.cuda()
        gpu.append(room[offset:offset + n].requires_grad_())
        cpu.append(x.clone().requires_grad_())
    return (gpu, AdamW(gpu, state_bits=bits, seed=11, **KW)), (cpu, AdamW(cpu, state_bits=bits, seed=11, **KW))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("gtype", [F, B])
def test_steps_match_the_definition_and_the_cpu(bits, offset, gtype):
    sizes = [1, 7, 8, 255, 256, 257, 2040, 2047, 2048, 2049, 5000, 70001]
    (gpu, opt), (cpu, ref) = _pair(sizes, [F, B], bits, offset)
    rooms = [p.detach().as_strided((p.numel() + 8,), (1,), p.storage_offset()) for p in gpu]
    gen = torch.Generator().manual_seed(5)
    for t in range(1, 5):
        grads = [(0.1 * torch.randn(n, generator=gen)).to(gtype) for n in sizes]
        before = [{k: x.clone() for k, x in opt.state[p].items()} for p in gpu]
        old = [p.detach().clone() for p in gpu]
        held = [torch.zeros(n + offset, dtype=gtype, device="cuda") for n in sizes]
        dev = []
        for h, g in zip(held, grads):
            h[offset:] = g.cuda()
            dev.append(h[offset:])
        opt.step(grads=dev, grad_scale=0.5)
        ref.step(grads=grads, grad_scale=0.5)
        for p, q, o, b, g in zip(gpu, cpu, old, before, dev):
            check(b, opt.state[p], o, p.detach(), g, t, HYPER, grad_scale=0.5)
            assert _same(p, q), p.numel()
        for k, x in opt.arenas().items():
            assert _same(x, ref.arenas()[k]), k
    for p, room in zip(gpu, rooms):  # what lies behind a parameter is left as it was
        assert not room[p.numel():].any()


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_missing_gradients_and_strided_ones(bits):
    sizes = [(1 + 37 * i) % 900 for i in range(430)]  # more than two sets of kernel arguments; some tensors are empty
    (gpu, opt), (cpu, ref) = _pair(sizes, [F, B, F], bits)
    gen = torch.Generator().manual_seed(6)
    for t in range(3):
        for i, (p, q) in enumerate(zip(gpu, cpu)):
            g = torch.randn(q.numel(), 2, generator=gen)[:, 0].to(q.dtype)
            p.grad = q.grad = None
            if (i + t) % 5:
                p.grad, q.grad = g.cuda().repeat_interleave(2)[::2], g
        opt.step()
        ref.step()
    for p, q in zip(gpu, cpu):
        assert _same(p, q)
    for k, x in opt.arenas().items():
        assert _same(x, ref.arenas()[k]), k


def test_groups_and_loaded_states():
    def make(dev):
        gen = torch.Generator().manual_seed(3)
        a, b = (torch.randn(3000, generator=gen).to(dev).requires_grad_(), torch.randn(70, 3, generator=gen).to(dev).requires_grad_())
        return [a, b], AdamW([{"params": [a]}, {"params": [b], "lr": 0.1, "weight_decay": 0.0}], state_bits=8, **KW)

    (pg, og), (pc, oc) = make("cuda"), make("cpu")

    def steps(ps, o, lo, hi):
        for t in range(lo, hi):
            gen = torch.Generator().manual_seed(t)
            for p in ps:
                p.grad = torch.randn(p.shape, generator=gen).to(p.device)
            o.step()

    steps(pg, og, 0, 3)
    steps(pc, oc, 0, 3)
    oc.load_state_dict(og.state_dict())  # across devices
    steps(pg, og, 3, 5)
    steps(pc, oc, 3, 5)
    for p, q in zip(pg, pc):
        assert _same(p, q)


def test_non_finite_gradients_match_the_cpu():
    (gpu, opt), (cpu, ref) = _pair([600], [F], 8)
    g = torch.randn(600, generator=torch.Generator().manual_seed(1))
    g[[0, 255]], g[256], g[599] = float("inf"), float("nan"), -float("inf")
    for _ in range(2):
        opt.step(grads=[g.cuda()])
        ref.step(grads=[g])
        for k in ("m", "r"):
            a, b = opt.arenas()[k].float().cpu(), ref.arenas()[k].float()
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~torch.isnan(a)], b[~torch.isnan(b)])
        a, b = gpu[0].detach().cpu(), cpu[0].detach()
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~torch.isnan(a)], b[~torch.isnan(b)])


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_replay_like_eager_ones(bits):
    sizes = [33, 4096, 70000]
    (gpu, opt), (cpu, ref) = _pair(sizes, [F, B], bits)
    grads = [torch.zeros(n, device="cuda", dtype=p.dtype) for n, p in zip(sizes, gpu)]
    other = [torch.zeros_like(g) for g in grads]
    graphs = []
    for src in (grads, other):  # two graphs of one optimizer, each with gradients of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step(grads=src)
        graphs.append(graph)
    gen = torch.Generator().manual_seed(8)
    for t in range(6):
        new = [torch.randn(n, generator=gen).to(g.dtype) for n, g in zip(sizes, grads)]
        for g, x in zip((grads, other)[t % 2], new):
            g.copy_(x)
        graphs[t % 2].replay()
        torch.cuda.synchronize()
        ref.step(grads=new)
        for p, q in zip(gpu, cpu):
            assert _same(p, q), t
        if t == 3:  # an eager step between the replays
            opt.step(grads=[x.cuda() for x in new])
            ref.step(grads=new)
    assert opt.arenas()["step"].tolist() == [7] * 3


def test_another_stream_than_the_tensors_own():
    (gpu, opt), (cpu, ref) = _pair([100000], [F], 8)
    side = torch.cuda.Stream()
    g = torch.randn(100000, generator=torch.Generator().manual_seed(2))
    dev = g.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step(grads=[dev])
    torch.cuda.current_stream().wait_stream(side)
    ref.step(grads=[g])
    assert _same(gpu[0], cpu[0])


def test_places_behind_two_to_the_31():
    n = (1 << 31) + 4101
    p = torch.zeros(n, dtype=B, device="cuda").requires_grad_()
    opt = AdamW([p], state_bits=8, seed=2, **KW)
    g = torch.zeros(n, dtype=B, device="cuda")
    g[:5000].normal_(generator=torch.Generator("cuda").manual_seed(1))
    g[-5000:].normal_(generator=torch.Generator("cuda").manual_seed(2))
    opt.step(grads=[g])
    lo = (n - 5000) // 256 * 256
    for a, b in ((0, 5000), (lo, n)):
        st = {k: x[a // 256:-(-b // 256)] if k.endswith("scale") else x[a:-(-b // 256) * 256]
              for k, x in opt.state[p].items() if k != "step"}
        zero = {k: torch.full_like(x, 2.0 ** -126) if k.endswith("scale") else torch.zeros(x.shape, device="cuda").to(x.dtype) for k, x in st.items()}
        check(zero, st, torch.zeros(b - a, dtype=B, device="cuda"), p.detach()[a:b], g[a:b], 1, HYPER)
    assert not p.detach()[5000:lo].any() and not opt.arenas()["m"].view(torch.uint8)[5120:lo].any()


def test_schedulers_and_a_tensor_changed_behind_the_optimizers_back():
    p = torch.ones(100, device="cuda", requires_grad=True)
    opt = AdamW([p], lr=1.0, weight_decay=0.0, eps=0.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    for want in (0.0, -0.5):  # the first steps of a constant gradient are lr long
        p.grad = torch.ones(100, device="cuda")
        opt.step()
        sched.step()
        assert bool(((p.detach() - want).abs() <= 16 * 2.0 ** -24).all())
    loss = (p * p).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    p.data = p.data.to(B)
    with pytest.raises(ValueError, match="has changed"):
        opt.step(grads=[torch.ones(100, device="cuda")])


def test_refusals_on_the_gpu():
    p = torch.zeros(8, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="one device"):
        AdamW([p, torch.zeros(8, requires_grad=True)])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.step(grads=[torch.ones(8)])
    with pytest.raises(ValueError):
        opt.step(grads=[torch.ones(9, device="cuda")])
    assert opt.arenas()["step"].tolist() == [0] and not p.detach().any()


@pytest.mark.parametrize("bits", [8, 32])
def test_two_captured_steps_over_different_parameters_replay_at_once(bits):
    """What the first kernel of a step leaves for the second is the step's own: another step's begin, which has no gradient for these
    parameters, must not reach it."""
    sizes = [40000, 3, 70001, 900]
    (gpu, opt), (cpu, ref) = _pair(sizes, [F, B], bits)
    grads = [torch.zeros(n, device="cuda", dtype=p.dtype) for n, p in zip(sizes, gpu)]
    halves = [[g if i % 2 == half else None for i, g in enumerate(grads)] for half in (0, 1)]
    graphs = []
    for half in halves:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step(grads=half)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    gen = torch.Generator().manual_seed(9)
    for t in range(8):
        new = [torch.randn(n, generator=gen).to(g.dtype) for n, g in zip(sizes, grads)]
        for g, x in zip(grads, new):
            g.copy_(x)
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for half in (0, 1):  # and eager steps, each on its stream
            with torch.cuda.stream(streams[half]):
                opt.step(grads=halves[half])
        torch.cuda.synchronize()
        ref.step(grads=new)
        ref.step(grads=new)
        for p, q in zip(gpu, cpu):
            assert _same(p, q), t
        for k, x in opt.arenas().items():
            assert _same(x, ref.arenas()[k]), (t, k)


@pytest.mark.parametrize("bits", [8, 32])
def test_more_chunks_than_a_launch_takes(bits):
    """2^24 chunks of 2048 elements are 2^32 threads.  The table here has that many entries for a tensor of two chunks: the others lie
    behind its end and are left at once."""
    from distributed_tensorflow_amd import native
    n, entries = 2048 + 300, (1 << 24) + 5
    (gpu, opt), (cpu, ref) = _pair([n], [F], bits)
    group = opt._groups[0]
    chunks = torch.zeros(entries, 2, dtype=torch.int32, device="cuda")
    chunks[:, 1] = 2  # (starts at element 4096)
    chunks[0, 1], chunks[-1, 1] = 1, 0
    places = {"shape": group.shape, "chunks": chunks, "step": group.step, **group.arenas}
    group.native = native.ext().AdamWGroup(group.params, {k: t.data_ptr() for k, t in places.items()}, entries, bits, group.seed)
    gen = torch.Generator().manual_seed(3)
    for _ in range(2):
        g = torch.randn(n, generator=gen)
        opt.step(grads=[g.cuda()])
        ref.step(grads=[g])
        assert _same(gpu[0], cpu[0])
        for k, x in opt.arenas().items():
            assert _same(x, ref.arenas()[k]), k
