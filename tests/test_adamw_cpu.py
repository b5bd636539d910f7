"""optim.adamw on the CPU: the eager form against the definition in float64, state dictionaries, refusals."""
import copy
import pickle

import pytest
import torch

from adamw_oracle import check, grid, held
from distributed_tensorflow_amd.optim.adamw import BLOCK, AdamW

HYPER = dict(lr=3e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.02)
KW = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.02)


def _params(sizes, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(0.3 * torch.randn(n, generator=gen)).to(dtype).requires_grad_() for n in sizes]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_follow_the_definition(bits, dtype):
    params = _params([1, 7, 255, 256, 257, 1000], dtype)
    opt = AdamW(params, state_bits=bits, seed=3, **KW)
    gen = torch.Generator().manual_seed(1)
    for t in range(1, 6):
        before = [{k: x.clone() for k, x in opt.state[p].items()} for p in params]
        old = [p.detach().clone() for p in params]
        for p in params:
            p.grad = (torch.randn(p.shape, generator=gen) * 0.1).to(dtype)
        opt.step(grad_scale=0.5)
        for p, q, b in zip(params, old, before):
            check(b, opt.state[p], q, p.detach(), p.grad, t, HYPER, grad_scale=0.5)
            assert int(opt.state[p]["step"]) == t


def test_eight_bit_moments_are_unbiased_and_reproducible():
    n = 1 << 17
    runs = []
    for seed in (5, 5, 6):
        p = torch.zeros(n, requires_grad=True)
        opt = AdamW([p], state_bits=8, seed=seed)
        gen = torch.Generator().manual_seed(2)
        for _ in range(2):
            p.grad = torch.randn(n, generator=gen)
            before = {k: x.clone() for k, x in opt.state[p].items()}
            opt.step()
        runs.append({k: x.clone() for k, x in opt.state[p].items()})
    for k in runs[0]:
        assert torch.equal(runs[0][k].view(torch.uint8), runs[1][k].view(torch.uint8))
    assert not torch.equal(runs[0]["m"].view(torch.uint8), runs[2]["m"].view(torch.uint8))
    m, v = held(before, n)
    m = 0.9 * m + 0.1 * p.grad.double()
    got, _ = held(runs[2], n)
    # a stochastic rounding's error in steps has mean 0 and a deviation of at most 1/2: five deviations of the mean of n of them
    err = (got - m) / grid(m, runs[2]["m_scale"].double().repeat_interleave(BLOCK))
    assert abs(float(err.mean())) < 5 * 0.5 / n ** 0.5
    up = (err > 0).double()
    assert abs(float((up[1:] * up[:-1]).mean()) - float(up.mean()) ** 2) < 5 / n ** 0.5  # neighbours' bits do not go together


def test_an_average_moves_although_each_step_is_below_the_grid():
    """v decays by 0.1 % a step, its grid is 6-12 %: rounding to nearest would hold it for ever."""
    p = torch.zeros(4096, requires_grad=True)
    opt = AdamW([p], state_bits=8, seed=1)
    p.grad = torch.ones(4096)
    opt.step()
    first = float(held(opt.state[p], 4096)[1].mean())
    p.grad = torch.zeros(4096)
    steps = 400
    for _ in range(steps):
        opt.step()
    last = float(held(opt.state[p], 4096)[1].mean())
    want = first * 0.999 ** steps
    # each step adds the variance of r's rounding to v = r^2: p(1-p) of a squared step of at most 1/8, p = 0.0005 / (1/16)
    # (v's own spread after that, < 50 %, leaves the mean of 4096 elements within 5 deviations = 4 %)
    assert want * 0.96 < last < want * (1 + steps * 0.0080 / 64) * 1.04


def test_non_finite_gradients_stay_in_their_elements():
    p = torch.zeros(512, requires_grad=True)
    opt = AdamW([p], state_bits=8)
    g = torch.randn(512, generator=torch.Generator().manual_seed(0))
    g[3], g[300], g[301] = float("nan"), float("inf"), -float("inf")
    p.grad = g
    opt.step()
    bad = torch.zeros(512, dtype=torch.bool)
    bad[[3, 300, 301]] = True
    m, v = held(opt.state[p], 512)
    assert bool(torch.isnan(m[bad]).all()) and bool(torch.isnan(v[bad]).all())
    assert bool(torch.isfinite(m[~bad]).all()) and bool(torch.isfinite(p[~bad]).all()) and bool(torch.isnan(p[3]))


def test_zero_and_tiny_gradients():
    p = torch.ones(300, requires_grad=True)
    opt = AdamW([p], state_bits=8, weight_decay=0.0)
    p.grad = torch.zeros(300)
    opt.step()
    assert torch.equal(p.detach(), torch.ones(300)) and not opt.state[p]["m"].view(torch.uint8).any()
    p.grad = torch.full((300,), 1e-30)
    opt.step()
    assert bool(torch.isfinite(p).all())


def test_parameters_without_gradients_keep_their_counters():
    a, b = _params([10, 20])
    opt = AdamW([a, b])
    b.grad = torch.ones(20)
    old = a.detach().clone()
    opt.step()
    assert torch.equal(a.detach(), old) and opt.arenas()["step"].tolist() == [0, 1]
    opt.step(grads=[torch.ones(10), None])
    assert opt.arenas()["step"].tolist() == [1, 1]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_loaded_state_continues_bit_for_bit(bits, tmp_path):
    def make():
        a, b = _params([300, 33], torch.float32), _params([5], torch.bfloat16)
        return a + b, AdamW([{"params": a}, {"params": b, "lr": 1e-2, "weight_decay": 0.0}], state_bits=bits, seed=9, **KW)

    def steps(params, opt, lo, hi):
        for t in range(lo, hi):
            gen = torch.Generator().manual_seed(t)
            for p in params:
                p.grad = torch.randn(p.shape, generator=gen).to(p.dtype)
            opt.step()

    params, opt = make()
    steps(params, opt, 0, 3)
    torch.save(opt.state_dict(), tmp_path / "s.pt")
    kept = [p.detach().clone() for p in params]
    steps(params, opt, 3, 6)
    again, opt2 = make()
    with torch.no_grad():
        for p, k in zip(again, kept):
            p.copy_(k)
    arena = opt2.arenas()["m"]
    opt2.load_state_dict(torch.load(tmp_path / "s.pt", weights_only=True))
    assert arena.data_ptr() == opt2.arenas()["m"].data_ptr() and opt2.param_groups[1]["lr"] == 1e-2
    steps(again, opt2, 3, 6)
    for p, q in zip(params, again):
        assert torch.equal(p, q)
    for k in opt.arenas(0):
        assert torch.equal(opt.arenas(0)[k].view(torch.uint8), opt2.arenas(0)[k].view(torch.uint8))


def test_groups_added_later_and_empty_tensors():
    (a,), (b,) = _params([40]), _params([0])
    opt = AdamW([a])
    opt.add_param_group({"params": [b], "lr": 0.1})
    a.grad, b.grad = torch.ones(40), torch.ones(0)
    opt.step()
    assert int(opt.state[a]["step"]) == 1 and opt.state[b]["m"].numel() == 0
    loss = opt.step(lambda: torch.tensor(2.0))
    assert float(loss) == 2.0
    opt.add_param_group({"params": []})
    opt.step()
    assert opt.arenas(2) == {} and int(opt.state[a]["step"]) == 3


def test_refusals_change_nothing():
    a, b = _params([6, 8])
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([a], state_bits=4)
    for bad in (dict(lr=-1.0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([a], **bad)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.zeros(4, 6).t().requires_grad_()])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        AdamW([torch.zeros(4, dtype=torch.float64, requires_grad=True)])
    with pytest.raises(ValueError):
        AdamW([a, a])
    opt = AdamW([a, b])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.zeros(3, dtype=torch.float16, requires_grad=True)]})
    assert len(opt.param_groups) == 1
    old = [a.detach().clone(), b.detach().clone()]
    for grads in ([torch.ones(6)], [torch.ones(6), torch.ones(7)], [torch.ones(6), torch.ones(8, dtype=torch.float16)],
                  [torch.ones(6), torch.ones(8).to_sparse()], [torch.ones(6), torch.ones(2, 4)]):
        with pytest.raises(ValueError):
            opt.step(grads=grads)
    with torch.no_grad():
        assert torch.equal(a, old[0]) and torch.equal(b, old[1])
    assert opt.arenas()["step"].tolist() == [0, 0]
    saved = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError):
        AdamW([a, b], state_bits=8).load_state_dict(saved)
    with pytest.raises(ValueError):
        AdamW([a]).load_state_dict(saved)
    with pytest.raises(TypeError):
        pickle.dumps(opt)
    a.data = a.data.to(torch.bfloat16)
    with pytest.raises(ValueError, match="has changed"):
        opt.step(grads=[torch.ones(6), torch.ones(8)])


def test_the_tensors_version_advances_so_that_a_stale_backward_is_refused():
    (a,) = _params([4])
    opt = AdamW([a])
    loss = (a * a).sum()
    a.grad = torch.ones(4)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
