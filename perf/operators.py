"""The cases on which the RMS norm, the 4-bit dense layer and AdamW are measured, with each operator's plain form.

``run`` computes an operator from elementary torch operations in 32 bits (``own = False``) or through the framework's entry
points (``own = True``); ``exact`` has the same results from the definitions in 64 bits.  Everything lives on the GPU."""
import math

import torch

own = False

DEV = "cuda"
E4M3 = torch.float8_e4m3fn
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "e4m3": E4M3}
SIZE = {"fp32": 4, "bf16": 2, "e4m3": 1}
EPS = 1e-6
BLOCK = 256                                   # elements that share the scale of their 8-bit moments
LR, BETA1, BETA2, ADAM_EPS, DECAY, T0, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100, 1234
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def listed():
    return [
        # one image's features before a quantised layer: latency
        {"name": "norm_e4m3_1x2048_bf16", "op": "norm_e4m3", "rows": 1, "dim": 2048, "dtype": "bf16", "residual": True},
        # the bottlenecks of an extraction batch, an odd width in float32
        {"name": "norm_e4m3_600x3137_fp32", "op": "norm_e4m3", "rows": 600, "dim": 3137, "dtype": "fp32", "residual": False},
        # a long batch of tokens through an inference norm: bandwidth
        {"name": "norm_fwd_16384x4096_bf16", "op": "norm_fwd", "rows": 16384, "dim": 4096, "dtype": "bf16", "residual": True},
        # a training step at the size of the MNIST network's dense layer: forward and all gradients
        {"name": "norm_train_100x1024_fp32", "op": "norm_train", "rows": 100, "dim": 1024, "dtype": "fp32", "residual": False},
        # a training step over 8192 rows of the Inception bottleneck's width, with the residual stream's gradient
        {"name": "norm_train_8192x2048_bf16", "op": "norm_train", "rows": 8192, "dim": 2048, "dtype": "bf16", "residual": True},
        # one image through Inception's own class layer: latency
        {"name": "w4_1x2048x1008_bf16", "op": "w4", "rows": 1, "k": 2048, "n": 1008, "dtype": "bf16", "group": 32},
        # one token through a wide layer: bandwidth of the weights
        {"name": "w4_1x8192x8192_bf16", "op": "w4", "rows": 1, "k": 8192, "n": 8192, "dtype": "bf16", "group": 64},
        # a few images through a layer of the MNIST network's flattened width, float32 rows, an odd number of outputs
        {"name": "w4_5x3136x1025_fp32", "op": "w4", "rows": 5, "k": 3136, "n": 1025, "dtype": "fp32", "group": 32},
        # a small batch behind the 8-bit norm, the widest layer
        {"name": "w4_16x16384x16384_e4m3", "op": "w4", "rows": 16, "k": 16384, "n": 16384, "dtype": "e4m3", "group": 128},
        # the MNIST network's eight parameters
        {"name": "adamw_mnist_fp32", "op": "adamw", "tensors": 8, "elements": 3274634, "p": "fp32", "g": "fp32", "bits": 32},
        # a network of Inception's size (weights and per-channel vectors), 8-bit moments
        {"name": "adamw_190x24M_fp32_8bit", "op": "adamw", "tensors": 190, "elements": 24000000, "p": "fp32", "g": "fp32", "bits": 8},
        # a large network trained in bf16, 8-bit moments: bandwidth
        {"name": "adamw_64x268M_bf16_8bit", "op": "adamw", "tensors": 64, "elements": 268435456, "p": "bf16", "g": "bf16", "bits": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_e4m3", "norm_fwd", "norm_train", "w4", "w4", "adamw"])
    if op == "w4":
        return {"op": op, "rows": _log(rng, 1, 16), "k": _log(rng, 64, 16384), "n": _log(rng, 10, 16384),
                "dtype": rng.choice(["fp32", "bf16", "e4m3"]), "group": rng.choice([32, 64, 128])}
    if op == "adamw":
        tensors = _log(rng, 1, 200)
        return {"op": op, "tensors": tensors, "elements": _log(rng, max(1000, 40 * tensors), 200000000),
                "p": rng.choice(["fp32", "bf16"]), "g": rng.choice(["fp32", "bf16"]), "bits": rng.choice([8, 32])}
    dim = _log(rng, 16, 8192)
    return {"op": op, "rows": _log(rng, 1, min(16384, 30000000 // dim)), "dim": dim, "dtype": rng.choice(["fp32", "bf16"]),
            "residual": rng.random() < 0.6}


# ----------------------------------------------------------------------------------------------------- inputs
def _sizes(case):
    """Element counts of the case's tensors: the MNIST network's own, or weights of several sizes between short vectors."""
    n, total = case["tensors"], case["elements"]
    if n == 8 and total == 3274634:
        return [3136 * 1024, 1024, 1024 * 10, 10, 5 * 5 * 32 * 64, 64, 5 * 5 * 32, 32]
    small = [0 if i % 2 == 0 else min(total // (4 * n) + 1, 33 + 32 * (i % 13)) for i in range(n)]
    share = [(1 + i % 7) if i % 2 == 0 else 0 for i in range(n)]
    rest = total - sum(small)
    return [s or max(1, rest * w // sum(share)) for s, w in zip(small, share)]


def _offsets(sizes):
    """Every tensor starts at a multiple of BLOCK in the arenas; the last entry is the arenas' length."""
    at = [0]
    for n in sizes:
        at.append(at[-1] + -(-n // BLOCK) * BLOCK)
    return at


def _pow2_scale(amax):
    """The power of two that brings ``amax`` into [128, 256)."""
    field = (amax.float().view(torch.int32) >> 23).clamp_(min=8)
    return ((field - 7) << 23).view(torch.float32)


def _to_e4m3(x):
    blocks = x.view(-1, BLOCK)
    scale = _pow2_scale(blocks.abs().amax(1))
    return (blocks / scale[:, None]).to(E4M3).view(-1), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=gen)  # noqa: E731
    st = {"case": case}
    if case["op"].startswith("norm"):
        rows, dim, dt = case["rows"], case["dim"], DTYPES[case["dtype"]]
        st["x"] = rand(rows, dim).to(dt)
        st["res"] = (3 * rand(rows, dim)).to(dt) if case["residual"] else None
        st["w"] = 1 + 0.2 * rand(dim)
        if case["op"] == "norm_train":
            st["dy"] = rand(rows, dim).to(dt)
            st["dh"] = rand(rows, dim).to(dt) if case["residual"] else None
            for k in ("x", "res", "w"):
                st[k] = st[k] if st[k] is None else st[k].requires_grad_()
    elif case["op"] == "w4":
        m, k, n, group = case["rows"], case["k"], case["n"], case["group"]
        kt, nt = -(-k // 128), -(-n // 16)
        code = torch.randint(0, 256, (nt, kt, 64, 16), device=DEV, generator=gen, dtype=torch.uint8)
        if k % 128 or n % 16:                 # codes behind the last row or column are zero
            full = _untile(code)
            full[k:] = 0
            full[:, n:] = 0
            code = _tile(full)
        st["wq"] = code
        st["scales"] = (torch.rand(nt, kt * 128 // group, 16, device=DEV, generator=gen) * 0.02 + 0.002).to(torch.bfloat16)
        st["bias"] = 0.1 * rand(n)
        x = rand(m, k)
        st["x_scale"] = None
        if case["dtype"] == "e4m3":
            st["x_scale"] = x.abs().amax(1) / 448
            x = x / st["x_scale"][:, None]
        st["x"] = x.to(DTYPES[case["dtype"]])
    else:
        sizes = _sizes(case)
        at = _offsets(sizes)
        inside = torch.zeros(at[-1], device=DEV)
        for a, n in zip(at, sizes):
            inside[a:a + n] = 1
        st["p"] = (0.05 * rand(at[-1]) * inside).to(DTYPES[case["p"]])
        st["g"] = (0.01 * rand(at[-1]) * inside).to(DTYPES[case["g"]])
        m = 0.003 * rand(at[-1]) * inside
        r = 0.01 * torch.exp(0.5 * rand(at[-1])) * inside
        st["step"] = torch.full((len(sizes),), T0, dtype=torch.int32, device=DEV)
        if case["bits"] == 8:
            st["m"], st["m_scale"] = _to_e4m3(m)
            st["r"], st["r_scale"] = _to_e4m3(r)
        else:
            st["m"], st["v"] = m, r * r
        if own:
            from distributed_tensorflow_amd.optim.adamw import AdamW
            params = [st["p"][a:a + n].requires_grad_() for a, n in zip(at, sizes)]
            for p, a, n in zip(params, at, sizes):
                p.grad = st["g"][a:a + n] if case["g"] == case["p"] else None
                st.setdefault("grads", []).append(st["g"][a:a + n])
            opt = AdamW(params, lr=LR, beta1=BETA1, beta2=BETA2, eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
            st["arenas"] = opt.arenas()
            for k, t in st["arenas"].items():
                t.copy_(st[k])
            st["opt"] = opt
    return st


# ----------------------------------------------------------------------------------------------------- plain forms
def _tile(code):
    """Codes [Kp, Np] (values 0..15) to the layout of the 4-bit weights, [Np/16, Kp/128, 64, 16] bytes."""
    kp, np_ = code.shape
    c = code.view(kp // 128, 4, 4, 4, 2, np_ // 16, 16)                 # kt, j, kb, pair, half, nt, n
    c = c.permute(5, 0, 2, 6, 1, 3, 4).reshape(np_ // 16, kp // 128, 64, 16, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _untile(wq):
    nt, kt = wq.shape[:2]
    c = torch.stack((wq & 15, wq >> 4), -1).view(nt, kt, 4, 16, 4, 4, 2)  # nt, kt, kb, n, j, pair, half
    return c.permute(1, 4, 2, 5, 6, 0, 3).reshape(kt * 128, nt * 16)


def _norm(st):
    h = st["x"].float() + st["res"].float() if st["res"] is not None else st["x"].float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    return h, rstd, h * rstd * st["w"]


def _plain_norm(st, case):
    dt = DTYPES[case["dtype"]]
    with torch.no_grad():
        h, rstd, y = _norm(st)
        out = {"h": h.to(dt)} if case["residual"] else {}
        if case["op"] == "norm_e4m3":
            scale = y.abs().amax(1) / 448
            return {**out, "q": (y / torch.where(scale > 0, scale, 1.0)[:, None]).to(E4M3), "scale": scale}
        out["y"] = y.to(dt)
        if case["op"] == "norm_train":
            g = st["dy"].float() * st["w"]
            dx = rstd * (g - h * (rstd * rstd * (g * h).mean(1, keepdim=True)))
            if case["residual"]:
                dx = dx + st["dh"].float()
            out["dx"] = dx.to(dt)
            out["dw"] = (st["dy"].float() * (h * rstd)).sum(0)
        return out


def _own_norm(st, case):
    from distributed_tensorflow_amd.ops import autograd, hip_ops
    if case["op"] == "norm_e4m3":
        q, scale, h = hip_ops.rms_norm_e4m3(st["x"], st["w"], st["res"], eps=EPS)
        return {"q": q, "scale": scale, **({"h": h} if case["residual"] else {})}
    if case["op"] == "norm_fwd":
        y, h, _ = hip_ops.rms_norm_forward(st["x"], st["w"], st["res"], eps=EPS)
        return {"y": y, **({"h": h} if case["residual"] else {})}
    if case["residual"]:
        y, h = autograd.rms_norm(st["x"], st["w"], st["res"], eps=EPS)
        dx, dres, dw = torch.autograd.grad((y, h), (st["x"], st["res"], st["w"]), (st["dy"], st["dh"]))
        return {"y": y, "h": h, "dx": dx, "dw": dw}
    y = autograd.rms_norm(st["x"], st["w"], eps=EPS)
    dx, dw = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def _weights(st, case, dt):
    """The [K, N] weights that the codes and scales stand for."""
    w = torch.tensor(E2M1, device=DEV, dtype=dt)[_untile(st["wq"])[:case["k"], :case["n"]].int()]
    s = st["scales"].to(dt).permute(1, 0, 2).reshape(st["scales"].shape[1], -1)
    return w * s.repeat_interleave(case["group"], 0)[:case["k"], :case["n"]]


def _plain_w4(st, case, dt=torch.float32):
    y = st["x"].to(dt) @ _weights(st, case, dt)
    if st["x_scale"] is not None:
        y = y * st["x_scale"].to(dt)[:, None]
    return {"y": y + st["bias"].to(dt)}


def _own_w4(st, case):
    from distributed_tensorflow_amd.ops import hip_ops
    return {"y": hip_ops.linear_w4(st["x"], st["wq"], st["scales"], case["n"], bias=st["bias"], x_scale=st["x_scale"])}


def _mix(x):
    """A hash of 32-bit integers (held in int32, products wrap): xor-shift and odd multipliers, digits of sqrt(2) and sqrt(3)."""
    x = (x ^ ((x >> 16) & 0xFFFF)) * 0x6A09E667
    x = (x ^ ((x >> 15) & 0x1FFFF)) * (0xBB67AE85 - (1 << 32))
    return x ^ ((x >> 16) & 0xFFFF)


def _random(step, blocks):
    """32 random bits an element, int32 [blocks, BLOCK], from the seed, the step and the element's place in the arena."""
    key = _mix(torch.full((1,), SEED, dtype=torch.int32, device=DEV) + step * (0x9E3779B9 - (1 << 32)))
    key = _mix(key ^ torch.arange(blocks, dtype=torch.int32, device=DEV))
    return _mix(key[:, None] + torch.arange(BLOCK, dtype=torch.int32, device=DEV))


def _stochastic(x, bits, at_least=None):
    """``x`` [blocks, BLOCK] as e4m3 values and their blocks' scales, rounded up where the 16 random bits say so."""
    scale = _pow2_scale(x.abs().amax(1))
    a = (x / scale[:, None]).abs()
    low = a < 2.0 ** -6                       # the subnormal grid of 2^-9: one binade up it has the same three bits
    u = torch.where(low, a + 2.0 ** -6, a).view(torch.int32) + (bits << 4)
    q = (u & -(1 << 20)).view(torch.float32) - torch.where(low, 2.0 ** -6, 0.0)
    if at_least is not None:
        q = torch.where(x > 0, q.clamp(min=at_least), q)
    return torch.copysign(q, x).to(E4M3).view(-1), scale


def _plain_adamw(st, case):
    st["step"] += 1
    t = st["step"][0].double()
    c1, c2 = 1 - BETA1 ** t, 1 - BETA2 ** t
    g, p = st["g"].float(), st["p"].float()
    eight = case["bits"] == 8
    if eight:
        m = (st["m"].float().view(-1, BLOCK) * st["m_scale"][:, None]).view(-1)
        v = (st["r"].float().view(-1, BLOCK) * st["r_scale"][:, None]).view(-1).square()
    else:
        m, v = st["m"], st["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    r = v.sqrt()
    p = p * (1 - LR * DECAY) - (LR / c1).float() * (m / (r / c2.sqrt().float() + ADAM_EPS))
    st["p"].copy_(p)
    if not eight:
        st["m"].copy_(m)
        st["v"].copy_(v)
        return {"p": st["p"], "m": st["m"], "v": st["v"]}
    bits = _random(st["step"][0], m.numel() // BLOCK)
    st["m"], st["m_scale"] = _stochastic(m.view(-1, BLOCK), bits & 0xFFFF)
    st["r"], st["r_scale"] = _stochastic(r.view(-1, BLOCK), (bits >> 16) & 0xFFFF, 2.0 ** -9)
    return {"p": st["p"], "m": st["m"], "m_scale": st["m_scale"], "r": st["r"], "r_scale": st["r_scale"]}


def _own_adamw(st, case):
    if case["g"] == case["p"]:
        st["opt"].step()
    else:                                     # gradients of another type than the parameters'
        st["opt"].step(grads=st["grads"])
    return {"p": st["p"].detach(), **{k: t for k, t in st["arenas"].items() if k != "step"}}


def run(st):
    case = st["case"]
    if own:
        return (_own_w4 if case["op"] == "w4" else _own_adamw if case["op"] == "adamw" else _own_norm)(st, case)
    return (_plain_w4 if case["op"] == "w4" else _plain_adamw if case["op"] == "adamw" else _plain_norm)(st, case)


# ----------------------------------------------------------------------------------------------------- definitions, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "w4":
            return _plain_w4(st, case, torch.float64)
        if case["op"] == "adamw":
            return _exact_adamw(st, case)
        x, w = st["x"].double(), st["w"].double()
        h = x if st["res"] is None else x + st["res"].double()
        ms = h.pow(2).sum(1) / case["dim"] + EPS
        unit = h / ms.sqrt()[:, None]
        y = unit * w
        out = {"h": h} if case["residual"] else {}
        if case["op"] == "norm_e4m3":
            scale = y.abs().max(1).values / 448
            return {**out, "q": y / scale[:, None], "scale": scale}
        out["y"] = y
        if case["op"] == "norm_train":
            dy = st["dy"].double()
            du = dy * w                       # through unit = h / |h|: the part along h falls out
            dx = (du - unit * (du * unit).sum(1, keepdim=True) / case["dim"]) / ms.sqrt()[:, None]
            out["dx"] = dx + st["dh"].double() if case["residual"] else dx
            out["dw"] = (dy * unit).sum(0)
        return out


def _exact_adamw(st, case):
    blocks = lambda x: x.view(-1, BLOCK)  # noqa: E731
    g, p = st["g"].double(), st["p"].double()
    if case["bits"] == 8:
        m = (blocks(st["m"].double()) * st["m_scale"].double()[:, None]).view(-1)
        v = (blocks(st["r"].double()) * st["r_scale"].double()[:, None]).pow(2).view(-1)
    else:
        m, v = st["m"].double(), st["v"].double()
    m = m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v = v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    t = T0 + 1
    step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    out = {"p": p - LR * (step + DECAY * p)}
    if case["bits"] == 32:
        return {**out, "m": m, "v": v}
    r = v.sqrt()                              # the held values before they are rounded to 8 bits
    ms, rs = _pow2_scale(blocks(m).abs().amax(1)), _pow2_scale(blocks(r).amax(1))
    # (the scales are powers of two picked by the 32-bit maximum: a maximum next to a power of two has no value in between)
    return {**out, "m": (blocks(m) / ms[:, None]).view(-1), "m_scale": None, "r": (blocks(r) / rs[:, None]).view(-1), "r_scale": None}


def work(case):
    if case["op"] == "w4":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": k * n * (0.5 + 2.0 / case["group"]) + m * k * SIZE[case["dtype"]] + 4 * m * n + 4 * n, "flops": 2.0 * m * k * n}
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        held = 8 if case["bits"] == 32 else 2 + 8.0 / BLOCK
        return {"bytes": n * (2 * SIZE[case["p"]] + SIZE[case["g"]] + 2 * held), "flops": 20.0 * n}
    e, size = case["rows"] * case["dim"], SIZE[case["dtype"]]
    res = int(case["residual"])
    if case["op"] == "norm_train":            # x, res, y, h; dy, dh, dx (h is what the backward pass reads)
        return {"bytes": e * size * (2 + 2 * res + 3 + res), "flops": 20.0 * e}
    return {"bytes": e * (size * (1 + 2 * res) + (1 if case["op"] == "norm_e4m3" else size)), "flops": 8.0 * e}
