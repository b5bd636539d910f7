"""AdamW from its definition in float64, with bounds on what 32-bit arithmetic may differ from it."""
import torch

U = 2.0 ** -24  # half a step of float32, relative


def held(st, n):
    """(m, v) that a state stands for, float64, the tensor's own elements."""
    if "v" in st:
        return st["m"][:n].double(), st["v"][:n].double()
    wide = lambda c, s: (c.double().view(-1, 256) * s.double()[:, None]).view(-1)[:n]  # noqa: E731
    return wide(st["m"], st["m_scale"]), wide(st["r"], st["r_scale"]).square()


def step(p, g, m, v, t, lr, b1, b2, eps, wd, grad_scale=1.0):
    """(p, m, v) after step t, and for p and m what their computation in float32 may be off by (rounding of p to bf16 not counted).

    m: the two constants, two products and the sum round once each, on terms of at most S = b1|m| + (1-b1)|g|; grad_scale's product
    once more: 5 U S.  v: as m plus g*g, all terms positive: 7 U v.  r = sqrt(v): 3.5 U + U.  The denominator adds four roundings, the
    quotient, lr1 and its product three more, each relative: |m/d| (4.5 + 4 + 3) U < 12 U |m/d|, plus m's own error over d.
    p: the decay constant and product on |p|, and the difference: 2 U |p| + U |new p|."""
    p, g, m, v = (x.double() for x in (p.reshape(-1), g.reshape(-1), m, v))
    g = g * grad_scale
    s = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    d = (v / (1 - b2 ** t)).sqrt() + eps
    lr1 = lr / (1 - b1 ** t)
    new = p * (1 - lr * wd) - lr1 * m / d
    return new, m, v, U * (2 * p.abs() + new.abs() + lr1 * (12 * m.abs() + 5 * s) / d), 5 * U * s


def grid(x, scale):
    """The spacing of scaled e4m3 at x (float64)."""
    e = torch.floor(torch.log2((x.abs() / scale).clamp(min=2.0 ** -6)))
    return torch.exp2(e - 3) * scale


def check(before, after, p0, p1, g, t, hyper, grad_scale=1.0):
    """Asserts that ``after`` and p1 follow from ``before`` and p0 by one step."""
    n = p0.numel()
    m, v = held(before, n)
    p, m, v, p_off, m_off = step(p0, g, m, v, t, grad_scale=grad_scale, **hyper)
    if p1.dtype == torch.bfloat16:
        p_off = p_off + (p.abs() + p_off) * 2.0 ** -8
    off = (p1.reshape(-1).double() - p).abs()
    assert bool((off <= p_off + 1e-38).all()), ("p", float((off / (p_off + 1e-38)).max()))
    m1, v1 = held(after, n)
    if "v" in after:
        assert bool(((m1 - m).abs() <= m_off + 1e-38).all()) and bool(((v1 - v).abs() <= 7 * U * v + 1e-38).all())
        return
    blocks = lambda s: s.double().repeat_interleave(256)[:n]  # noqa: E731
    r, r1 = v.sqrt(), v1.sqrt()
    for x, x1, s, off in ((m, m1, blocks(after["m_scale"]), m_off), (r, r1, blocks(after["r_scale"]), 5 * U * r)):
        # within one step of the grid, on either side (one step of the upper binade next to a power of two)
        assert bool(((x1 - x).abs() <= torch.maximum(grid(x, s), grid(x1, s)) + off).all())
        f = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1)
        scale = s[::256]
        assert bool((torch.frexp(scale).mantissa == 0.5).all())
        assert bool((f < 256 * scale * (1 + 1e-6)).all()) and bool(((f >= 128 * scale * (1 - 1e-6)) | (scale == 2.0 ** -126)).all())
    assert bool((r1[r > 0] > 0).all())
