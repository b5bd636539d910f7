"""The RMS norm in float64 from its definition, and bounds on what 32-bit arithmetic and the outputs' rounding may add."""
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def forward(x, w, res, eps):
    x, w = x.double(), w.double()
    h = x if res is None else x + res.double()
    rstd = 1 / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return h * rstd * w, h, rstd


def check_forward(y, h, rstd, x, w, res, eps):
    """h: one rounding of the sum in float32 and one of the output's type.  The mean of squares of rows of D: every square carries h's
    rounding twice and its own, every partial sum (at most 32 in a thread, 6 + 5 joining) one, all terms positive: below 64 U; the root
    halves that; quotient, root and mean round once each: rstd within 40 U.  y: h's, rstd's and two products': 44 U, then its type."""
    Y, H, R = forward(x, w, res, eps)
    d = x.dtype
    tiny = 1e-37
    assert bool(((h.double() - H).abs() <= H.abs() * (HALF[d] + 2 * U) + tiny).all())
    assert bool(((rstd.double() - R[..., 0]).abs() <= R[..., 0] * 40 * U).all())
    assert bool(((y.double() - Y).abs() <= Y.abs() * (HALF[d] * (1 + 50 * U) + 46 * U) + tiny).all())


def check_e4m3(q, scale, x, w, res, eps):
    Y, _, _ = forward(x, w, res, eps)
    top = Y.abs().amax(-1)
    assert bool(((scale.double() - top / 448).abs() <= top / 448 * 50 * U).all())
    want = Y / torch.where(scale > 0, scale, 1.0).double()[..., None]
    # half a step of e4m3, relative 2^-4, or of its subnormal grid of 2^-9
    assert bool(((q.double() - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, device=q.device)) * (1 + 1e-4) + 1e-4 * 2.0 ** -10).all())


def check_backward(dx, dw, dy, x, rstd, w, res, dh):
    """From rstd as it was saved.  Every term of mean(g h rstd) carries 4 roundings and those of its sums (below 48): 64 U of the
    mean of magnitudes, on top of a few for the rest: dx within 64 U of the magnitudes of its terms, and its type's rounding.
    dw: terms of 3 roundings, and the sums over rows (a workgroup's rows / 512, four waves, 512 / 16 rows of partial sums, 16 waves; up to 512 rows
    a thread's rows / 16 and 16 sets: 48)."""
    h64, dy64, w64, rstd = x.double() + (0.0 if res is None else res.double()), dy.double(), w.double(), rstd.double()[..., None]
    dim, d = x.shape[-1], x.dtype
    n, g = h64 * rstd, dy64 * w64
    want = rstd * (g - n * (g * n).mean(-1, keepdim=True))
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    if dh is not None:
        want, size = want + dh.double(), size + dh.double().abs()
    assert bool(((dx.double() - want).abs() <= want.abs() * HALF[d] + size * 64 * U * (1 + HALF[d]) + 1e-37).all())
    if dw is not None:
        t = (dy64 * n).reshape(-1, dim)
        assert bool(((dw.double() - t.sum(0)).abs() <= t.abs().sum(0) * (60 + t.shape[0] / 512) * U + 1e-37).all())
