"""AdamW (Adam with decoupled weight decay) over many tensors at once, moments in 32 or in 8 bits.

    m = b1*m + (1-b1)*g ;  v = b2*v + (1-b2)*g*g
    p = p*(1 - lr*weight_decay) - lr * (m / (1-b1^t)) / (sqrt(v / (1-b2^t)) + eps)

On a GPU a step is two kernels (``csrc/hip/adamw.hip``; the first once for every 200 tensors, the second once for every pair of parameter and
gradient types in use): the parameters and gradients stay where the
program has them, contiguous fp32 or bf16 tensors in any mix, and the moments live in arenas in which every tensor starts at a
multiple of 256 elements.  The step counters are on the device, so a captured step advances when it is replayed (with the learning rate and
the other settings that it was captured with).  Steps over different parameters of one optimizer share nothing that is written, and may
run at once: on two streams, or as two captured graphs.  bf16 parameters
are updated in fp32 and rounded to nearest: an update below half a bf16 step of its parameter is lost, so keep fp32 parameters
where that matters.

``state_bits=8``: m and r = sqrt(v) are held as e4m3 with one power of two for every 256 elements, rounded stochastically (to
nearest, the slow average of v would freeze: a step moves r by 0.05 %, the grid is 6-12 %) from a hash of ``seed``, step and place, so
a run can be repeated bit for bit.  A moment that is not finite is held as NaN.  On the CPU the same arithmetic runs as torch
operations.
"""
from __future__ import annotations

import math
from typing import Dict, Iterable, Optional, Sequence

import torch

from .. import native

BLOCK = 256    # elements that share a scale; tensors start at multiples of it (BLOCK, CHUNK: csrc/hip/adamw.hip)
CHUNK = 2048   # elements of a workgroup
E4M3 = torch.float8_e4m3fn


def _i32(x: int) -> int:
    """A 32-bit constant as torch's int32 takes it."""
    x &= 0xFFFFFFFF
    return x - (1 << 32) if x >> 31 else x


class _Group:
    """The moments and tables of one parameter group."""

    def __init__(self, params: Sequence[torch.Tensor], bits: int, seed: int):
        self.params, self.bits, self.seed = list(params), bits, seed & 0xFFFFFFFF
        self.device = params[0].device
        self.sizes = [p.numel() for p in params]
        self.dtypes = [p.dtype for p in params]
        self.at = [0]
        for n in self.sizes:
            self.at.append(self.at[-1] + -(-n // BLOCK) * BLOCK)
        total, dev = self.at[-1], self.device
        self.step = torch.zeros(len(params), dtype=torch.int32, device=dev)
        if bits == 32:
            self.arenas = {"m": torch.zeros(total, device=dev), "v": torch.zeros(total, device=dev)}
        else:
            tiny = torch.full((total // BLOCK,), 2.0 ** -126, device=dev)  # (what the scale of a block of zeros is)
            self.arenas = {"m": torch.zeros(total, dtype=torch.uint8, device=dev).view(E4M3), "m_scale": tiny,
                           "r": torch.zeros(total, dtype=torch.uint8, device=dev).view(E4M3), "r_scale": tiny.clone()}
        if self.device.type == "cuda":
            counts = torch.tensor([-(-n // CHUNK) for n in self.sizes])
            owner = torch.repeat_interleave(torch.arange(len(self.sizes)), counts)
            first = torch.cumsum(counts, 0) - counts
            self.chunks = torch.stack((owner, torch.arange(owner.numel()) - first[owner]), 1).to(torch.int32).to(dev)
            self.shape = torch.tensor(list(zip(self.sizes, self.at)), dtype=torch.int64).to(dev)
            places = {"shape": self.shape, "chunks": self.chunks, "step": self.step, **self.arenas}
            self.native = native.ext().AdamWGroup(self.params, {k: t.data_ptr() for k, t in places.items()}, self.chunks.shape[0], bits, self.seed)

    def views(self, i: int) -> Dict[str, torch.Tensor]:
        """Tensor i's part of the arenas, to the end of its last block."""
        lo, hi = self.at[i], self.at[i + 1]
        out = {"step": self.step[i:i + 1]}
        for k, t in self.arenas.items():
            out[k] = t[lo // BLOCK:hi // BLOCK] if k.endswith("scale") else t[lo:hi]
        return out

    def gather(self, given: Optional[Sequence[Optional[torch.Tensor]]]) -> bool:
        """Takes the parameters' gradients, or the given ones; what does not fit the group is refused here, before anything is changed.
        Whether there is one at all."""
        if self.device.type == "cuda":
            return self.native.gather(given)
        self.grads = []
        for p, g, n, dt in zip(self.params, [p.grad for p in self.params] if given is None else given, self.sizes, self.dtypes):
            if p.dtype != dt or p.numel() != n or p.device != self.device or not p.is_contiguous():
                raise ValueError("a parameter's type, size, device or layout has changed since it was given to AdamW")
            if g is not None:
                if g.dtype not in (torch.float32, torch.bfloat16) or g.layout != torch.strided:
                    raise ValueError("gradients are dense float32 or bfloat16 tensors (got %s, %s)" % (g.dtype, g.layout))
                if g.device != self.device or g.shape != p.shape:
                    raise ValueError("a gradient of shape %s on %s for a parameter of shape %s on %s"
                                     % (tuple(g.shape), g.device, tuple(p.shape), self.device))
            self.grads.append(g if n else None)
        return any(g is not None for g in self.grads)

    def apply(self, o: dict, grad_scale: float) -> None:
        """One step from the gradients that ``gather`` took."""
        if self.device.type == "cuda":
            self.native.launch(o["lr"], o["beta1"], o["beta2"], o["eps"], o["weight_decay"], grad_scale)
        else:
            grads, self.grads = self.grads, None
            self._eager(grads, o, grad_scale)

    # ------------------------------------------------------------------ CPU
    def _eager(self, grads, o, grad_scale) -> None:
        b1, b2 = o["beta1"], o["beta2"]
        for i, (p, g, n) in enumerate(zip(self.params, grads, self.sizes)):
            if g is None:
                continue
            st = self.views(i)
            st["step"] += 1
            t = int(st["step"])
            g = g.reshape(-1).float() * grad_scale
            m, v = self._moments(st)
            m[:n] = m[:n] * b1 + g * (1.0 - b1)
            v[:n] = v[:n] * b2 + (g * g) * (1.0 - b2)
            r = v.double().sqrt().float()  # (torch's float32 root is not the nearest one)
            step = m[:n] / (r[:n] * (1.0 / math.sqrt(1.0 - b2 ** t)) + o["eps"])
            new = p.reshape(-1).float() * (1.0 - o["lr"] * o["weight_decay"]) - step * (o["lr"] / (1.0 - b1 ** t))
            p.copy_(new.view_as(p))
            if self.bits == 32:
                st["m"].copy_(m)
                st["v"].copy_(v)
            else:
                rnd = self._random(t, self.at[i] // BLOCK, m.numel() // BLOCK)
                self._hold(st["m"], st["m_scale"], m, rnd & 0xFFFF, False)
                self._hold(st["r"], st["r_scale"], r, (rnd >> 16) & 0xFFFF, True)

    def _moments(self, st):
        if self.bits == 32:
            return st["m"].clone(), st["v"].clone()
        wide = lambda c, s: (c.float().view(-1, BLOCK) * s[:, None]).reshape(-1)  # noqa: E731
        return wide(st["m"], st["m_scale"]), wide(st["r"], st["r_scale"]).square()

    def _random(self, t: int, block: int, count: int) -> torch.Tensor:
        """adamw.hip's random bits of ``count`` blocks from ``block`` on: int32 [count, BLOCK] (products wrap)."""
        def mix(x):
            x = (x ^ ((x >> 16) & 0xFFFF)) * _i32(0x6A09E667)
            x = (x ^ ((x >> 15) & 0x1FFFF)) * _i32(0xBB67AE85)
            return x ^ ((x >> 16) & 0xFFFF)
        key = mix(torch.tensor([_i32(self.seed + t * 0x9E3779B9)], dtype=torch.int32))
        key = mix(key ^ torch.arange(block, block + count, dtype=torch.int32))
        return mix(key[:, None] + torch.arange(BLOCK, dtype=torch.int32))

    @staticmethod
    def _hold(codes, scales, x, rnd, keep_positive: bool) -> None:
        x = x.view(-1, BLOCK)
        bits = x.view(torch.int32) & 0x7FFFFFFF
        finite = bits < 0x7F800000
        field = (torch.where(finite, bits, 0).amax(1) >> 23).clamp_(min=8)
        a = x.abs() * ((261 - field) << 23).view(torch.float32)[:, None]
        # 16 random bits are added right below the three mantissa bits that stay, and what is below those is cut.  Under 2^-6 the grid is
        # 2^-9; one binade up a float has that grid, so 2^-6 is added there (to a multiple of 2^-29: what the sum would round is cut)
        low = a < 2.0 ** -6
        up = torch.floor(a * 2.0 ** 29) * 2.0 ** -29 + 2.0 ** -6
        c = ((torch.where(low, up, a).view(torch.int32) + (rnd << 4)) >> 20) - torch.where(low, 968, 960)
        if keep_positive:
            c = torch.where(x > 0, c.clamp(min=1), c)
        c = torch.where(finite, c, 0x7F) | torch.where(torch.signbit(x), 0x80, 0)
        codes.view(torch.uint8).copy_(c.to(torch.uint8).view(-1))
        scales.copy_(((field - 7) << 23).view(torch.float32))


class AdamW(torch.optim.Optimizer):
    """``AdamW(params, lr, beta1, beta2, eps, weight_decay, state_bits=32 | 8, seed)``; parameter groups as in ``torch.optim``
    (each its own ``lr``, ``beta1``, ``beta2``, ``eps``, ``weight_decay``; a group's tensors share a device).  A parameter without a
    gradient is left alone, its step counter too."""

    def __init__(self, params: Iterable, lr: float = 1e-3, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is 8 or 32 (got %r)" % (state_bits,))
        self.state_bits, self.seed, self._groups = state_bits, int(seed), []
        super().__init__(params, dict(lr=lr, beta1=beta1, beta2=beta2, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        grp = self.param_groups[-1]
        try:
            self._check(grp)
            st = _Group(grp["params"], self.state_bits, self.seed + 0x632BE5AB * len(self._groups)) if grp["params"] else None
        except Exception:
            self.param_groups.pop()
            raise
        self._groups.append(st)
        for i, p in enumerate(grp["params"]):
            self.state[p] = st.views(i)

    @staticmethod
    def _check(grp: dict) -> None:
        if not (grp["lr"] >= 0 and grp["eps"] >= 0 and grp["weight_decay"] >= 0 and 0 <= grp["beta1"] < 1 and 0 <= grp["beta2"] < 1):
            raise ValueError("lr, eps and weight_decay are not negative, beta1 and beta2 lie in [0, 1): %r"
                             % {k: v for k, v in grp.items() if k != "params"})
        if len(set(map(id, grp["params"]))) < len(grp["params"]):
            raise ValueError("a parameter is twice in one group")
        for p in grp["params"]:
            if p.dtype not in (torch.float32, torch.bfloat16) or p.layout != torch.strided or not p.is_contiguous() or p.is_neg():
                raise ValueError("AdamW takes contiguous float32 or bfloat16 parameters (got %s, strides %s)" % (p.dtype, tuple(p.stride())))
            if p.device != grp["params"][0].device or p.device.type not in ("cpu", "cuda"):
                raise ValueError("a group's parameters share one device, a GPU or the CPU")

    def arenas(self, group: int = 0) -> Dict[str, torch.Tensor]:
        """The group's live moments: ``m`` and ``v`` (fp32), or ``m`` and ``r`` = sqrt(v) (e4m3) with ``m_scale`` and ``r_scale``, one
        for 256 elements; and the step counters, one a tensor.  Tensor i starts at a multiple of 256 elements."""
        st = self._groups[group]
        return {} if st is None else {**st.arenas, "step": st.step}

    @torch.no_grad()
    def step(self, closure=None, *, grads: Optional[Sequence[Optional[torch.Tensor]]] = None, grad_scale: float = 1.0):
        """One update from the parameters' ``grad``, or from ``grads``: one tensor or None for every parameter in the groups' order,
        where they are kept elsewhere or in another type.  ``grad_scale`` multiplies them (1 / ranks, 1 / loss scale)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grads is not None and len(grads) != sum(len(g["params"]) for g in self.param_groups):
            raise ValueError("%d gradients for %d parameters" % (len(grads), sum(len(g["params"]) for g in self.param_groups)))
        todo, at = [], 0
        for o, st in zip(self.param_groups, self._groups):
            if st is not None:
                given = None if grads is None else list(grads[at:at + len(st.params)])
                at += len(st.params)
                if st.gather(given):
                    todo.append((o, st))
        for o, st in todo:
            st.apply(o, grad_scale)
        return loss

    # ------------------------------------------------------------------ state
    def load_state_dict(self, state_dict: dict) -> None:
        """Copies a ``state_dict()`` of the same parameters and ``state_bits`` into the arenas (the base class would replace them by
        tensors of the parameters' types)."""
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state's groups have other numbers of parameters")
        copies = []
        for saved, grp in zip(groups, self.param_groups):
            for key, p in zip(saved["params"], grp["params"]):
                mine, theirs = self.state[p], state_dict["state"].get(key, {})
                if {k: (t.dtype, t.shape) for k, t in mine.items()} != {k: (t.dtype, t.shape) for k, t in theirs.items()}:
                    raise ValueError("the state of a parameter of shape %s does not fit (another size, or other state_bits)" % (tuple(p.shape),))
                copies += [(mine[k], theirs[k]) for k in mine]
        for mine, theirs in copies:
            mine.copy_(theirs)
        for saved, grp in zip(groups, self.param_groups):
            grp.update({k: v for k, v in saved.items() if k != "params"})

    def __getstate__(self):
        raise TypeError("AdamW is saved by state_dict(): its tables hold device addresses")
