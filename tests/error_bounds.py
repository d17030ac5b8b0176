"""Values in 64 bits with a bound of how far an fp32 computation of them may be off, carried through the operations: every
fp32 operation rounds by at most half a step (2^-24 of its result), a sum of n terms in any order by at most n 2^-24 of the
sum of their magnitudes, and a result held in a type by half a step of it (eps / 2) or half its least number."""

import torch

STEP = 2.0**-24


class Bounded:
    def __init__(self, value, error=None):
        self.v = value.double()
        self.e = torch.zeros_like(self.v) if error is None else error

    @property
    def most(self):
        return self.v.abs() + self.e

    def rounded(self):
        return Bounded(self.v, self.e + STEP * self.most)

    def __add__(self, o):
        return Bounded(self.v + o.v, self.e + o.e).rounded()

    def __sub__(self, o):
        return Bounded(self.v - o.v, self.e + o.e).rounded()

    def __mul__(self, o):
        if not isinstance(o, Bounded):
            o = Bounded(torch.as_tensor(o, dtype=torch.float64, device=self.v.device), STEP * torch.tensor(abs(o)).to(self.v.device))
        return Bounded(self.v * o.v, self.most * o.e + self.e * o.v.abs()).rounded()

    def sum(self, dim, keepdim=False):
        n = self.v.shape[dim]
        return Bounded(self.v.sum(dim, keepdim), (self.e + n * STEP * self.most).sum(dim, keepdim))

    def mean(self):
        return self.sum(-1, True) * (1.0 / self.v.shape[-1])

    def over_root(self, eps):
        """1 / sqrt(self + eps), self >= 0."""
        x = Bounded(self.v + eps, self.e + STEP * eps).rounded()
        r = 1.0 / x.v.sqrt()
        low = (x.v - x.e).clamp_min(1e-300)
        return Bounded(r, (1.0 / low.sqrt() - r) + 3 * STEP * r)

    def held(self, dtype):
        info = torch.finfo(dtype)
        return Bounded(self.v, self.e + info.eps / 2 * self.most + info.smallest_normal * info.eps / 2)

    def holds(self, got):
        return bool(((got.double().cpu() - self.v.cpu()).abs() <= self.e.cpu()).all())
