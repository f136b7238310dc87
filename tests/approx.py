"""Values with a bound on their error: the arithmetic of a kernel that computes in fp32, followed in 64 bits.

An `Approx` holds what a formula gives exactly (fp64) and how far an fp32 evaluation of it, in any order of its sums, may be from that:
every operation adds u = 2^-24 times the magnitude of its result to what its operands bring along (first-order running error analysis;
the factor SLACK covers the products of two errors).  A tolerance read off it is derived from the inputs, not from a kernel's outputs."""
import torch

U = 2.0 ** -24
SLACK = 1.01


class Approx:
    def __init__(self, v, e=None):
        self.v = v
        self.e = torch.zeros_like(v) if e is None else e

    @staticmethod
    def of(x):
        return x if isinstance(x, Approx) else Approx(torch.as_tensor(x, dtype=torch.float64))

    @staticmethod
    def _new(v, e, ulps=1.0):
        return Approx(v, SLACK * e + ulps * U * v.abs())

    def __add__(self, o):
        o = Approx.of(o)
        return Approx._new(self.v + o.v, self.e + o.e)

    def __sub__(self, o):
        o = Approx.of(o)
        return Approx._new(self.v - o.v, self.e + o.e)

    def __mul__(self, o):
        o = Approx.of(o)
        return Approx._new(self.v * o.v, self.v.abs() * o.e + o.v.abs() * self.e)

    def sum(self, dim):
        """A sum of n terms in any order: n - 1 additions of partial sums no larger than the sum of the magnitudes."""
        n = self.v.shape[dim]
        mag = self.v.abs().sum(dim, keepdim=True)
        return Approx(self.v.sum(dim, keepdim=True), SLACK * self.e.sum(dim, keepdim=True) + n * U * mag)

    def mean(self, dim):
        return self.sum(dim) * (1.0 / self.v.shape[dim])

    def rsqrt(self):
        """1 / sqrt within 2 units in the last place (4 u); the derivative carries the argument's error."""
        r = self.v.rsqrt()
        return Approx._new(r, 0.5 * r ** 3 * self.e, 4.0)

    def sqrt(self):
        r = self.v.sqrt()
        return Approx._new(r, torch.where(r > 0, 0.5 * self.e / r.clamp_min(1e-300), self.e.sqrt()), 2.0)

    def __truediv__(self, o):
        """A quotient within 1.5 units in the last place (3 u)."""
        o = Approx.of(o)
        q = self.v / o.v
        return Approx._new(q, (self.e + q.abs() * o.e) / o.v.abs(), 3.0)

    def sigmoid(self, fast=False):
        """1 / (1 + exp(-v)): exp within 2 units in the last place, one sum, a reciprocal within 1: 8 u covers them.  fast: exp(-v) as
        exp2 of the rounded product v log2(e): the product is off by u |v| log2(e), log2(e) itself by u relative, so the power by
        ln 2 (2 u |v| log2(e)) = 2 u |v| relative, and the sigmoid by at most as much."""
        a = torch.sigmoid(self.v)
        return Approx._new(a, a * (1.0 - a) * self.e, 8.0 + (2.0 * self.v.abs() if fast else 0.0))

    def view(self, *shape):
        return Approx(self.v.reshape(*shape), self.e.expand_as(self.v).reshape(*shape))


def assert_within(got, want, name=""):
    """got (any floating type) against an Approx: its error bound, plus half a step of got's type for the rounding at the store."""
    v = want.v.to(got.device)
    fi = torch.finfo(got.dtype)
    tol = want.e.expand_as(want.v).to(got.device) + 0.5 * fi.eps * v.abs() + 0.5 * fi.smallest_normal * fi.eps
    assert got.shape == v.shape, (name, tuple(got.shape), tuple(v.shape))
    off = (got.double() - v).abs()
    bad = ~(off <= tol * (1 + 1e-6))
    bad &= ~(torch.isnan(v) & torch.isnan(got.double()))
    bad &= ~(torch.isinf(v) & (got.double() == v))
    if bool(bad.any()):
        i = int(torch.where(bad.reshape(-1))[0][0])
        raise AssertionError("%s: %d of %d outside; first at %d: got %r, want %r +- %r" % (
            name, int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]), float(v.reshape(-1)[i]), float(tol.reshape(-1)[i])))
