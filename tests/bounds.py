"""Running error analysis in 64 bits: a value beside a bound of what an fp32
evaluation of the same formula may be off by.  Every operation adds U of its
result: 2^-23, twice fp32's half step, as kernels may take products and sums in
another order or fused.  A sum's terms add U per operation of the longest chain
that they pass."""
import torch

U = 2.0 ** -23
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}   # half a step near 0


class E:
    def __init__(self, v, e=0.0):
        self.v = v.double() if isinstance(v, torch.Tensor) else torch.tensor(float(v), dtype=torch.float64)
        self.e = torch.as_tensor(e, dtype=torch.float64, device=self.v.device)

    @staticmethod
    def of(x):
        return x if isinstance(x, E) else E(x)

    def to(self, device):
        return E(self.v.to(device), self.e.to(device))

    def _pair(self, other):
        o = E.of(other)
        return o if o.v.device == self.v.device else o.to(self.v.device)

    def __add__(self, other):
        o = self._pair(other)
        v = self.v + o.v
        return E(v, self.e + o.e + U * v.abs())

    def __sub__(self, other):
        o = self._pair(other)
        return self + E(-o.v, o.e)

    def __mul__(self, other):
        o = self._pair(other)
        v = self.v * o.v
        return E(v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e + U * v.abs())

    __radd__, __rmul__ = __add__, __mul__

    def sum(self, dim, chain, keepdim=True):
        return E(self.v.sum(dim, keepdim=keepdim),
                 self.e.expand(self.v.shape).sum(dim, keepdim=keepdim) + U * chain * self.v.abs().sum(dim, keepdim=keepdim))

    def mean(self, chain):
        return self.sum(-1, chain) * (1.0 / self.v.shape[-1])

    def rsqrt(self):
        """1/sqrt; its relative error is half the argument's, which may be large where the argument is small."""
        y = 1 / torch.sqrt(self.v)
        rel = (self.e / self.v).clamp(max=0.75)
        return E(y, y * (1 / torch.sqrt(1 - rel) - 1 + 4 * U))

    def rounded(self, t):
        """What a store of type t makes of it (fp32 has its U already)."""
        return self if t is torch.float32 else E(self.v, self.e + torch.finfo(t).eps / 2 * (self.v.abs() + self.e) + TINY[t])

    def where(self, cond):
        return E(torch.where(cond, self.v, 0.0), torch.where(cond, self.e, 0.0))

    def view(self, *s):
        return E(self.v.reshape(*s), self.e.expand(self.v.shape).reshape(*s))


def worst(got, want):
    """The largest error of `got` over its bound, the rounding to its type included."""
    assert tuple(got.shape) == tuple(want.v.shape), (got.shape, want.v.shape)
    if got.numel() == 0:
        return 0.0
    w = want.rounded(got.dtype)
    bound = w.e.expand(w.v.shape) + TINY[got.dtype] + U * w.v.abs()
    return ((got.double() - w.v).abs() / bound).nan_to_num(nan=float("inf")).max().item()


def norm(x, eps, chain):
    """(x − mean)·rstd and rstd."""
    dev = x - x.mean(chain)
    r = ((dev * dev).mean(chain) + eps).rsqrt()
    return dev * r, r


def norm_back(g, xh, r, chain):
    return (g - g.mean(chain) - xh * (g * xh).mean(chain)) * r
