"""A paged cache held in 8 bits for the tests: what its codes are, from the definition
(bits and whole numbers, no cast of the library's), and a ragged batch over one."""
import math

import torch

from ragged import DEV, HND, I32, NEG, NHD, Ragged, i32, within

E4M3 = torch.float8_e4m3fn
LOW, HIGH, MOST = -15, 8, 61440.0


def exponent(top):
    """The smallest e with top <= 448 * 2^e, held to LOW .. HIGH (fp64 in, whole out)."""
    m, x = torch.frexp(top.clamp(min=2.0 ** -24))  # top = m * 2^x, 1/2 <= m < 1; 448 = 0.875 * 2^9
    return (x - 9 + (m > 0.875).to(x.dtype)).clamp(LOW, HIGH).to(torch.int32)


def two_to(e):
    """2^e in fp64, by its bits (a power on the GPU may be off in the last place)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def held(x, e):
    """What a code at exponent e stands for, for x in fp64: four significant bits, no
    finer than 2^(e - 9), to the nearest even; NaN for what is not finite."""
    y = torch.where(x.isfinite(), x, torch.zeros_like(x)).clamp(-MOST, MOST)
    _, k = torch.frexp(y)  # 2^(k - 1) <= |y| < 2^k
    step = two_to(torch.maximum(k - 4, (e - 9).expand_as(k).to(k.dtype)))
    y = torch.round(y / step) * step
    return torch.where(x.isfinite(), y, torch.full_like(y, float("nan")))


def values(codes, exp):
    """[pages, 2, H, S, D] of codes (uint8) in fp64."""
    c = codes.to(torch.int32)
    m, x, s = c & 7, (c >> 3) & 15, 1 - 2 * (c >> 7).double()
    v = torch.where(x > 0, (8 + m).double() * two_to(x - 10), m.double() * two_to(x * 0 - 9))
    v = torch.where((c & 0x7F) == 0x7F, torch.full_like(v, float("nan")), v)
    return s * v * two_to(exp.to(torch.int32))[..., None, None]


def code_of(v, exp):
    """The codes (uint8) of values that are held exactly (fp64, [pages, 2, H, S, D])."""
    y = v / two_to(exp.to(torch.int32))[..., None, None]
    a = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y))
    _, k = torch.frexp(a)
    k = torch.maximum(k, torch.full_like(k, -5))  # (below 2^-6: steps of 2^-9)
    n = a / two_to(k - 4)                         # 8 .. 15, below 8 where subnormal
    c = torch.where(n >= 8, (k + 6) * 8 + n.int() - 8, n.int())
    c = torch.where(y.isfinite(), c, torch.full_like(c, 0x7F))
    return (c + 128 * torch.signbit(y).int()).to(torch.uint8)


def finite_top(x, dims):
    return torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(dims)


class Coded(Ragged):
    """The batch of ``Ragged`` over a cache of codes; blocks of different size."""

    def __init__(self, *a, sizes=True, **k):
        super().__init__(*a, **k)
        x = self.hnd().double()
        if sizes:  # (keys less: their size goes into the exponent of the softmax)
            n = x.shape[:3]
            e = torch.randint(-10, 4, n, generator=self.g, device=DEV)
            e[:, 0] = torch.randint(-2, 1, (n[0], n[2]), generator=self.g, device=DEV)
            x = x * two_to(e)[..., None, None]
        self.code(x)

    def code(self, x):
        """The cache holds x [pages, 2, H, S, D] (fp64)."""
        e = exponent(finite_top(x, (3, 4)))
        c = code_of(held(x, e[..., None, None]), e)
        self.exp = e.to(torch.int8).contiguous()
        self.kv = (c if self.layout == HND else c.transpose(2, 3)).contiguous().view(E4M3)

    def bytes(self):
        c = self.kv.view(torch.uint8)
        return c if self.layout == HND else c.transpose(2, 3)

    def cached(self, b, which):
        pages = self.pages(b)
        x = values(self.bytes()[pages], self.exp[pages])[:, which].transpose(0, 1)
        return x.reshape(self.H, -1, self.D)[:, :self.lens[b]]

    def table(self):
        return self.kv, self.exp, self.indptr, self.indices, self.last


__all__ = ["Coded", "E4M3", "exponent", "held", "values", "code_of", "finite_top", "two_to",
           "within", "i32", "DEV", "I32", "NEG", "HND", "NHD", "math"]
