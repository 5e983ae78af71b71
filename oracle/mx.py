"""Block-scaled numbers in plain torch: 8-bit (e4m3) and 4-bit (e2m1) elements, one power of two for
each 32 of a row, in 64 bits and on whatever device the input is.  Test infrastructure, as the
rest of this package; the reference has no such format."""
from __future__ import annotations

import torch

TOP = {8: 464.0, 4: 7.0}          # half a step above the largest value
LARGEST = {8: 448.0, 4: 6.0}
MANTISSA = {8: 3, 4: 1}
LOWEST = {8: -6, 4: 0}            # the smallest normal number's exponent


def power(k):
    """2^k in fp64, by its bits."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def exponent(v):
    """floor(log2 |v|) of fp64 v, by its bits; -1023 for zero."""
    return ((v.view(torch.int64) >> 52) & 0x7ff) - 1023


def nearest(v, bits):
    """v to the nearest number of the format, ties to even, the ends saturating."""
    e = exponent(v).clamp(min=LOWEST[bits])
    step = power(e - MANTISSA[bits])
    return (torch.round(v / step) * step).clamp(-LARGEST[bits], LARGEST[bits])


def quantize(x, bits):
    """(values over their scales (R, 128 ceil(K / 128)), scale bytes (R, 4 ceil(K / 128))) of x (R, K); a block with a
    number that is not finite: NaN, 255."""
    R, K = x.shape
    v = torch.zeros(R, -(-K // 128) * 128, dtype=torch.float64, device=x.device)
    v[:, :K] = x.double()
    v = v.view(R, -1, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], 0.0, v)
    amax = v.abs().amax(-1)
    k = (exponent(amax) - exponent(torch.tensor(TOP[bits], dtype=torch.float64)).item()).clamp(min=-126)
    k = torch.where(amax > TOP[bits] * power(k), k + 1, k)
    if bits == 4:
        k = k.clamp(max=125)                                      # every number is finite in bf16
    q = nearest(v / power(k)[..., None], bits)
    q = torch.where(bad[..., None], float('nan'), q)
    return q.flatten(1), torch.where(bad, 255, k + 127).to(torch.uint8)


def scales(b):
    """The numbers that scale bytes stand for."""
    return torch.where(b == 255, float('nan'), power(b.long() - 127))


def rounded(x, bits):
    """x (R, K) as its blocks stand for it, fp64."""
    q, b = quantize(x, bits)
    return (q.view(q.shape[0], -1, 32) * scales(b)[..., None]).flatten(1)[:, :x.shape[1]]


def rms_norm(h, gamma, eps):
    d = h.double()
    return d / torch.sqrt((d * d).sum(-1, keepdim=True) / h.shape[-1] + eps) * gamma.double()
