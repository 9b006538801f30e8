"""Microscaled 4-bit floating point in 64 bits, from its definition, and the error bounds that go
with it.  Test infrastructure only."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(w):
    """The numbers that a tensor's rows become, in 64 bits."""
    v = w.detach().cpu().double()
    if v.numel() > 1 << 21 and v.dim() > 1:                  # in pieces: the distances take eight times the room
        return torch.cat([quantize(part) for part in v.split(max(1, v.shape[0] * (1 << 20) // v.numel()))])
    cols = v.shape[-1]
    blocks = -(-cols // 32)
    full = torch.zeros(v.shape[:-1] + (blocks * 32,), dtype=torch.float64)
    full[..., :cols] = v
    full = full.reshape(v.shape[:-1] + (blocks, 32))
    out = torch.empty_like(full)
    largest = full.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(largest)                              # largest = m 2^e, 0.5 <= m < 1
    exponent = torch.where(largest > 0, e.double() - 3, torch.full_like(largest, -127.0)).clamp(min=-127)
    scale = torch.exp2(exponent)
    u = (full / scale).abs()
    # nearest grid point by distance; on a tie the even code, which is the even index
    d = (u.unsqueeze(-1) - GRID).abs()
    best = d.amin(-1, keepdim=True)
    tie = d == best
    index = torch.where(tie, torch.arange(8) * 2 % 16 + (torch.arange(8) % 2) * 100, 1000).argmin(-1)
    out = torch.copysign(GRID[index], full) * scale
    out = torch.where(torch.isfinite(largest), out, torch.full_like(out, math.nan))
    return out.flatten(-2)[..., :cols]


def product(x, w, bias=None):
    """(y, bound) of q(x) q(w)^T + bias in 64 bits.  Bound of an fp32 sum of products: the products
    of 4-bit numbers and powers of two are exact; the tensor core adds 64 of them at a time and may
    cut each sum, and each addition to the accumulator, at 2^-23 of the largest magnitude on the
    way, which the sum of magnitudes S bounds: (K / 32 + 2) 2^-23 S; then one rounding to the type
    of x, half a step: eps / 2 of the value (and half the smallest subnormal)."""
    xq, wq = quantize(x), quantize(w)
    y = xq @ wq.t()
    s = xq.abs() @ wq.abs().t()
    if bias is not None:
        b = bias.detach().cpu().double()
        y, s = y + b, s + b.abs()
    sums = (x.shape[-1] / 32 + 2) * 2.0 ** -23 * s
    info = torch.finfo(x.dtype)
    return y, sums + info.eps / 2 * (y.abs() + sums) + info.smallest_normal * info.eps / 2


def check(got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = ((got - want).abs() - bound)[~torch.isnan(want)]
    assert off.numel() == 0 or off.max().item() <= 0, f"{off.max().item()} over the bound"
