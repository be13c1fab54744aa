"""The definitions of the 4-bit and 8-bit blocks in 64 bits, for the tests of their kernels."""
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BLOCK = 32


def power(b):
    """2^(b - 127) for a byte, NaN for 255."""
    b = b.to(torch.float64)
    return torch.where(b == 255, torch.full_like(b, float("nan")), torch.exp2(b - 127))


def values4(codes, scales):
    """[n, k/2] codes and [n, k/32] bytes to float64 [n, k]."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    w = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(1)
    return w * power(scales).repeat_interleave(BLOCK, 1)


def values8(codes, scales):
    return codes.to(torch.float32).double() * power(scales).repeat_interleave(BLOCK, 1)


def bytes_of(x, top):
    """The smallest power of two s with max|block| <= top * s, as its byte, by trying every byte."""
    m = x.double().unflatten(1, (-1, BLOCK)).abs()
    odd = ~torch.isfinite(m).all(-1)
    limits = top * torch.exp2(torch.arange(255, dtype=torch.float64, device=x.device) - 127)
    b = torch.searchsorted(limits, m.nan_to_num(0, 0, 0).amax(-1).contiguous())        # the first limit that is not below
    return torch.where(odd, torch.full_like(b, 255), b).to(torch.uint8)


def nearest(v, grid):
    """The grid's value nearest to v (float64), ties to the even place in it; grid ascending from 0."""
    a = v.abs().contiguous()
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)         # they differ on a tie
    at = torch.where(lo % 2 == 0, lo, hi)
    return torch.copysign(grid[at], v)


def grid8(device):
    """e4m3's magnitudes: subnormal steps of 2^-9, then eight to a power of two up to 448."""
    g = [i * 2.0 ** -9 for i in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)]
    return torch.tensor(g[:-1], dtype=torch.float64, device=device)


def pack8(y):
    """float64 rows to (values over their scale, bytes); a block with a NaN or an infinity is NaN."""
    b = bytes_of(y, 448.0)
    v = nearest(y / power(b).repeat_interleave(BLOCK, 1), grid8(y.device)) if bool((b < 255).all()) else None
    if v is None:
        ok = (b < 255).repeat_interleave(BLOCK, 1)
        v = nearest(torch.where(ok, y, 0.0) / power(b.clamp(max=254)).repeat_interleave(BLOCK, 1), grid8(y.device))
        v = torch.where(ok, v, float("nan"))
    return v, b
