"""The 4-bit cache restated in 64 bits from its definition, with its bytes, for the tests (CPU tensors, loops and all)."""
import math

import torch

F64 = torch.float64


def round5(x: float) -> float:
    """x rounded to five significant bits, ties to even."""
    if x == 0:
        return 0.0
    m, e = math.frexp(x)
    return math.ldexp(float(round(m * 32)), e - 5)          # (Python rounds ties to even)


def scale_of(group) -> float:
    """The scale of a group of 32 numbers (a float64 vector)."""
    values = group.tolist()
    if not all(math.isfinite(v) for v in values):
        return math.nan
    size = max(abs(v) for v in values)
    if size < 2.0 ** -117:
        return 0.0
    return round5((-size if size in values else size) / 8)


def hold(x):
    """(codes, scales) of x float64 [..., hd]: whole numbers [..., hd] and float64 [..., hd / 32]."""
    g = x.unflatten(-1, (-1, 32))
    scales = torch.tensor([scale_of(v) for v in g.reshape(-1, 32)], dtype=F64).view(g.shape[:-1])
    d = scales.unsqueeze(-1)
    codes = torch.where((d == 0) | d.isnan(), torch.zeros_like(g), (g / d).round().clamp(-8, 7))
    return codes.flatten(-2), scales


def numbers(codes, scales):
    return (codes.unflatten(-1, (-1, 32)) * scales.unsqueeze(-1)).flatten(-2)


def nibble(c: int, hd: int, per: int) -> int:
    return (c % 32 // per * (hd // 32) + c // 32) * per + c % per


def write_token(page, off: int, codes, scales, per: int) -> None:
    """Token ``off`` of a head's page (a uint8 vector); per: 8 for keys, 4 for values."""
    hd = codes.numel()
    tile, r = off // 16 * 9 * hd, off % 16
    row = page[tile + r * hd // 2: tile + (r + 1) * hd // 2]
    for c in range(hd):
        i, code = nibble(c, hd, per), int(codes[c]) + 8
        row[i // 2] = (int(row[i // 2]) & (0xf0 if i % 2 == 0 else 0x0f)) | code << (4 * (i % 2))
    at = tile + 8 * hd + r * (hd // 32) * 2
    page[at: at + hd // 32 * 2] = scales.to(torch.bfloat16).view(torch.uint8)


def read_token(page, off: int, hd: int, per: int):
    """(codes, scales) of token ``off``."""
    tile, r = off // 16 * 9 * hd, off % 16
    row = page[tile + r * hd // 2: tile + (r + 1) * hd // 2]
    codes = torch.tensor([(int(row[nibble(c, hd, per) // 2]) >> (4 * (nibble(c, hd, per) % 2)) & 15) - 8 for c in range(hd)], dtype=F64)
    at = tile + 8 * hd + r * (hd // 32) * 2
    return codes, page[at: at + hd // 32 * 2].clone().view(torch.bfloat16).to(F64)


def random_pool(pages: int, nkv: int, page_size: int, hd: int, seed: int):
    """(kcache, vcache) of random codes and ordinary scales, as uint8, and what they stand for, float64 [pages, nkv, page_size, hd]."""
    g = torch.Generator().manual_seed(seed)
    pools, dense = [], []
    G = hd // 32
    for per in (8, 4):
        codes = torch.randint(-8, 8, (pages, nkv, page_size, hd), generator=g)
        scales = (torch.randn(pages, nkv, page_size, G, generator=g).abs() * 0.2 + 0.05) * torch.where(torch.rand(pages, nkv, page_size, G, generator=g) < 0.5, -1.0, 1.0)
        scales = ((scales.float().view(torch.int32) + 0x40000) & ~0x7ffff).view(torch.float32)         # five significant bits
        place = torch.tensor([nibble(c, hd, per) for c in range(hd)])
        placed = torch.empty(pages, nkv, page_size, hd, dtype=torch.uint8)
        placed[..., place] = (codes + 8).to(torch.uint8)
        packed = (placed[..., 0::2] | placed[..., 1::2] << 4).view(pages, nkv, page_size // 16, 16 * hd // 2)
        raw = scales.to(torch.bfloat16).contiguous().view(torch.uint8).view(pages, nkv, page_size // 16, 16 * G * 2)
        pools.append(torch.cat([packed, raw], dim=-1).view(pages, nkv, -1).contiguous())
        dense.append(numbers(codes.to(F64), scales.to(F64)))
    return pools, dense
