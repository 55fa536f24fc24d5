"""What a cache in 4 bits stores of turned keys that lie next to a border between two codes or two scales, against exact rational arithmetic."""
from fractions import Fraction

import pytest
import torch

import kv4_plain as plain
from test_kv4_gpu import BF16, DEV, F32, status

pytestmark = pytest.mark.gpu

HALF = 16           # pairs of a head of 32 channels
# The kernel holds a turned key as two float32, each of 24 bits: products and the sum with their errors, which are added up with a few roundings of 2^-24
# of themselves, some 2^-46 of the pair's size. What is nearer to a border than that is left out of the comparison.
TOO_NEAR = Fraction(1, 2 ** 44)


def exact_pair(a, b, c, s):
    """(a c - b s, b c + a s) as fractions of float32 (or bfloat16) numbers."""
    a, b, c, s = (Fraction(float(x)) for x in (a, b, c, s))
    return a * c - b * s, b * c + a * s


def five_bits(x):
    """(x > 0 rounded to five significant bits, ties to even; its distance from a border between two, relative)."""
    e = 0
    while x >= 32:
        x, e = x / 2, e + 1
    while x < 16:
        x, e = x * 2, e - 1
    whole = x.numerator // x.denominator
    rest = x - whole
    up = rest > Fraction(1, 2) or (rest == Fraction(1, 2) and whole % 2 == 1)
    return (whole + up) * Fraction(2) ** e, abs(rest - Fraction(1, 2)) / x


def expected(y):
    """(scale, codes, whether the scale is too near to a border to say, and each code) of 32 fractions."""
    high, low = max(y), -min(y)
    size = max(high, low)
    d, near = five_bits(size / 8)
    unsure = near < TOO_NEAR or abs(high - low) < TOO_NEAR * size
    if high >= low:
        d = -d
    codes, doubt = [], []
    for v in y:
        r = v / d
        down = r.numerator // r.denominator
        rest = r - down
        up = rest > Fraction(1, 2) or (rest == Fraction(1, 2) and down % 2 == 1)
        codes.append(max(-8, min(7, down + up)))
        doubt.append(abs(rest - Fraction(1, 2)) < 16 * TOO_NEAR)
    return d, codes, unsure, doubt


def stored(x, table, dtype):
    """(codes, scales) that the cache holds of keys x [n, 32] at positions 0 .. n - 1."""
    from glassbox_b200 import kernels
    n = x.shape[0]
    pages = -(-n // 16)
    qkv = torch.cat([torch.zeros(n, 32), x.float(), torch.zeros(n, 32)], 1).to(dtype).to(DEV)
    pools = [torch.zeros(pages, 1, kernels.kv4_page_bytes(16, 32), dtype=torch.uint8, device=DEV) for _ in range(2)]
    at, st = torch.arange(n, dtype=torch.int32, device=DEV), status()
    kernels.kv4_write(qkv, torch.empty(n, 32, dtype=dtype, device=DEV), table.to(DEV), at, at, *pools, 1, 1, 32, 32, 16, True, st)
    assert int(st) == 0
    keys = pools[0].cpu()
    return [plain.read_token(keys[r // 16, 0], r % 16, 32, 8) for r in range(n)]


def solved(target, a, b, s):
    """A float32 cosine for which a c - b s comes next to the target (float64 [n])."""
    return ((target + b.double() * s.double()) / a.double()).float()


def rows(dtype, n, seed):
    """Numbers of ordinary size, none near zero (they are divided by), and sines."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.rand(n, 32, generator=g) * 0.75 + 0.5) * torch.where(torch.rand(n, 32, generator=g) < 0.5, -1.0, 1.0)
    s = torch.rand(n, HALF, generator=g) * 2 - 1
    return x.to(dtype).float(), s, g


def compare(x, table, dtype, least):
    """Every stored scale and code is the exact rotation's, and at least ``least`` of the groups and of the codes are compared."""
    seen = [0, 0]
    for r, (codes, scales) in enumerate(stored(x, table, dtype)):
        pairs = [exact_pair(x[r, i], x[r, i + HALF], table[r, i, 0], table[r, i, 1]) for i in range(HALF)]
        y = [p[0] for p in pairs] + [p[1] for p in pairs]
        d, want, unsure, doubt = expected(y)
        if unsure:
            continue
        seen[0] += 1
        assert Fraction(float(scales[0])) == d, (r, float(scales[0]), float(d))
        for c in range(32):
            if not doubt[c]:
                seen[1] += 1
                assert int(codes[c]) == want[c], (r, c, int(codes[c]), want[c], float(y[c] / d))
    assert seen[0] >= least * x.shape[0] and seen[1] >= least * 32 * seen[0], seen


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_numbers_next_to_a_border_between_two_codes(dtype):
    n = 300
    x, s, g = rows(dtype, n, 1)
    d = 0.5
    x[:, 0], x[:, HALF] = -4.0, 0.25                             # (the group's largest: its scale is a half)
    halves = torch.randint(-7, 7, (n, HALF), generator=g).double() + 0.5
    c = solved(halves * d, x[:, :HALF], x[:, HALF:], s)
    c[:, 0], s[:, 0] = 1.0, 0.0
    # (the partners b c + a s may be anything; those that would be the largest are turned less)
    big = ((x[:, HALF:] * c + x[:, :HALF] * s).abs() > 3.9)
    c, s = torch.where(big, 1.0, c), torch.where(big, 0.0, s)
    compare(x, torch.stack([c, s], -1).contiguous(), dtype, 0.9)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_numbers_next_to_a_border_between_two_scales(dtype):
    n = 600
    x, s, g = rows(dtype, n, 2)
    sign = torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0).double()
    border = (torch.randint(16, 32, (n,), generator=g).double() + 0.5) / 4 * sign      # (5 bits of an eighth of it are a half past a whole number)
    x[:, HALF] *= 0.125                                          # (its partner stays small beside it)
    c = torch.full((n, HALF), 0.7)
    c[:, 0] = solved(border, x[:, 0], x[:, HALF], s[:, 0])
    compare(x, torch.stack([c, s], -1).contiguous(), dtype, 0.9)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_larger_of_two_of_unlike_signs(dtype):
    n = 300
    x, s, g = rows(dtype, n, 3)
    x[:, HALF:HALF + 2] = (x[:, HALF:HALF + 2] * 0.125).to(dtype).float()
    top = 5 + 2 * torch.rand(n, generator=g).double()
    c = torch.full((n, HALF), 0.7)
    for i, sign in ((0, 1.0), (1, -1.0)):
        c[:, i] = solved(sign * top, x[:, i], x[:, HALF + i], s[:, i])
    compare(x, torch.stack([c, s], -1).contiguous(), dtype, 0.9)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ordinary_angles(dtype):
    n = 1500
    g = torch.Generator().manual_seed(4)
    x = torch.randn(n, 32, generator=g).to(dtype).float()
    angle = torch.rand(n, HALF, generator=g) * 6.28
    compare(x, torch.stack([angle.cos(), angle.sin()], -1).contiguous(), dtype, 0.99)
