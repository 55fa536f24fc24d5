"""Prompts over a cache in 4 bits: what the pages that are unpacked into held before, and what other requests' pages hold, reaches no row that does
not see it; queries and results as columns of wider rows, behind rows that are another kernel's."""
import math

import pytest
import torch

import kv4_plain as plain
from test_kv4_gpu import BF16, DEV, F32, F64, allowed, status, tables_for
from test_kv4_shapes_gpu import pool_of, reference

pytestmark = pytest.mark.gpu


def spoil(pool, page, off, hd):
    """All scales of a token (of the first head) become NaN."""
    at = off // 16 * 9 * hd + 8 * hd + off % 16 * (hd // 32) * 2
    pool[page, 0, at:at + hd // 32 * 2] = torch.tensor([0xc0, 0x7f] * (hd // 32), dtype=torch.uint8, device=pool.device)


def batch(requests):
    """(row_seq, positions, seq_first_row, seq_start_pos) of (rows, tokens before) each, on the device."""
    first, row_seq, positions = [0], [], []
    for i, (rows, past) in enumerate(requests):
        first.append(first[-1] + rows)
        row_seq += [i] * rows
        positions += list(range(past, past + rows))
    return [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (row_seq, positions, first, [p for _, p in requests])]


def prompt(q, pools, tables, ints, requests, nh, nkv, hd, page_size, window, pages):
    from glassbox_b200 import kernels
    st, out = status(), torch.full_like(q, 7.0)
    kernels.kv4_attention_prefill(q, out, *pools, tables, *ints, max(r for r, _ in requests), nh, nkv, hd, page_size, 1 / math.sqrt(hd), window,
                                  max(r + p for r, p in requests), *pages, st)
    assert int(st) == 0
    return out


# nh, nkv, hd, page size: a shape for each kernel over unpacked pages, the one of head size 128 with and without clusters
SHAPES = [(2, 1, 64, 16), (4, 2, 64, 128), (2, 1, 128, 16), (2, 2, 128, 64), (2, 1, 64, 256), (2, 1, 128, 256), (2, 1, 32, 16), (2, 1, 96, 16), (2, 1, 160, 16), (32, 32, 32, 16),
          (27, 27, 96, 16)]
LENGTHS = [[(40, 0), (70, 130)], [(130, 20), (5, 0)], [(16, 48), (200, 1500)], [(9, 24), (140, 2600)]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh, nkv, hd, page_size", SHAPES)
@pytest.mark.parametrize("window", [None, 37])
@pytest.mark.parametrize("requests", LENGTHS, ids=str)
def test_what_no_row_sees_does_not_matter(dtype, nh, nkv, hd, page_size, window, requests):
    """The same step three times: with pages of zeros to unpack into; with pages of NaN; and with a NaN in page 0 of the cache, which the first
    request sees (its last token's key and value), after which the second request's rows are what they were."""
    lengths = [r + p for r, p in requests]
    count = sum(-(-x // page_size) for x in lengths) + 1
    pools, _ = pool_of(count, nkv, page_size, hd, 5)
    tables = tables_for(lengths, count, page_size, 3)
    last = lengths[0] - 1                                        # the page of the first request's last token becomes page 0
    other = int(tables[0, last // page_size])
    swapped = torch.arange(count, dtype=torch.int32)
    swapped[0], swapped[other] = other, 0
    tables = torch.where(tables >= 0, swapped[tables.clamp(min=0).long()], tables).to(DEV)
    ints, n = batch(requests), sum(r for r, _ in requests)
    q = torch.randn(n, nh * hd, generator=torch.Generator().manual_seed(9)).to(dtype).to(DEV)

    def unpacked(value):
        return [torch.full((count, nkv, page_size, hd), value, dtype=dtype, device=DEV) for _ in range(2)]

    args = (tables, ints, requests, nh, nkv, hd, page_size, window)
    want = prompt(q, pools, *args, unpacked(0.0))
    assert not want.isnan().any()
    assert torch.equal(prompt(q, pools, *args, unpacked(math.nan)), want)
    bad = [p.clone() for p in pools]
    for p in bad:
        spoil(p, 0, last % page_size, hd)
    pages = unpacked(0.0)
    got = prompt(q, bad, *args, pages)
    own = requests[0][0]
    assert got[own - 1, :hd].isnan().all()                       # (the row that sees it)
    assert torch.equal(got[own:], want[own:])
    # the NaN is gone from the cache and the request with it; the pages that were unpacked into are the same (the second request alone, since
    # fewer rows may take another kernel)
    args = (tables[1:], batch(requests[1:]), requests[1:], nh, nkv, hd, page_size, window)
    assert torch.equal(prompt(q[own:], pools, *args, pages), prompt(q[own:], pools, *args, unpacked(0.0)))


STRIDED = [  # nh, nkv, hd, page size, window, (rows, tokens before)
    (32, 8, 128, 16, None, [(150, 40), (1, 300)]), (6, 2, 128, 32, 150, [(257, 70), (130, 300)]), (8, 2, 128, 16, None, [(200, 3000)]),
    (3, 1, 128, 64, 700, [(129, 1664), (1, 1535)]), (9, 3, 64, 16, None, [(300, 0), (129, 200)]), (4, 1, 32, 16, 33, [(70, 150), (5, 0)]),
    (6, 2, 96, 16, None, [(130, 20), (64, 64)]), (16, 16, 32, 16, 33, [(150, 50), (45, 0)]),
    (12, 12, 96, 16, None, [(130, 20), (125, 64)]), (24, 24, 64, 48, 90, [(129, 100), (1, 0)]), (2, 1, 256, 16, None, [(40, 33)]), (2, 1, 128, 256, None, [(150, 20)])]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh, nkv, hd, page_size, window, requests", STRIDED)
def test_columns_of_wider_rows_behind_other_rows(dtype, nh, nkv, hd, page_size, window, requests):
    """As a model calls it: queries are the first columns of rows of queries, keys and values, and the requests' rows come behind single
    tokens' rows, which are left alone."""
    from glassbox_b200 import kernels
    lead = 3
    lengths = [r + p for r, p in requests]
    count = sum(-(-x // page_size) for x in lengths) + 1
    pools, dense = pool_of(count, nkv, page_size, hd, 5)
    tables = tables_for(lengths, count, page_size, 3)
    row_seq, positions, first, start = batch(requests)
    n = int(first[-1])
    wide = torch.randn(lead + n, (nh + 2 * nkv) * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    want, size, most = reference(wide[lead:, :nh * hd], dense, tables, row_seq.cpu(), positions.cpu(), nh, nkv, 1 / math.sqrt(hd), window)
    room = torch.full((lead + n, nh * hd + 16), 7.0, dtype=dtype, device=DEV)
    q, out = wide.to(DEV)[:, :nh * hd], room[:, 8:8 + nh * hd]
    st = status()
    pages = [torch.zeros(count, nkv, page_size, hd, dtype=dtype, device=DEV) for _ in range(2)]
    leading = torch.full((lead,), -1, dtype=torch.int32, device=DEV)
    kernels.kv4_attention_prefill(q, out, *pools, tables.to(DEV), torch.cat([leading * 0, row_seq]), torch.cat([leading, positions]), first + lead, start,
                                  max(r for r, _ in requests), nh, nkv, hd, page_size, 1 / math.sqrt(hd), window, max(lengths), *pages, st)
    assert int(st) == 0
    off = (out[lead:].to(F64) - want).abs() - allowed(dtype, want, size, 2 * most, hd, max(lengths))
    assert (off <= 0).all(), float(off.max())
    assert (room[:, :8] == 7).all() and (room[:, 8 + nh * hd:] == 7).all()
    tiles = kernels.kv4_prompt_kernel(q, out, nh, nkv, hd, page_size) is not None
    assert (out[:lead] == (7 if tiles else 0)).all()             # (row by row, what is no token is padding)
