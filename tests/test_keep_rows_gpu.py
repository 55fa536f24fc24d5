"""Keeping the accepted rows of a tree: keys and values move in all layers."""
import random

import pytest
import torch

from glassbox_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def batch(dtype, layers, heads, hd, vd, page, shapes, seed):
    """shapes: (tokens before, rows, kept)."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    need = [-(-(max(p, 0) + r) // page) for p, r, _ in shapes]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((len(shapes), max(need) + 1), -1, dtype=torch.int32)
    firsts, paths = [0], []
    for i, (past, rows, kept) in enumerate(shapes):
        for j in range(need[i]):
            tables[i, j] = order.pop()
        paths += sorted(rng.sample(range(1, rows), kept - 1) + [0] if kept else []) + [-1] * (rows - kept)
        firsts.append(firsts[-1] + rows)
    k = torch.randn(layers, pages, heads, page, hd, generator=g).to(dtype)
    v = torch.randn(layers, pages, heads, page, vd, generator=g).to(dtype)
    return dict(k=k, v=v, tables=tables, firsts=firsts, starts=[s[0] for s in shapes], path=paths, accepted=[s[2] for s in shapes], page=page, most=max(s[1] for s in shapes))


def plain(b):
    k, v = b["k"].clone(), b["v"].clone()
    for i, start in enumerate(b["starts"]):
        if start < 0:
            continue
        for j in range(b["accepted"][i]):
            src, dst = start + b["path"][b["firsts"][i] + j], start + j
            at = lambda p: (int(b["tables"][i, p // b["page"]]), p % b["page"])
            for old, new in ((b["k"], k), (b["v"], v)):
                new[:, at(dst)[0], :, at(dst)[1]] = old[:, at(src)[0], :, at(src)[1]]
    return k, v


def run(b):
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    k, v, status = b["k"].to(DEV), b["v"].to(DEV), as_int([0])
    kernels.keep_rows(k, v, b["tables"].to(DEV), as_int(b["firsts"]), as_int(b["starts"]), as_int(b["path"]), as_int(b["accepted"]), b["page"], b["most"], status)
    return k.cpu(), v.cpu(), int(status.item())


SHAPES = [(1003, 8, 4), (0, 1, 1), (15, 40, 12), (16, 2, 2), (7, 5, 5), (30, 33, 1), (-1, 4, 3), (3, 6, 0)]


@pytest.mark.parametrize("dtype,layers,heads,hd,vd,page", [(torch.bfloat16, 3, 3, 64, 64, 16), (torch.float32, 2, 5, 64, 64, 16), (torch.bfloat16, 1, 1, 128, 96, 32),
                                                           (torch.bfloat16, 2, 2, 6, 10, 16), (torch.float32, 2, 1, 3, 5, 7), (torch.bfloat16, 1, 2, 3, 3, 16),
                                                           (torch.float32, 2, 9, 256, 256, 8)])
def test_moves(dtype, layers, heads, hd, vd, page):
    b = batch(dtype, layers, heads, hd, vd, page, SHAPES, hd)
    k, v, status = run(b)
    want_k, want_v = plain(b)
    assert status == 0 and torch.equal(k, want_k) and torch.equal(v, want_v)


def test_long_paths():
    """A path that reads what it has written over: every second row."""
    b = batch(torch.bfloat16, 2, 2, 64, 64, 16, [(11, 300, 150), (5, 1024, 512)], 1)
    b["path"] = list(range(0, 300, 2)) + [-1] * 150 + list(range(0, 1024, 2)) + [-1] * 512
    k, v, status = run(b)
    want_k, want_v = plain(b)
    assert status == 0 and torch.equal(k, want_k) and torch.equal(v, want_v)


def test_bad_paths_and_pages_are_reported():
    good = [(20, 6, 3)]
    for spoil in ("beyond", "back", "page", "many"):
        b = batch(torch.bfloat16, 2, 2, 64, 64, 16, [(20, 6, 3), (40, 4, 2)], 2)
        a = b["firsts"][0]
        if spoil == "beyond":
            b["path"][a + 2] = 6
        elif spoil == "back":
            b["path"][a + 2] = 1
        elif spoil == "many":
            b["accepted"][0] = 7
        else:
            b["tables"][0, 1] = 10 ** 6
        kept = dict(b, accepted=[0, 2])
        k, v, status = run(b)
        want_k, want_v = plain(kept)
        assert status != 0, spoil
        assert torch.equal(k, want_k) and torch.equal(v, want_v), spoil
