"""Attention of trees of drafted tokens against a plain form in float64."""
import math
import random

import numpy as np
import pytest
import torch

import tree_plain as plain
from glassbox_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Batch:
    """Requests with trees over a paged cache whose unused places hold NaN."""

    def __init__(self, dtype, nh, nkv, hd, shapes, page=16, window=None, width=3, seed=0, behind=3, see=None, spare=1):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.dtype, self.nh, self.nkv, self.hd, self.page, self.window, self.shapes = dtype, nh, nkv, hd, page, window, shapes
        self.scale = 1.0 / math.sqrt(hd)
        need = [-(-(max(p, 0) + r) // page) for p, r in shapes]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g).tolist()
        width_pages = max(need) + spare
        tables = np.full((len(shapes), width_pages), -1, dtype=np.int32)
        nan = float("nan")
        k, v = (torch.full((pages, nkv, page, hd), nan, dtype=dtype) for _ in range(2))
        firsts, starts, positions, bits, self.see, self.k, self.v = [0], [], [], [], [], [], []
        most = max(r for _, r in shapes)
        for i, (past, rows) in enumerate(shapes):
            parents = plain.random_tree(rng, rows, width) if rows else []
            s = plain.ancestors(parents) if see is None else see(rng, rows)
            self.see.append(s)
            d = plain.depths(parents)
            kk, vv = (torch.randn(max(past, 0) + rows, nkv, hd, generator=g).to(dtype) for _ in range(2))
            self.k.append(kk)
            self.v.append(vv)
            for j in range(need[i]):
                tables[i, j] = order.pop()
                n = min(page, len(kk) - j * page)
                k[tables[i, j], :, :n] = kk[j * page:j * page + n].transpose(0, 1)
                v[tables[i, j], :, :n] = vv[j * page:j * page + n].transpose(0, 1)
            if window and past > 0:                       # pages that the window has passed are given back
                for j in range(max(0, past - window + 1) // page):
                    k[tables[i, j]], v[tables[i, j]] = nan, nan
                    tables[i, j] = -1
            firsts.append(firsts[-1] + rows)
            starts.append(past)
            positions += [max(past, 0) + x for x in d]
            if rows:
                bits.append(plain.words(s, -(-most // 32)))
        n = firsts[-1] + behind
        self.n = n
        self.q = torch.randn(n, nh * hd, generator=g).to(dtype)
        self.firsts, self.starts, self.positions = firsts, starts, positions + [0] * behind
        as_int = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
        words = np.concatenate(bits + [np.zeros((behind, -(-most // 32)), np.int32)])
        self.dev = dict(k=k.to(DEV), v=v.to(DEV), tables=as_int(tables), first=as_int(firsts), start=as_int(starts), pos=as_int(self.positions), bits=as_int(words))
        self.most, self.reach = most, max(max(p, 0) + r for p, r in shapes)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def run(self, q=None, out=None, reach=None):
        d = self.dev
        q = self.q.to(DEV) if q is None else q
        out = torch.full((self.n, self.nh * self.hd), 7.0, dtype=self.dtype, device=DEV) if out is None else out
        reach = self.reach if reach is None else reach
        parts = kernels.tree_attention_parts(q, self.nh, self.nkv, self.hd, len(self.shapes), self.most, reach, self.window)
        kernels.tree_attention(q, out, d["k"], d["v"], d["tables"], d["first"], d["start"], d["pos"], d["bits"], self.most, self.nh, self.nkv, self.hd, self.page,
                               self.scale, self.window, reach, parts, self.status)
        return out

    def check(self, out, status=0):
        got = out.float().cpu().double().view(self.n, self.nh, self.hd)
        for i, (past, rows) in enumerate(self.shapes):
            a, b = self.firsts[i], self.firsts[i + 1]
            if past < 0:
                assert (got[a:b] == 0).all()
                continue
            if not rows:
                continue
            want, size, reach = plain.attention(self.q[a:b].view(rows, self.nh, self.hd), self.k[i], self.v[i], past, self.positions[a:b], self.see[i], self.scale, self.window)
            tol = plain.tolerance(want, size, reach, self.hd, past + rows, self.dtype)
            assert torch.isfinite(got[a:b]).all(), f"request {i}: not finite"
            off = (got[a:b] - want).abs() - tol
            assert off.max() <= 0, f"request {i}: {off.max():.3e} over the tolerance"
        assert (got[self.firsts[-1]:] == 7.0).all(), "rows behind the last request changed"
        assert int(self.status.item()) == status


BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,nh,nkv,hd", [(BF, 9, 3, 64), (BF, 4, 4, 64), (BF, 8, 1, 128), (BF, 32, 2, 64), (BF, 6, 2, 32), (BF, 6, 3, 96), (BF, 4, 2, 80), (BF, 4, 1, 256),
                                             (BF, 2, 1, 6), (F32, 9, 3, 64), (F32, 4, 2, 48), (F32, 4, 1, 128), (F32, 2, 2, 256), (F32, 3, 1, 10)])
def test_heads(dtype, nh, nkv, hd):
    b = Batch(dtype, nh, nkv, hd, [(100, 7), (0, 1), (37, 20), (255, 5), (64, 1), (5, 0)], seed=hd + nh)
    b.check(b.run())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shapes", [[(0, 1)], [(1, 1)], [(15, 1), (16, 1), (63, 1), (64, 1)], [(0, 64)], [(31, 33), (32, 32), (33, 31)], [(700, 70), (3, 2)],
                                    [(1500, 9)], [(0, 200), (130, 257)], [(-1, 3), (20, 4), (-1, 1)]])
def test_lengths(dtype, shapes):
    b = Batch(dtype, 6, 2, 64, shapes, seed=len(shapes))
    b.check(b.run())


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
@pytest.mark.parametrize("rows", [5, 17, 40, 100])
def test_long_contexts_are_shared(dtype, hd, rows):
    b = Batch(dtype, 4, 2, hd, [(2100, rows), (900, max(1, rows // 2))], seed=rows)
    b.check(b.run())


@pytest.mark.parametrize("dtype,page", [(BF, 16), (BF, 8), (BF, 64), (BF, 256), (BF, 12), (F32, 16), (F32, 5)])
def test_pages(dtype, page):
    b = Batch(dtype, 4, 2, 64, [(130, 11), (64, 64), (9, 3)], page=page, seed=page)
    b.check(b.run())


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 5000])
def test_windows(dtype, hd, window):
    b = Batch(dtype, 4, 2, hd, [(300, 21), (0, 9), (63, 30), (170, 1)], window=window, seed=window)
    b.check(b.run())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_see_any_of_the_tree(dtype):
    """Bits in no tree's shape, rows without any: behind nothing they come out as zeros."""
    def see(rng, rows):
        s = np.array([[rng.random() < 0.4 for _ in range(rows)] for _ in range(rows)]).reshape(rows, rows)
        s[rows // 2:rows // 2 + 2] = False
        return s
    b = Batch(dtype, 4, 2, 64, [(0, 40), (77, 40), (0, 3)], seed=3, see=see)
    out = b.run()
    b.check(out)
    assert (out[20:22] == 0).all()


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 3e38])
def test_masked_places_hold_anything(dtype, hd, value):
    """What a row does not see, another branch's keys and values, does not reach it."""
    parents = [-1, 0, 0, 1, 2, 4]
    b = Batch(dtype, 4, 2, hd, [(50, 6)], seed=9, see=lambda rng, rows: plain.ancestors(parents))
    clean = b.run()
    place = 50 + 2                                         # row 2: seen by rows 2, 4 and 5
    page = int(b.dev["tables"][0, place // 16])
    b.dev["k"][page, :, place % 16] = value
    b.dev["v"][page, :, place % 16] = value
    dirty = b.run()
    for r in (0, 1, 3):
        assert torch.isfinite(dirty[r]).all()
        off = (dirty[r].float() - clean[r].float()).abs().max()
        assert off <= 2.0 ** -7 * clean[r].float().abs().max()      # (values go one by one there: another order, weights not rounded)
    if math.isnan(value):
        assert torch.isnan(dirty[2]).all()


@pytest.mark.parametrize("hd,nh,nkv", [(64, 4, 2), (128, 4, 2), (128, 4, 1)])
@pytest.mark.parametrize("shapes", [[(600, 40)], [(513, 64), (40, 33)], [(127, 64), (128, 1), (129, 50), (0, 64), (1030, 40)], [(-1, 40), (700, 50), (-1, 2)],
                                    [(640, 128), (640, 100)], [(100, 300)], [(2000, 65), (0, 0), (90, 64)]])
@pytest.mark.parametrize("reach", [None, 2048])
def test_many_rows(hd, nh, nkv, shapes, reach):
    """Enough query rows a key/value head for tcgen05 (contexts are said to be long): one unit's rows, two, several pairs."""
    b = Batch(BF, nh, nkv, hd, shapes, seed=hd + nkv)
    b.check(b.run(reach=reach))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nkv", [1, 2])
@pytest.mark.parametrize("page", [8, 16, 32, 128, 256])
def test_many_rows_and_pages(hd, nkv, page):
    b = Batch(BF, 4, nkv, hd, [(700, 45), (1300, 33), (5, 40)], page=page, seed=page)
    b.check(b.run())


@pytest.mark.parametrize("hd", [64, 128])
def test_many_rows_of_many_requests(hd):
    """More pieces a block than its list holds."""
    rng = random.Random(hd)
    b = Batch(BF, 4, 1, hd, [(rng.choice([0, 5, 130, 600]), rng.choice([1, 20, 33])) for _ in range(700)], seed=5)
    b.check(b.run(reach=1024))


@pytest.mark.parametrize("hd,nkv", [(64, 2), (128, 2), (128, 1)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("past", [590, 639, 5000])
def test_masked_places_of_many_rows_hold_anything(hd, nkv, value, past):
    rng = random.Random(4)
    parents = plain.random_tree(rng, 64, 4)
    see = plain.ancestors(parents)
    b = Batch(BF, 4, nkv, hd, [(past, 64)], seed=9, see=lambda rng, rows: see)
    clean = b.run()
    where = past + 20
    page = int(b.dev["tables"][0, where // 16])
    b.dev["v"][page, :, where % 16, 3:5] = value
    dirty = b.run()
    hit = torch.from_numpy(see[:, 20])
    assert 0 < hit.sum() < 63
    off = (dirty[:64][~hit].float() - clean[:64][~hit].float()).abs().max()
    assert torch.isfinite(dirty[:64][~hit]).all() and off == 0
    got = dirty[:64][hit].view(-1, 4, hd)
    assert (torch.isnan(got[..., 3:5]) if math.isnan(value) else torch.isinf(got[..., 3:5])).all()
    assert torch.isfinite(got[..., :3]).all() and torch.isfinite(got[..., 5:]).all()
    want = clean[:64][hit].view(-1, 4, hd)
    rest = [c for c in range(hd) if c not in (3, 4)]
    assert (got[..., rest].float() - want[..., rest].float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()      # (its weight is not rounded there)
    b.dev["k"][page, :, where % 16] = value               # a key, too
    dirty = b.run()
    assert torch.isfinite(dirty[:64][~hit]).all() and (dirty[:64][~hit].float() - clean[:64][~hit].float()).abs().max() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_other_pools(dtype):
    b = Batch(dtype, 6, 2, 64, [(90, 12), (200, 3)], seed=4)
    wide = torch.zeros(b.n, 900, dtype=dtype, device=DEV)
    wide[:, 100:100 + 384] = b.q.to(DEV)
    out = torch.full((b.n, 700), 7.0, dtype=dtype, device=DEV)
    b.run(q=wide[:, 100:484], out=out[:, 50:434])
    b.check(out[:, 50:434].contiguous())
    assert (out[:, :50] == 7).all() and (out[:, 434:] == 7).all()
    # rows that start at odd places
    odd = torch.zeros(b.n, 401, dtype=dtype, device=DEV)
    odd[:, 3:387] = b.q.to(DEV)
    b.check(b.run(q=odd[:, 3:387]))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_missing_pages_are_reported(dtype):
    b = Batch(dtype, 4, 2, 64, [(100, 5), (60, 5)], seed=5)
    b.dev["tables"][0, 1] = b.dev["k"].shape[0] + 5
    b.dev["tables"][0, 3] = -1
    out = b.run()
    assert int(b.status.item()) == 2
    b.status.zero_()
    b.shapes = [(-1, 5), (60, 5)]
    out[:5] = 0
    b.check(out)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_longer_than_said(dtype):
    b = Batch(dtype, 4, 2, 64, [(1200, 5)], seed=6)
    b.check(b.run(reach=10))
    b.check(b.run(reach=100000))


def test_recorded_and_on_another_stream():
    b = Batch(BF, 4, 2, 64, [(1200, 5), (40, 9)], seed=7)
    q, out = b.q.to(DEV), torch.full((b.n, 256), 7.0, dtype=BF, device=DEV)
    want = b.run(q=q).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(b.run(q=q), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(q=q, out=out)
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_the_last_page_of_a_large_pool():
    """Offsets beyond 2^31 numbers."""
    nkv, hd, page = 8, 128, 16
    pages = (1 << 31) // (nkv * hd * page) + 40
    k = torch.zeros(pages, nkv, page, hd, dtype=BF, device=DEV)
    v = torch.zeros(pages, nkv, page, hd, dtype=BF, device=DEV)
    b = Batch(BF, 16, nkv, hd, [(40, 5)], seed=8)
    for i, p in enumerate(b.dev["tables"][0].tolist()):
        if p >= 0:
            k[pages - 1 - i], v[pages - 1 - i] = b.dev["k"][p], b.dev["v"][p]
            b.dev["tables"][0, i] = pages - 1 - i
    b.dev["k"], b.dev["v"] = k, v
    b.check(b.run())


FAR = 1 << 17      # contexts said to be this long


@pytest.mark.parametrize("hd,nh,nkv", [(64, 4, 2), (128, 4, 2), (128, 4, 1), (64, 6, 6)])
@pytest.mark.parametrize("shapes", [[(600, 40)], [(513, 64), (40, 33)], [(127, 64), (128, 1), (129, 50), (0, 64), (1030, 40)], [(-1, 40), (700, 50), (-1, 2)],
                                    [(640, 128), (640, 100)], [(100, 300)], [(2000, 65), (0, 0), (90, 64)], [(0, 33)], [(5300, 70), (1, 36)]])
def test_many_rows_said_to_be_far(hd, nh, nkv, shapes):
    b = Batch(BF, nh, nkv, hd, shapes, seed=hd + nkv + 1)
    b.check(b.run(reach=FAR))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nkv", [1, 2])
@pytest.mark.parametrize("page", [8, 16, 32, 128, 256])
def test_many_rows_said_to_be_far_and_pages(hd, nkv, page):
    b = Batch(BF, 4, nkv, hd, [(700, 45), (1300, 33), (5, 40)], page=page, seed=page + 1)
    b.check(b.run(reach=FAR))


@pytest.mark.parametrize("hd,nkv", [(64, 2), (128, 2), (128, 1)])
@pytest.mark.parametrize("past", [0, 40, 590, 639])
def test_masked_places_said_to_be_far_hold_anything(hd, nkv, past):
    rng = random.Random(4)
    see = plain.ancestors(plain.random_tree(rng, 64, 4))
    b = Batch(BF, 4, nkv, hd, [(past, 64)], seed=10, see=lambda rng, rows: see)
    clean = b.run(reach=FAR)
    where = past + 20
    page = int(b.dev["tables"][0, where // 16])
    b.dev["k"][page, :, where % 16] = float("nan")
    b.dev["v"][page, :, where % 16, 3:5] = float("inf")
    dirty = b.run(reach=FAR)
    hit = torch.from_numpy(see[:, 20])
    assert 0 < hit.sum() < 63
    assert torch.equal(dirty[:64][~hit], clean[:64][~hit])
    assert torch.isnan(dirty[:64][hit]).all()


@pytest.mark.parametrize("reach", [None, FAR])
def test_missing_pages_of_many_rows_are_reported(reach):
    b = Batch(BF, 4, 2, 64, [(300, 64), (700, 40)], seed=5)
    b.dev["tables"][0, 3] = b.dev["k"].shape[0] + 5
    out = b.run(reach=reach)
    assert int(b.status.item()) == 2
    b.status.zero_()
    b.shapes = [(-1, 64), (700, 40)]
    out[:64] = 0
    b.check(out)


@pytest.mark.parametrize("nh,nkv,hd,shapes", [(4, 4, 64, [(2000, 20)] * 40), (3, 1, 64, [(30000, 1)]), (8, 8, 128, [(9000, 1), (7000, 1)]), (6, 6, 32, [(1500, 12)] * 60),
                                              (6, 6, 96, [(700, 33)] * 30)])
def test_keys_cut_evenly(nh, nkv, hd, shapes):
    b = Batch(BF, nh, nkv, hd, shapes, seed=nh)
    b.check(b.run())


def test_two_recorded_calls_that_share_scratch():
    a, b = Batch(BF, 4, 4, 64, [(3000, 20)] * 20, seed=1), Batch(BF, 8, 2, 128, [(2500, 40), (900, 64)], seed=2)
    first, second = torch.full((a.n, 256), 7.0, dtype=BF, device=DEV), torch.full((b.n, 1024), 7.0, dtype=BF, device=DEV)
    qs = a.q.to(DEV), b.q.to(DEV)
    sizes = [kernels.tree_attention_floats(x.n, x.nh, x.nkv, x.hd, len(x.shapes), x.most, FAR) for x in (a, b)]
    parts = torch.full((max(max(sizes), 1),), float("nan"), device=DEV)

    def call(x, q, out):
        d = x.dev
        kernels.tree_attention(q, out, d["k"], d["v"], d["tables"], d["first"], d["start"], d["pos"], d["bits"], x.most, x.nh, x.nkv, x.hd, x.page, x.scale,
                               None, FAR, parts, x.status)
    call(a, qs[0], first)
    call(b, qs[1], second)
    torch.cuda.synchronize()
    graphs = []
    for x, q, out in ((a, qs[0], first), (b, qs[1], second)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(x, q, out)
    for _ in range(3):
        first.fill_(7.0)
        second.fill_(7.0)
        parts.fill_(float("nan"))
        for g in (graphs[0], graphs[1], graphs[0]):
            g.replay()
        a.check(first)
        b.check(second)


@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (4, 2, 128), (6, 6, 64), (2, 2, 128)])
@pytest.mark.parametrize("shapes", [[(9000, 1)], [(8300, 7), (40, 3)], [(0, 1), (128, 8), (127, 5)], [(-1, 3), (511, 2), (0, 0), (6, 6)]])
def test_few_rows_said_to_be_far(nh, nkv, hd, shapes):
    b = Batch(BF, nh, nkv, hd, shapes, seed=hd + nkv + 2)
    b.check(b.run(reach=FAR))
