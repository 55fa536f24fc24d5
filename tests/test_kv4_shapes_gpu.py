"""Attention over a cache in 4 bits at shapes that take the kernels' other paths: many tiles and heads of a prompt, many rows and ragged lengths of a
decode step, other head sizes, calls at once and recorded ones. The reference is the definition in 64 bits (on the GPU, for speed)."""
import math

import pytest
import torch

import kv4_plain as plain
from test_kv4_gpu import BF16, DEV, F32, F64, allowed, status, tables_for

pytestmark = pytest.mark.gpu


def reference(q, dense, tables, row_seq, positions, nh, nkv, scale, window):
    """(out, sum of p |v|, largest sum of |q k| scale) in float64, on the GPU; dense [pages, nkv, page, hd] float64."""
    n, hd = q.shape[0], dense[0].shape[-1]
    out, size, most = torch.zeros(n, nh, hd, dtype=F64, device=DEV), torch.zeros(n, nh, hd, dtype=F64, device=DEV), 0.0
    x = q.to(DEV, F64).view(n, nkv, nh // nkv, hd)
    for s in row_seq.unique().tolist():
        rows = [r for r in range(n) if int(row_seq[r]) == s and int(positions[r]) >= 0]
        if not rows:
            continue
        at = positions[rows].to(DEV)
        keys = int(at.max()) + 1
        pages = tables[s][:-(-keys // dense[0].shape[2])].long().to(DEV)
        k, v = (d[pages].transpose(0, 1).flatten(1, 2)[:, :keys] for d in dense)
        y = torch.arange(keys, device=DEV)[None, :]
        hidden = (y > at[:, None]) | ((y <= at[:, None] - window) if window else torch.zeros_like(y > at[:, None]))
        scores = torch.einsum("rghc,gkc->rghk", x[rows], k) * scale
        w = torch.softmax(scores.masked_fill(hidden[:, None, None], -math.inf), -1)
        out[rows] = torch.einsum("rghk,gkc->rghc", w, v).flatten(1, 2)
        size[rows] = torch.einsum("rghk,gkc->rghc", w, v.abs()).flatten(1, 2)
        magnitudes = torch.einsum("rghc,gkc->rghk", x[rows].abs(), k.abs()) * scale
        most = max(most, float(magnitudes.masked_fill(hidden[:, None, None], 0.0).max()))
    return out.flatten(1), size.flatten(1), most


def pool_of(pages, nkv, page_size, hd, seed):
    """A pool that the kernel under test has not written: bytes of random codes, scales around 2^-3."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pools, dense = [], []
    for per in (8, 4):
        tiles = pages * nkv * page_size // 16
        codes = torch.randint(0, 256, (tiles, 8 * hd), generator=g, device=DEV, dtype=torch.uint8)
        scales = (2.0 ** -3 * torch.randint(16, 32, (tiles, 16, hd // 32), generator=g, device=DEV) / 16).to(BF16)
        scales = scales * (torch.randint(0, 2, scales.shape, generator=g, device=DEV) * 2 - 1).to(BF16)
        pools.append(torch.cat([codes, scales.view(torch.uint8).flatten(1)], 1).view(pages, nkv, -1))
        place = torch.tensor([plain.nibble(c, hd, per) for c in range(hd)], device=DEV)
        low, high = codes.view(tiles, 16, hd // 2).int() & 15, codes.view(tiles, 16, hd // 2).int() >> 4
        nibbles = torch.stack([low, high], -1).flatten(2)[..., place] - 8
        dense.append((nibbles.to(F64) * scales.to(F64).repeat_interleave(32, -1)).view(pages, nkv, page_size, hd))
    return pools, dense


PROMPTS = [  # nh, nkv, hd, page size, window, (rows, tokens before) of the requests; None: a padding request
    (4, 4, 128, 16, None, [(300, 0), (129, 200), None, (1, 511)]), (6, 2, 128, 32, 150, [(257, 70), (128, 1), (130, 300)]),
    (5, 1, 128, 128, None, [(140, 33), (260, 0)]), (3, 3, 128, 16, 1, [(200, 5), (3, 0)]), (8, 1, 128, 8 * 16, 129, [(127, 129), (385, 0)]),
    (7, 1, 64, 16, None, [(300, 0), None, (129, 200)]), (2, 1, 256, 16, 100, [(140, 33)]), (3, 1, 160, 48, None, [(40, 100), (1, 0)]),
    (2, 2, 128, 48, None, [(150, 20)]), (2, 2, 128, 256, 40, [(150, 20)]),
    # few blocks behind many keys, which clusters share: all of four, one tile of a request that is short, a window, a row behind its last tile
    (8, 2, 128, 16, None, [(200, 3000)]), (4, 2, 128, 32, None, [(5, 0), None, (130, 2500), (1, 1700)]), (6, 2, 128, 16, 900, [(256, 4000), (128, 0)]),
    (3, 1, 128, 64, None, [(257, 1664), (1, 1535)]), (1, 1, 128, 16, None, [(129, 800)])]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh, nkv, hd, page_size, window, requests", PROMPTS)
def test_prompts_of_many_tiles(dtype, nh, nkv, hd, page_size, window, requests):
    from glassbox_b200 import kernels
    lengths = [sum(r) if r else 0 for r in requests]
    pages = sum(-(-x // page_size) for x in lengths) + 1
    pools, dense = pool_of(pages, nkv, page_size, hd, 5)
    tables = tables_for(lengths, pages, page_size, 3)
    first, row_seq, positions, start = [0], [], [], []
    for i, r in enumerate(requests):
        rows, past = r or (9, -1)
        first.append(first[-1] + rows)
        row_seq += [i] * rows
        positions += list(range(past, past + rows)) if r else [-1] * rows
        start.append(past)
    n, scale = first[-1], 1 / math.sqrt(hd)
    row_seq, positions, first, start = (torch.tensor(x, dtype=torch.int32) for x in (row_seq, positions, first, start))
    q = torch.randn(n, nh * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    want, size, most = reference(q, dense, tables, row_seq, positions, nh, nkv, scale, window)
    st, out = status(), torch.full((n, nh * hd), 7.0, dtype=dtype, device=DEV)
    kp, vp = (torch.zeros(pages, nkv, page_size, hd, dtype=dtype, device=DEV) for _ in range(2))
    kernels.kv4_attention_prefill(q.to(DEV), out, *pools, *[t.to(DEV) for t in (tables, row_seq, positions, first, start)],
                                  max(r[0] if r else 9 for r in requests), nh, nkv, hd, page_size, scale, window, max(lengths), kp, vp, st)
    assert int(st) == 0
    off = (out.to(F64) - want).abs() - allowed(dtype, want, size, 2 * most, hd, max(lengths))
    assert (off[positions.to(DEV) >= 0] <= 0).all(), float(off.max())
    assert (out[positions.to(DEV) < 0] == 0).all()


DECODES = [  # kind, rows, nh, nkv, hd, longest, what the call says of the longest, window
    ("even", 70, 4, 2, 64, 3000, 9000, None), ("cluster", 70, 4, 2, 64, 3000, 9000, 700), ("even", 5, 16, 2, 128, 9000, 9000, None),
    ("even", 300, 9, 1, 32, 700, 8193, None), ("cluster", 33, 6, 2, 96, 2500, 2500, None), ("even", 90, 6, 2, 96, 2500, 20000, None),
    ("cluster", 12, 2, 1, 256, 5000, 9000, 4000), ("even", 12, 2, 1, 256, 5000, 9000, None), ("cluster", 1030, 4, 2, 64, 400, 9000, None),
    ("cluster", 2, 4, 2, 128, 900, 900, None), ("cluster", 1, 3, 3, 64, 2500, 2500, 100), ("rows", 5, 6, 2, 160, 1500, 1500, None),
    ("rows", 3, 2, 1, 224, 900, 900, 333), ("even", 3, 2, 2, 64, 16, 8200, None), ("even", 2, 3, 1, 96, 12000, 12000, 9000)]


@pytest.mark.parametrize("kind, n, nh, nkv, hd, longest, reach, window", DECODES)
def test_ragged_decode_steps(kind, n, nh, nkv, hd, longest, reach, window):
    from glassbox_b200 import kernels
    assert kernels.kv4_decode_plan(n, nh, nkv, hd, reach, window)[0] == kind
    g = torch.Generator().manual_seed(n)
    lengths = [1, longest] + torch.randint(1, longest + 1, (n,), generator=g).tolist()
    lengths = lengths[:n] if n > 1 else [longest]
    pages = sum(-(-x // 16) for x in lengths) + 1
    pools, dense = pool_of(pages, nkv, 16, hd, 5)
    tables = tables_for(lengths, pages, 16, 3)
    row_seq = torch.randperm(n, generator=g).to(torch.int32)
    positions = torch.tensor(lengths, dtype=torch.int32)[row_seq.long()] - 1
    if n > 4:
        positions[3] = -1
    scale = 1 / math.sqrt(hd)
    q = torch.randn(n, nh * hd, generator=g).to(BF16)
    want, size, most = reference(q, dense, tables, row_seq, positions, nh, nkv, scale, window)
    qd, args = q.to(DEV), [t.to(DEV) for t in (tables, row_seq, positions)]
    outs = []
    for _ in range(2):
        st, out = status(), torch.full_like(qd, 7.0)
        parts = kernels.kv4_decode_parts(qd, nh, nkv, hd, reach, window)
        if parts is not None:
            parts.fill_(math.nan)
        kernels.kv4_attention_decode(qd, out, *pools, *args, nh, nkv, hd, 16, scale, window, reach, parts, st)
        assert int(st) == 0
        off = (out.to(F64) - want).abs() - allowed(BF16, want, size, most, hd, longest)
        assert (off <= 0).all(), float(off.max())
        outs.append(out)
    assert torch.equal(*outs)


def test_two_steps_at_once():
    """Two decode steps and two prompts on two streams, each with scratch of its own, come out as one after the other."""
    from glassbox_b200 import kernels
    nh, nkv, hd, n, longest, reach = 4, 2, 64, 40, 2500, 9000
    pages = 40 * 157
    pools, _ = pool_of(pages, nkv, 16, hd, 5)
    tables = tables_for([longest] * n, pages, 16, 3).to(DEV)
    row_seq = torch.arange(n, dtype=torch.int32, device=DEV)
    positions = torch.full((n,), longest - 1, dtype=torch.int32, device=DEV)
    rows = 200
    ints = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0] * rows, list(range(300, 300 + rows)), [0, rows], [300])]

    def step(seed):
        q = torch.randn(n + rows, nh * hd, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(BF16)
        parts = kernels.kv4_decode_parts(q[:n], nh, nkv, hd, reach)
        assert parts is not None
        return q, torch.empty_like(q), parts, [torch.zeros(pages, nkv, 16, hd, dtype=BF16, device=DEV) for _ in range(2)], status()

    def run(q, out, parts, unpacked, st):
        kernels.kv4_attention_decode(q[:n], out[:n], *pools, tables, row_seq, positions, nh, nkv, hd, 16, 0.1, None, reach, parts, st)
        kernels.kv4_attention_prefill(q[n:], out[n:], *pools, tables[:1], *ints, rows, nh, nkv, hd, 16, 0.1, None, longest, *unpacked, st)

    after = [step(s) for s in (1, 2)]
    for a in after:
        run(*a)
    torch.cuda.synchronize()
    at_once = [step(s) for s in (1, 2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for a in at_once:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                run(*a)
    torch.cuda.synchronize()
    for a, b in zip(after, at_once):
        assert torch.equal(a[1], b[1]) and int(a[4]) == int(b[4]) == 0


def test_a_context_longer_than_said_is_reported():
    from glassbox_b200 import kernels
    pools, _ = pool_of(8, 1, 16, 64, 5)
    ints = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([[0, 1, 2, 3]], [0] * 6, list(range(40, 46)), [0, 6], [40])]
    q = torch.randn(6, 64, device=DEV).to(BF16)
    for most, said in ((46, 0), (48, 0), (32, 4)):
        pages, st = [torch.zeros(8, 1, 16, 64, dtype=BF16, device=DEV) for _ in range(2)], status()
        kernels.kv4_attention_prefill(q, torch.empty_like(q), *pools, *ints, 6, 1, 1, 64, 16, 0.1, None, most, *pages, st)
        assert int(st) == said


@pytest.mark.parametrize("hd", [64, 128])
def test_recorded_prompts(hd):
    from glassbox_b200 import kernels
    nh, nkv, rows, pages = 4, 2, 150, 40
    pools, _ = pool_of(pages, nkv, 16, hd, 5)
    tables = tables_for([400], pages, 16, 3).to(DEV)
    ints = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0] * rows, list(range(rows)), [0, rows], [0])]
    q = torch.randn(rows, nh * hd, device=DEV).to(BF16)

    def buffers():
        return torch.empty_like(q), [torch.zeros(pages, nkv, 16, hd, dtype=BF16, device=DEV) for _ in range(2)], status()

    def run(out, unpacked, st):
        kernels.kv4_attention_prefill(q, out, *pools, tables, *ints, rows, nh, nkv, hd, 16, 0.1, None, 400, *unpacked, st)

    recorded = buffers()
    run(*recorded)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(*recorded)
    for past in (0, 77, 250):
        q.copy_(torch.randn(rows, nh * hd, device=DEV))
        ints[1].copy_(torch.arange(past, past + rows, device=DEV))
        ints[3].fill_(past)
        plainly = buffers()
        run(*plainly)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(plainly[0], recorded[0]) and int(plainly[2]) == int(recorded[2]) == 0
