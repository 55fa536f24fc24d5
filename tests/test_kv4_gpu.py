"""The 4-bit cache's kernels against their definition in 64 bits: what is stored, byte by byte, and attention over it."""
import math

import pytest
import torch

import kv4_plain as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F64 = torch.float64
BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}       # half a step of a rounding, relative


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def turned(x, angle, rot):
    """x float64 [n, heads, hd], angle float64 [n, rot / 2, 2]."""
    if not rot:
        return x
    a, b, c, s = x[..., :rot // 2], x[..., rot // 2:rot], angle[:, None, :, 0], angle[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], dim=-1)


def check_held(got_codes, got_scales, x, slack):
    """The codes and scales read from a cache hold x (float64 [..., hd]), where a number next to a border between two codes or two
    scales may have fallen to either side: ``slack``, the relative error of the number that was rounded."""
    for c, d, v in zip(got_codes.reshape(-1, 32), got_scales.reshape(-1), x.reshape(-1, 32)):
        d, allowed = float(d), set()
        want = plain.scale_of(v)
        if math.isnan(want):
            assert math.isnan(d)
            continue
        size = float(v.abs().max())
        for f in (1 - slack, 1, 1 + slack):
            for sign in ((-1, 1) if bool((v >= size * (1 - slack)).any()) and bool((v <= -size * (1 - slack)).any()) else (1,)):
                allowed.add(sign * plain.round5(want if f == 1 else math.copysign(size * f / 8, want)))
        assert d in allowed, (d, want, size)
        if d == 0.0:
            assert (c == 0).all()
            continue
        ratio = (v / d).clamp(-8, 7)
        assert ((c - ratio).abs() <= 0.5 + 16 * slack).all() and (c == c.round()).all() and (c >= -8).all() and (c <= 7).all()


def write(qkv, positions, slots, table, kc, vc, nh, nkv, hd, rot, page_size, q=None, write_kv=True, st=None):
    from glassbox_b200 import kernels
    if q is None:
        q = torch.full((qkv.shape[0], nh * hd), 7.0, dtype=qkv.dtype, device=DEV)
    st = status() if st is None else st
    kernels.kv4_write(qkv, q, table, positions, slots, kc, vc, nh, nkv, hd, rot, page_size, write_kv, st)
    return q, int(st)


WRITES = [  # n, nh, nkv, hd, rot, page size
    (1, 1, 1, 32, 32, 16), (5, 9, 3, 64, 64, 16), (37, 4, 2, 96, 96, 48), (18, 6, 2, 96, 32, 16), (9, 2, 1, 128, 0, 32), (7, 3, 3, 64, 6, 16),
    (3, 2, 2, 256, 256, 16), (6, 5, 1, 32, 16, 16), (12, 3, 1, 64, 40, 16), (300, 2, 1, 64, 32, 16)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n, nh, nkv, hd, rot, page_size", WRITES)
def test_write_rotates_and_holds(dtype, n, nh, nkv, hd, rot, page_size):
    g = torch.Generator().manual_seed(n * 7 + hd)
    pages = -(-n // page_size) + 2
    qkv = (torch.randn(n, (nh + 2 * nkv) * hd, generator=g) * torch.exp(torch.randn((nh + 2 * nkv) * hd, generator=g))).to(dtype)
    angle = torch.rand(n + 20, max(rot // 2, 1), generator=g) * 6.28
    table = torch.stack([angle.cos(), angle.sin()], dim=-1) if rot else None
    positions = torch.randperm(n + 20, generator=g)[:n].to(torch.int32)
    slots = torch.randperm(pages * page_size, generator=g)[:n].to(torch.int32)
    from glassbox_b200 import kernels
    size = kernels.kv4_page_bytes(page_size, hd)
    before = [torch.randint(0, 256, (pages, nkv, size), generator=g, dtype=torch.uint8) for _ in range(2)]
    pools = [b.to(DEV) for b in before]
    dev = [t.to(DEV) for t in (qkv, positions, slots)]
    q, st = write(dev[0], dev[1], dev[2], table.to(DEV) if rot else None, *pools, nh, nkv, hd, rot, page_size)
    assert st == 0 and torch.equal(dev[0].cpu(), qkv)                 # the rows themselves stay as they were
    x = qkv.to(F64).view(n, -1, hd)
    at = table[positions.long()].to(F64) if rot else None
    want = turned(x[:, :nh + nkv], at, rot)
    # two products and a sum in float32 of the pair's numbers, then the rounding to the row's type
    size_of = x[:, :nh + nkv].abs()
    if rot:
        pair = size_of[..., :rot // 2] + size_of[..., rot // 2:rot]
        size_of = torch.cat([pair, pair, size_of[..., rot:]], dim=-1)
    bound = want[:, :nh].abs() * HALF_STEP[dtype] * (1 + 2.0 ** -20) + size_of[:, :nh] * 2 * 2.0 ** -24
    assert ((q.cpu().to(F64).view(n, nh, hd) - want[:, :nh]).abs() <= bound).all()
    after = [p.cpu() for p in pools]
    marked = [b.clone() for b in before]
    for r in range(n):
        page, off = int(slots[r]) // page_size, int(slots[r]) % page_size
        for h in range(nkv):
            key = plain.read_token(after[0][page, h], off, hd, 8)
            value = plain.read_token(after[1][page, h], off, hd, 4)
            # (a rotation may cancel: what is rounded is off by the pair's size, not its own)
            small = want[r, nh + h].abs().view(-1, 32).amax(-1)
            slack = float((size_of[r, nh + h].view(-1, 32).amax(-1) / small.clamp(min=1e-30)).max()) * 2.0 ** -22
            check_held(*key, want[r, nh + h], min(slack, 1e-3))
            codes, scales = plain.hold(x[r, nh + nkv + h])
            assert torch.equal(value[1], scales) and torch.equal(value[0], codes)       # (nothing but the rounding itself)
            plain.write_token(marked[0][page, h], off, *key, 8)
            plain.write_token(marked[1][page, h], off, *value, 4)
    assert torch.equal(marked[0], after[0]) and torch.equal(marked[1], after[1])         # no other byte has changed
    # ... and what is read back is what the bytes stand for, in both types
    for out in (BF16, F32):
        k, v = (torch.full((n, nkv, hd), 7.0, dtype=out, device=DEV) for _ in range(2))
        st2 = status()
        kernels.kv4_read(pools[0], pools[1], dev[2], k, v, page_size, st2)
        assert int(st2) == 0
        for r in range(min(n, 40)):
            page, off = int(slots[r]) // page_size, int(slots[r]) % page_size
            for h in range(nkv):
                assert torch.equal(k[r, h].cpu().to(F64), plain.numbers(*plain.read_token(after[0][page, h], off, hd, 8)))
                assert torch.equal(v[r, h].cpu().to(F64), plain.numbers(*plain.read_token(after[1][page, h], off, hd, 4)))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups_at_the_edges(dtype):
    """Zeros, tiny and huge numbers, ties of both kinds, NaN and infinities: each in a group of its own (keys and values, not turned)."""
    from glassbox_b200 import kernels
    hd, inf, nan = 256, math.inf, math.nan
    x = torch.zeros(8, 32, dtype=F64)
    x[1] = torch.randn(32, generator=torch.Generator().manual_seed(2), dtype=F64) * 2.0 ** -120
    x[2] = torch.randn(32, generator=torch.Generator().manual_seed(3), dtype=F64) * 1e37
    x[3, :17] = torch.arange(-8, 9).to(F64) * 0.5 - 0.25                       # halves of steps of a scale of a half
    x[3, 20] = 4.0
    x[4, 3], x[4, 9] = -2.0, 2.0                                              # the positive one of two
    x[5, 7] = nan
    x[6, 0], x[6, 1] = inf, 1.0
    x[7, 31], x[7, 2] = -inf, nan
    x = x.to(dtype).to(F64)
    row = x.reshape(1, -1)
    qkv = torch.cat([torch.zeros(1, hd, dtype=F64), row, row], dim=1).to(dtype).to(DEV)
    pools = [torch.zeros(1, 1, kernels.kv4_page_bytes(16, hd), dtype=torch.uint8, device=DEV) for _ in range(2)]
    one = torch.full((1,), 5, dtype=torch.int32, device=DEV)
    _, st = write(qkv, one, one, None, *pools, 1, 1, hd, 0, 16)
    codes, scales = plain.hold(x.reshape(-1))
    assert st == 0 and scales[0] == 0 and scales[1] == 0 and scales[4] == -0.25 and scales[5:].isnan().all()
    k, v = (torch.zeros(1, 1, hd, dtype=F32, device=DEV) for _ in range(2))
    kernels.kv4_read(*pools, one, k, v, 16, status())
    for pool, per, back in ((pools[0], 8, k), (pools[1], 4, v)):
        got = plain.read_token(pool[0, 0].cpu(), 5, hd, per)
        assert torch.equal(got[0], codes) and torch.equal(got[1][:5], scales[:5]) and got[1][5:].isnan().all()
        assert torch.equal(back[0, 0, :160].cpu().to(F64), plain.numbers(codes, scales)[:160]) and back[0, 0, 160:].isnan().all()


def test_rows_that_are_not_stored():
    """Padding, slots and positions outside their ranges, a step that does not write the cache, rows with room between them."""
    from glassbox_b200 import kernels
    n, nh, nkv, hd = 6, 3, 1, 64
    wide = torch.randn(n, 5 * hd + 24, device=DEV).to(BF16)
    qkv = wide[:, 8:8 + 5 * hd]
    q_wide = torch.full((n, nh * hd + 8), 7.0, dtype=BF16, device=DEV)
    angle = torch.rand(10, 32, device=DEV)
    table = torch.stack([angle.cos(), angle.sin()], -1).contiguous()
    positions = torch.tensor([0, 9, -1, 10, 3, 4], dtype=torch.int32, device=DEV)          # 10: beyond the table
    slots = torch.tensor([3, 31, 0, 5, 32, -2], dtype=torch.int32, device=DEV)             # 32, -2: outside the pool
    pools = [torch.zeros(2, 1, kernels.kv4_page_bytes(16, hd), dtype=torch.uint8, device=DEV) for _ in range(2)]
    st = status()
    kernels.kv4_write(qkv, q_wide[:, :nh * hd], table, positions, slots, *pools, nh, nkv, hd, hd, 16, True, st)
    assert int(st) == 2 | 4
    assert (q_wide[2] == 7).all() and (q_wide[:, nh * hd:] == 7).all()
    want = turned(qkv.to(F64).view(n, 5, hd)[:, :nh], table[positions.clamp(0, 9).long()].to(F64), hd)
    want[3] = qkv[3].to(F64).view(5, hd)[:nh]                                               # no angle: as it is
    kept = [0, 1, 3, 4, 5]
    got = q_wide[:, :nh * hd].to(F64).view(n, nh, hd)
    assert ((got - want)[kept].abs() <= want[kept].abs() * 2.0 ** -8 + 1e-5).all()
    written = {3, 31, 5}
    for off in range(32):
        codes, scales = plain.read_token(pools[1][off // 16, 0].cpu(), off % 16, hd, 4)
        assert bool((codes != -8).any()) == (off in written)
    # in place, and without storing: the same queries, the cache as it was
    before = [p.clone() for p in pools]
    own, st = qkv.contiguous(), status()
    kernels.kv4_write(own, own[:, :nh * hd], table, positions, slots, *pools, nh, nkv, hd, hd, 16, False, st)
    assert int(st) == 4 and torch.equal(own[kept, :nh * hd], q_wide[kept, :nh * hd]) and torch.equal(own[:, nh * hd:], qkv[:, nh * hd:])
    assert torch.equal(own[2], qkv[2]) and all(torch.equal(a, b) for a, b in zip(before, pools))
    # reading: a negative slot leaves the row, one behind the pool is reported
    k, v = (torch.full((3, 1, hd), 7.0, device=DEV) for _ in range(2))
    st = status()
    kernels.kv4_read(*pools, torch.tensor([3, -1, 32], dtype=torch.int32, device=DEV), k, v, 16, st)
    assert int(st) == 2 and (k[1:] == 7).all() and (v[1:] == 7).all() and not (k[0] == 7).all()


def test_nothing_to_do():
    from glassbox_b200 import kernels
    pools = [torch.zeros(2, 1, kernels.kv4_page_bytes(16, 64), dtype=torch.uint8, device=DEV) for _ in range(2)]
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    kernels.kv4_write(torch.empty(0, 192, device=DEV), torch.empty(0, 64, device=DEV), None, none, none, *pools, 1, 1, 64, 0, 16, True, status())
    kernels.kv4_read(*pools, none, torch.empty(0, 1, 64, device=DEV), torch.empty(0, 1, 64, device=DEV), 16, status())
    q = torch.empty(0, 64, device=DEV)
    kernels.kv4_attention_decode(q, q.clone(), *pools, torch.zeros(1, 1, dtype=torch.int32, device=DEV), none, none, 1, 1, 64, 16, 0.1, None, 16, None, status())
    kernels.token_logprobs(torch.empty(0, 9, device=DEV), none, torch.empty(0, device=DEV))


# ------------------------------------------------------------------------------------------------ attention
def tables_for(lengths, pages, page_size, seed, spare=1):
    g = torch.Generator().manual_seed(seed)
    ids, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    need = [-(-x // page_size) for x in lengths]
    t = torch.full((len(lengths), max(need + [1]) + spare), -1, dtype=torch.int32)
    for i, c in enumerate(need):
        t[i, :c] = ids[at:at + c]
        at += c
    return t


def reference(q, dense, tables, row_seq, positions, nh, nkv, scale, window):
    """(out, sum of p |v|, largest sum of |q k| scale) in float64; q [n, nh * hd]."""
    hd, page_size = dense[0].shape[-1], dense[0].shape[2]
    n, out = q.shape[0], torch.zeros(q.shape[0], nh, q.shape[1] // nh, dtype=F64)
    size, most = torch.zeros_like(out), 0.0
    q = q.to(F64).view(n, nh, hd)
    for r in range(n):
        p = int(positions[r])
        if p < 0:
            continue
        pages = tables[int(row_seq[r])][:p // page_size + 1].long()
        lo = max(0, p + 1 - window) if window else 0
        missing = (pages < 0) | (pages >= dense[0].shape[0])
        k, v = (d[pages.clamp(0, d.shape[0] - 1)].transpose(0, 1).flatten(1, 2)[:, :p + 1] for d in dense)
        hidden = missing.repeat_interleave(page_size)[:p + 1].clone()
        hidden[:lo] = True
        for h in range(nh):
            kk, vv = k[h // (nh // nkv)], v[h // (nh // nkv)]
            if bool(hidden.all()):
                continue
            s = (kk @ q[r, h] * scale).masked_fill(hidden, -math.inf)
            w = torch.softmax(s, 0)
            w_seen, v_seen = w[~hidden], vv[~hidden]
            out[r, h], size[r, h] = w_seen @ v_seen, w_seen @ v_seen.abs()
            most = max(most, float((kk[~hidden].abs() @ q[r, h].abs()).max()) * scale)
    return out.flatten(1), size.flatten(1), most


def allowed(dtype, want, size, most, hd, keys):
    """What the arithmetic may be off by: scores are float32 sums of hd products and hd / 32 scales (each addition half a step of the sum of
    magnitudes; ``most`` bounds it), their exponential moves by as much and some 2^-21 of its own, in numerator and denominator; sums
    over the keys likewise; in bfloat16 a weight (with its value's scale) may be rounded before its product, once; then the result."""
    scores = (hd + 16) * 2.0 ** -24 * most + 2.0 ** -21
    weights = 2 * scores + (keys / 16 + 32) * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0.0)
    return size * weights + want.abs() * HALF_STEP[dtype] + 1e-30


LAYOUTS = [(9, 3, 64), (4, 4, 64), (8, 2, 128), (3, 1, 32), (6, 2, 96), (4, 1, 256), (12, 1, 64), (20, 1, 128), (2, 2, 128), (17, 1, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh, nkv, hd", LAYOUTS)
@pytest.mark.parametrize("page_size, window", [(16, None), (48, 21), (64, None)])
def test_decode(dtype, nh, nkv, hd, page_size, window):
    from glassbox_b200 import kernels
    lengths = [1, 16, 17, 33, 130, 300, 64, 15]
    pages = sum(-(-x // page_size) for x in lengths) + 2
    pools, dense = plain.random_pool(pages, nkv, page_size, hd, nh + hd)
    tables = tables_for(lengths, pages, page_size, 3)
    n, scale = len(lengths) + 1, 1 / math.sqrt(hd)
    q = torch.randn(n, nh * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    row_seq = torch.tensor(list(range(len(lengths)))[::-1] + [0], dtype=torch.int32)
    positions = torch.tensor([x - 1 for x in lengths[::-1]] + [-1], dtype=torch.int32)
    want, size, most = reference(q, dense, tables, row_seq, positions, nh, nkv, scale, window)
    room = torch.full((n, nh * hd + 16), 7.0, dtype=dtype, device=DEV)
    q_room = torch.zeros(n, nh * hd + 8, dtype=dtype, device=DEV)
    q_room[:, :nh * hd] = q.to(DEV)
    dev = [t.to(DEV) for t in (*pools, tables, row_seq, positions)]
    for reach in (300, 5000):                                    # (more shares than the keys fill, too)
        st, out = status(), room[:, 8:8 + nh * hd]
        qd = q_room[:, :nh * hd]
        parts = kernels.kv4_decode_parts(qd, nh, nkv, hd, reach)
        if parts is not None:
            parts.fill_(math.nan)
        kernels.kv4_attention_decode(qd, out, *dev, nh, nkv, hd, page_size, scale, window, reach, parts, st)
        assert int(st) == 0
        off = (out.cpu().to(F64) - want).abs() - allowed(dtype, want, size, most, hd, 300)
        assert (off <= 0).all(), float(off.max())
        assert (out[-1] == 0).all() and (room[:, :8] == 7).all() and (room[:, 8 + nh * hd:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_skips_bad_pages_and_positions(dtype, hd):
    from glassbox_b200 import kernels
    pools, dense = plain.random_pool(8, 1, 16, hd, 4)
    tables = torch.tensor([[0, -1, 2, 3], [4, 8, 5, 1], [-1, -1, -1, -1], [6, 7, 1, 0]], dtype=torch.int32)
    positions = torch.tensor([40, 40, 20, 64], dtype=torch.int32)            # the last: behind what its table covers
    row_seq = torch.arange(4, dtype=torch.int32)
    q = torch.randn(4, 2 * hd, generator=torch.Generator().manual_seed(1)).to(dtype)
    want, size, most = reference(q[:3], dense, tables, row_seq, positions[:3], 2, 1, 0.1, None)
    st, out = status(), torch.full((4, 2 * hd), 7.0, dtype=dtype, device=DEV)
    qd = q.to(DEV)
    parts = kernels.kv4_decode_parts(qd, 2, 1, hd, 64)
    kernels.kv4_attention_decode(qd, out, *[t.to(DEV) for t in (*pools, tables, row_seq, positions)], 2, 1, hd, 16, 0.1, None, 64, parts, st)
    assert int(st) == 2 | 4
    assert ((out[:3].cpu().to(F64) - want).abs() <= allowed(dtype, want, size, most, hd, 41)).all()
    assert (out[2:] == 0).all()


def poison(pool, page, off, hd, group):
    """A group's scale becomes NaN."""
    at = off // 16 * 9 * hd + 8 * hd + (off % 16 * (hd // 32) + group) * 2
    pool[page, 0, at:at + 2] = torch.tensor([0xc0, 0x7f], dtype=torch.uint8)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_nan_is_seen_only_where_its_token_is(dtype, hd):
    """Tokens behind a row, before its window or of other requests may hold NaN; one in sight makes the head's row (a key) or the
    channels of its group (a value) NaN."""
    from glassbox_b200 import kernels
    for at, tensor in ((30, 0), (30, 1), (2, 0), (2, 1), (20, 0), (20, 1)):
        pools, dense = plain.random_pool(3, 1, 16, hd, 6)
        poison(pools[tensor], at // 16, at % 16, hd, 1)
        args = [t.to(DEV) for t in (*pools, torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.tensor([25], dtype=torch.int32))]
        q = torch.randn(1, 2 * hd, generator=torch.Generator().manual_seed(1)).to(dtype)
        out = torch.empty(1, 2 * hd, dtype=dtype, device=DEV)
        qd = q.to(DEV)
        kernels.kv4_attention_decode(qd, out, *args, 2, 1, hd, 16, 0.1, 16, 48, kernels.kv4_decode_parts(qd, 2, 1, hd, 48), status())
        nan = out.cpu().view(2, hd // 32, 32).isnan()
        if at != 20:
            assert not nan.any()
        elif tensor == 0:
            assert nan.all()
        else:
            assert nan[:, 1].all() and not nan[:, 0].any() and not nan[:, 2:].any()
    # prompts: what lies behind the request's last token, and before its window
    for at, tensor in ((30, 0), (30, 1), (2, 0), (2, 1)):
        pools, dense = plain.random_pool(3, 1, 16, hd, 6)
        clean = [p.clone() for p in pools]
        poison(pools[tensor], at // 16, at % 16, hd, 1)
        outs = []
        for pair in (clean, pools):
            pages = [torch.zeros(3, 1, 16, hd, dtype=dtype, device=DEV) for _ in range(2)]
            q = torch.randn(6, 2 * hd, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
            ints = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([[0, 1, 2]], [0] * 6, list(range(20, 26)), [0, 6], [20])]
            outs.append(torch.empty_like(q))
            kernels.kv4_attention_prefill(q, outs[-1], *[p.to(DEV) for p in pair], *ints, 6, 2, 1, hd, 16, 0.1, 16, 48, *pages, status())
        assert torch.equal(outs[0], outs[1]) and not outs[1].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh, nkv, hd", LAYOUTS)
@pytest.mark.parametrize("page_size, window", [(16, None), (16, 40), (64, None)])
def test_prompts(dtype, nh, nkv, hd, page_size, window):
    from glassbox_b200 import kernels
    rows, past = [1, 70, 5, 16], [40, 0, 129, 16]
    total = [r + p for r, p in zip(rows, past)]
    pages = sum(-(-x // page_size) for x in total) + 2
    pools, dense = plain.random_pool(pages, nkv, page_size, hd, nh + hd)
    tables = torch.cat([tables_for(total, pages, page_size, 3), torch.full((2, max(-(-x // page_size) for x in total) + 1), -1, dtype=torch.int32)])
    first, row_seq, positions = [0], [], []
    for i, (r, p) in enumerate(zip(rows, past)):
        first.append(first[-1] + r)
        row_seq += [i] * r
        positions += list(range(p, p + r))
    n, pad = first[-1], 4                                        # rows behind the last request: padding
    first, start = first + [n, n], past + [-1, -1]
    row_seq, positions = row_seq + [0] * pad, positions + [-1] * pad
    q = torch.randn(n + pad, nh * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    ints = [torch.tensor(v, dtype=torch.int32) for v in (row_seq, positions, first, start)]
    scale = 1 / math.sqrt(hd)
    want, size, most = reference(q[:n], dense, tables, ints[0], ints[1][:n], nh, nkv, scale, window)
    st, out = status(), torch.zeros(n + pad, nh * hd, dtype=dtype, device=DEV)
    kp, vp = (torch.zeros(pages, nkv, page_size, hd, dtype=dtype, device=DEV) for _ in range(2))
    kernels.kv4_attention_prefill(q.to(DEV), out, *[t.to(DEV) for t in (*pools, tables, *ints)], max(rows), nh, nkv, hd, page_size, scale, window,
                                  max(total), kp, vp, st)
    assert int(st) == 0
    # (float32 prompts form products of exact three-term splits: a few more roundings than a fused sum, all within hd + 16)
    off = (out[:n].cpu().to(F64) - want).abs() - allowed(dtype, want, size, 2 * most, hd, 140)
    assert (off <= 0).all(), float(off.max())
    # unpacked, the pages in sight hold exactly what the codes stand for
    dev = [t.to(DEV) for t in (*pools, tables, ints[2], ints[3])]
    kernels.kv4_expand(dev[0], dev[1], kp.zero_(), vp.zero_(), *dev[2:], max(total), window, st)
    assert int(st) == 0
    for d, p in zip(dense, (kp, vp)):
        for i, x in enumerate(total):
            lo = max(0, past[i] + 1 - window) if window else 0
            for j in range(lo // page_size, -(-x // page_size)):
                assert torch.equal(p[int(tables[i, j])].cpu().to(F64), d[int(tables[i, j])])


def test_prompt_reports_missing_pages():
    from glassbox_b200 import kernels
    pools, _ = plain.random_pool(3, 1, 16, 64, 6)
    pages = [torch.zeros(3, 1, 16, 64, dtype=BF16, device=DEV) for _ in range(2)]
    q = torch.randn(6, 64, device=DEV).to(BF16)
    ints = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([[0, -1, 2]], [0] * 6, list(range(30, 36)), [0, 6], [30])]
    st, out = status(), torch.empty_like(q)
    kernels.kv4_attention_prefill(q, out, *[p.to(DEV) for p in pools], *ints, 6, 1, 1, 64, 16, 0.1, None, 48, *pages, st)
    assert int(st) & 2


def test_pools_beyond_32_bits():
    """Pages whose bytes lie behind 2^32 in their pool: written, read back and attended to."""
    from glassbox_b200 import kernels
    nkv, hd, size = 8, 128, kernels.kv4_page_bytes(16, 128)
    pages = (1 << 32) // (nkv * size) + 300
    pools = [torch.zeros(pages, nkv, size, dtype=torch.uint8, device=DEV) for _ in range(2)]
    n = 40
    qkv = torch.randn(n, 3 * nkv * hd, generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
    ids = [pages - 1, pages - 7, pages - 2]
    slots = torch.tensor([ids[i // 16] * 16 + i % 16 for i in range(n)], dtype=torch.int32, device=DEV)
    positions = torch.arange(n, dtype=torch.int32, device=DEV)
    q, st = write(qkv, positions, slots, None, *pools, nkv, nkv, hd, 0, 16)
    assert st == 0
    k, v = (torch.empty(n, nkv, hd, device=DEV) for _ in range(2))
    kernels.kv4_read(*pools, slots, k, v, 16, status())
    codes, scales = plain.hold(qkv[3].cpu().to(F64).view(3, nkv, hd)[1])
    assert torch.equal(k[3].cpu().to(F64), plain.numbers(codes, scales))
    out = torch.empty_like(q)
    tables = torch.tensor([ids], dtype=torch.int32, device=DEV)
    zeros = torch.zeros(n, dtype=torch.int32, device=DEV)
    kernels.kv4_attention_decode(q, out, *pools, tables, zeros, positions, nkv, nkv, hd, 16, 0.1, None, n, kernels.kv4_decode_parts(q, nkv, nkv, hd, n), status())
    s = torch.einsum("rhc,khc->hrk", q.double().view(n, nkv, hd), k.double()) * 0.1
    w = torch.softmax(s.masked_fill(torch.arange(n, device=DEV)[None, :] > torch.arange(n, device=DEV)[:, None], -math.inf), -1)
    want, most = torch.einsum("hrk,khc->rhc", w, v.double()).flatten(1), float(s.abs().max()) * 30
    size_of = torch.einsum("hrk,khc->rhc", w, v.double().abs()).flatten(1)
    assert ((out.double() - want).abs() <= allowed(BF16, want, size_of, most, hd, n)).all()


def test_recorded_and_on_another_stream():
    """Write, then attend, recorded into a graph and replayed with other inputs, and run on a stream of its own."""
    from glassbox_b200 import kernels
    n, nh, nkv, hd, past = 3, 4, 2, 64, 700
    pools, dense = plain.random_pool(200, nkv, 16, hd, 8)
    tables = tables_for([past + 1] * n, 200, 16, 5).to(DEV)
    positions = torch.full((n,), past, dtype=torch.int32, device=DEV)
    row_seq = torch.arange(n, dtype=torch.int32, device=DEV)
    slots = (tables[:, past // 16] * 16 + past % 16).to(torch.int32)
    qkv = torch.randn(n, 8 * hd, device=DEV).to(BF16)
    start = [p.to(DEV) for p in pools]

    def run(pools, q, out, parts, st):
        kernels.kv4_write(qkv, q, None, positions, slots, *pools, nh, nkv, hd, 0, 16, True, st)
        kernels.kv4_attention_decode(q, out, *pools, tables, row_seq, positions, nh, nkv, hd, 16, 0.1, None, past + 1, parts, st)

    def buffers():
        q = torch.empty(n, nh * hd, dtype=BF16, device=DEV)
        return [p.clone() for p in start], q, torch.empty_like(q), kernels.kv4_decode_parts(q, nh, nkv, hd, past + 1), status()

    recorded = buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*recorded)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(*recorded)
    for _ in range(3):
        qkv.copy_(torch.randn(n, 8 * hd, device=DEV))
        torch.cuda.synchronize()
        plainly = buffers()
        run(*plainly)
        on_side = buffers()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*on_side)
        graph.replay()
        torch.cuda.synchronize()
        for other in (recorded, on_side):
            assert torch.equal(other[2], plainly[2]) and torch.equal(other[0][0], plainly[0][0]) and torch.equal(other[0][1], plainly[0][1])
            assert int(other[4]) == 0
