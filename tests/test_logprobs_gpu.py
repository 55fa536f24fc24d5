"""Log probabilities of given tokens, entropies and most probable tokens against softmax in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F64 = torch.float64


def score(logits, tokens, top, entropy=True):
    from glassbox_b200 import kernels
    n = logits.shape[0]
    lp, h = torch.full((n,), 7.0, device=DEV), torch.full((n,), 7.0, device=DEV) if entropy else None
    best = torch.full((n, top), 7.0, device=DEV) if top else None
    ids = torch.full((n, top), -7, dtype=torch.int32, device=DEV) if top else None
    kernels.token_logprobs(logits, tokens, lp, h, best, ids)
    return lp, h, best, ids


def check(logits, tokens, top):
    """All of the results against 64 bits. What the arithmetic may be off by: a logit less the largest is rounded once, as is its product
    with log2(e); an exponential is good to some 2^-22, and the terms of a sum are each at most vocab / 256 + 64 additions deep: all of it relative to the sum
    of exponentials, each weighted with 1 + |x - m|, whose mean over the distribution is at most 1 + ln(vocab) + |x - m| of the rest."""
    vocab = logits.shape[1]
    lp, h, best, ids = score(logits, tokens, top)
    x = logits.to(F64)
    m = x.amax(-1, keepdim=True)
    z = torch.logsumexp(x, -1, keepdim=True)
    p = torch.softmax(x, -1)
    d = torch.where(p > 0, x - z, 0.0)
    want_h = -(p * d).sum(-1)
    far = (p * torch.where(p > 0, (x - m).abs(), 0.0)).sum(-1)                        # mean distance below the largest
    relative = (vocab / 256 + 64) * 2.0 ** -24 + 4 * 2.0 ** -24 * (1 + far)
    ok = (tokens >= 0) & (tokens < vocab)
    want = (x - z).gather(1, tokens.clamp(0, vocab - 1).long()[:, None])[:, 0]
    assert torch.equal(lp.isnan(), ~ok)
    finite = ok & want.isfinite()
    assert torch.equal(lp[ok & ~finite], want[ok & ~finite].float())
    assert ((lp.double() - want).abs() <= relative + 3 * 2.0 ** -24 * ((x - z).gather(1, tokens.clamp(0, vocab - 1).long()[:, None])[:, 0].abs() + (m - z)[:, 0].abs() + 1))[finite].all()
    assert ((h.double() - want_h).abs() <= relative * (2 + 2 * far)).all(), float((h.double() - want_h).abs().max())
    if top:
        value, index = torch.sort(x + 0.0, dim=-1, descending=True, stable=True)
        assert torch.equal(ids.long(), index[:, :top])
        want = value[:, :top] - z
        inf = want.isinf()
        assert torch.equal(best[inf], want[inf].float())
        assert ((best.double() - want).abs() <= relative[:, None] + 3 * 2.0 ** -24 * (want.abs() + (m - z).abs() + 1))[~inf].all()
    return lp, h, best, ids


SHAPES = [(1, 1, 1), (1, 5, 5), (3, 33, 32), (2, 511, 4), (5, 513, 20), (1, 49152, 8), (4, 49153, 32), (7, 8191, 0), (2, 100003, 20), (300, 1000, 3), (1, 262144, 32),
          (17, 16384, 1), (40, 4097, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab, top", SHAPES)
def test_scores(dtype, rows, vocab, top):
    g = torch.Generator(device=DEV).manual_seed(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
    check(logits, tokens, top)
    logits = logits.masked_fill(torch.rand(rows, vocab, generator=g, device=DEV) < 0.9, -math.inf)
    logits[:, vocab // 2] = 1.0
    check(logits, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("start, room", [(0, 0), (1, 3), (4, 12), (3, 1)])
def test_rows_with_room_between_them(dtype, start, room):
    g = torch.Generator(device=DEV).manual_seed(start)
    wide = torch.full((6, start + 5003 + room), 90.0, device=DEV).to(dtype)                # (what lies between must not count)
    wide[:, start:start + 5003] = torch.randn(6, 5003, generator=g, device=DEV).to(dtype)
    check(wide[:, start:start + 5003], torch.arange(6, device=DEV, dtype=torch.int32) * 1000, 20)


@pytest.mark.parametrize("vocab", [40, 5000, 60000])
def test_orders_of_all_kinds(vocab):
    """Rows that only rise, only fall, are all the same, hold few different numbers, a single token, signed zeros, huge numbers."""
    x = torch.zeros(9, vocab, device=DEV)
    ramp = torch.arange(vocab, device=DEV, dtype=torch.float32) / vocab * 20
    x[0], x[1], x[2] = ramp, -ramp, 0.25
    x[3] = (torch.arange(vocab, device=DEV) * 7919 % 3).float()
    x[4], x[4, vocab - 2] = -math.inf, -5.0
    x[5, ::2] = -0.0
    x[6] = torch.where(torch.arange(vocab, device=DEV) % 2 == 0, 3e38, -3e38)
    x[7] = torch.where(torch.arange(vocab, device=DEV) < vocab - 3, -math.inf, 1.0)
    x[8] = torch.where(torch.arange(vocab, device=DEV) % 5 == 4, ramp, -math.inf)
    tokens = torch.tensor([0, 3, 5, 7, vocab - 2, 2, 0, vocab - 1, 4], dtype=torch.int32, device=DEV)
    rows = [0, 1, 2, 3, 4, 5, 7, 8]
    check(x[rows].contiguous(), tokens[rows], 32)
    lp, h, best, ids = score(x[6:7].contiguous(), tokens[6:7], 32)
    half = -math.log((vocab + 1) // 2)
    assert abs(float(lp) - half) < 1e-4 and abs(float(h) + half) < 1e-4
    assert ids[0].tolist()[:20] == list(range(0, 40, 2))[:20]


def test_rows_without_a_distribution():
    x = torch.randn(6, 700, device=DEV)
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, 9] = math.inf
    x[3], x[3, 1] = math.nan, 2.0
    tokens = torch.tensor([3, 3, 9, 1, -1, 700], dtype=torch.int32, device=DEV)
    lp, h, best, ids = score(x, tokens, 8)
    assert lp.isnan().all() and h[:4].isnan().all() and best[:4].isnan().all()
    assert not h[4:].isnan().any() and not best[4:].isnan().any()
    assert ids[0].tolist() == list(range(8)) and ids[2, 0] == 9 and ids[3].tolist() == [1, 0, 2, 3, 4, 5, 6, 7]
    assert ids[1].tolist() == torch.where(x[1].isnan(), -math.inf, x[1]).topk(8).indices.tolist()


def test_what_is_not_asked_for():
    x, tokens = torch.randn(4, 300, device=DEV), torch.arange(4, device=DEV, dtype=torch.int32)
    whole = score(x, tokens, 4)
    assert torch.equal(score(x, tokens, 0, entropy=False)[0], whole[0])
    from glassbox_b200 import kernels
    lp, ids = torch.empty(4, device=DEV), torch.empty(4, 4, dtype=torch.int32, device=DEV)
    kernels.token_logprobs(x, tokens, lp, None, None, ids)
    assert torch.equal(ids, whole[3])


def test_a_row_does_not_depend_on_the_others_and_repeats():
    x = torch.randn(200, 50001, device=DEV) * 3
    tokens = torch.randint(0, 50001, (200,), device=DEV, dtype=torch.int32)
    a, b = score(x, tokens, 20), score(x, tokens, 20)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = score(x[7:8], tokens[7:8], 20)
    assert (one[0] - a[0][7]).abs() < 1e-5 and torch.equal(one[3][0], a[3][7])


def test_recorded():
    x = torch.randn(3, 49152, device=DEV)
    tokens = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    from glassbox_b200 import kernels
    lp, h, best, ids = torch.empty(3, device=DEV), torch.empty(3, device=DEV), torch.empty(3, 9, device=DEV), torch.empty(3, 9, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.token_logprobs(x, tokens, lp, h, best, ids)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.token_logprobs(x, tokens, lp, h, best, ids)
    for _ in range(2):
        x.copy_(torch.randn(3, 49152, device=DEV))
        graph.replay()
        want = score(x, tokens, 9)
        assert torch.equal(lp, want[0]) and torch.equal(h, want[1]) and torch.equal(best, want[2]) and torch.equal(ids, want[3])
