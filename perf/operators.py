"""The operators of a cache held in 4 bits, and of scoring, as cases that can be timed and compared.

Three operators and what a program that serves a model calls of them:

* ``write``: the rows of a step are rotated, their keys and values rounded to 4 bits and stored in the pages of a
  cache; then what the cache now holds for these rows is read back.
* ``decode``, ``prompt``: softmax attention over such a cache, for single decoded tokens and for portions of prompts.
* ``score``: the log probabilities of given tokens, the entropy of each row's distribution and its most probable tokens.

How a cache in 4 bits looks. 32 neighbouring channels of a token and head are a group. With m the group's number of the largest
magnitude (the positive one of two), its scale is -m / 8 rounded to five significant bits, and a number x is held as the whole
number s nearest to x / scale (ties to even), from -8 to 7: it stands for s * scale, which bfloat16 holds exactly. A group with a number
that is not finite stands for NaN, one whose numbers are all below 2^-117 for zeros. A page of a head is a run of tiles of 16 tokens;
a tile is 16 rows of codes (s + 8, two in a byte, the first in the low half), then 16 rows of scales (bfloat16, one a group). In a row of codes
of hd channels, G = hd / 32 groups, channel c of a key is nibble ((c % 32) // 8 * G + c // 32) * 8 + c % 8, of a value
((c % 32) // 4 * G + c // 32) * 4 + c % 4.

Sizes are those of the SmolLM2 shapes (9/3, 15/5 and 32/32 heads of 64) and of wider layouts (32/8 heads of 128).
"""
import math

import torch

own = False

PAGE = 16
TILE = 16
GROUP = 32
ROPE_BASE = 100000.0
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
F64 = torch.float64


def listed():
    return [
        # eight decoded tokens of the smallest model: one small launch, where latency is all
        dict(name="write_decode_8", kind="write", dtype="bfloat16", rows=8, nh=9, nkv=3, hd=64, rot=64),
        # a prompt in the 32-bit path, a number of rows that is no round one
        dict(name="write_fp32_1001", kind="write", dtype="float32", rows=1001, nh=15, nkv=5, hd=64, rot=64),
        # a long prompt of a wide model, half of every head rotated
        dict(name="write_wide_8000", kind="write", dtype="bfloat16", rows=8000, nh=32, nkv=8, hd=128, rot=64),
        # one user's generation with a short context: the smallest attention call there is
        dict(name="decode_135m_b1", kind="decode", dtype="bfloat16", seqs=1, past=1023, ragged=False, nh=9, nkv=3, hd=64, window=0),
        # a full decode batch at the benchmark's context, every head with keys of its own
        dict(name="decode_1.7b_b64", kind="decode", dtype="bfloat16", seqs=64, past=4095, ragged=False, nh=32, nkv=32, hd=64, window=0),
        # a service's decode batch of unequal contexts, four queries a key
        dict(name="decode_wide_b24", kind="decode", dtype="bfloat16", seqs=24, past=9001, ragged=True, nh=32, nkv=8, hd=128, window=0),
        # two requests with very long contexts: few rows, a long axis
        dict(name="decode_long_b2", kind="decode", dtype="bfloat16", seqs=2, past=131071, ragged=False, nh=32, nkv=8, hd=128, window=0),
        # later portions of two prompts behind what the cache already holds
        dict(name="prompt_360m_1500", kind="prompt", dtype="bfloat16", seqs=2, rows=1500, past=900, nh=15, nkv=5, hd=64, window=0),
        # a long portion of a wide model's prompt
        dict(name="prompt_wide_2048", kind="prompt", dtype="bfloat16", seqs=1, rows=2048, past=2048, nh=32, nkv=8, hd=128, window=0),
        # the token that one request has just been given, with eight alternatives
        dict(name="score_1", kind="score", dtype="float32", rows=1, vocab=49152, top=8, masked=False),
        # a whole prompt scored, with twenty alternatives a token
        dict(name="score_2048", kind="score", dtype="float32", rows=2048, vocab=49152, top=20, masked=False),
        # bfloat16 logits of a large odd vocabulary, parts of which a grammar rules out
        dict(name="score_odd_1000", kind="score", dtype="bfloat16", rows=1000, vocab=100003, top=5, masked=True),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "prompt", "score", "score"])
    dtype = "bfloat16" if rng.random() < 0.75 else "float32"
    if kind == "score":
        rows, vocab = _between(rng, 1, 2048), _between(rng, 300, 150000)
        rows = max(1, min(rows, 2048 * 49152 // vocab))
        return dict(kind="score", dtype=dtype, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, 32]), masked=rng.random() < 0.3)
    nh, nkv = rng.choice([(9, 3), (15, 5), (32, 32), (32, 8), (16, 2), (12, 1), (7, 7)])
    hd = rng.choice([32, 64, 64, 96, 128, 128, 256])
    if kind == "write":
        rows = min(_between(rng, 1, 8000), 8000 * 48 * 128 // ((nh + 2 * nkv) * hd))
        return dict(kind="write", dtype=dtype, rows=rows, nh=nh, nkv=nkv, hd=hd, rot=rng.choice([hd, hd // 2, 0]))
    window = rng.choice([0, 0, _between(rng, 10, 2000)])
    if kind == "decode":
        seqs = _between(rng, 1, 64)
        most = 64 * 4096 * 32 * 64 // (seqs * nkv * hd * (1 if dtype == "bfloat16" else 8))
        past = _between(rng, 1, max(2, min(most, 131071)))
        return dict(kind="decode", dtype=dtype, seqs=seqs, past=past, ragged=rng.random() < 0.7, nh=nh, nkv=nkv, hd=hd, window=window)
    rows = min(_between(rng, 70, 2048), 2048 * 32 * 128 // (nh * hd))
    past = rng.choice([0, _between(rng, 20, 2048)])
    if dtype == "float32":
        rows, past = min(rows, 600), min(past, 600)
    return dict(kind="prompt", dtype=dtype, seqs=rng.randint(1, 3), rows=max(rows, 3), past=past, nh=nh, nkv=nkv, hd=hd, window=window)


# ------------------------------------------------------------------------------------------------ shapes of a batch
def _spread(case):
    """(rows, tokens in the cache before them) of each sequence: decoded tokens behind between half and all of ``past``, portions
    of prompts of unequal lengths behind ``past`` tokens."""
    n = case["seqs"]
    if case["kind"] == "decode":
        past = case["past"]
        return [1] * n, [past - (past // 2) * i // max(n - 1, 1) if case["ragged"] else past for i in range(n)]
    first = case["rows"] // n
    rows = [first - first // 3 * (i % 2) for i in range(n)]
    rows[-1] += case["rows"] - sum(rows)
    return rows, [case["past"]] * n


def _visible(case):
    """(keys that some row sees, pairs of a row and a key that it sees), over all sequences."""
    window, keys, pairs = case["window"], 0, 0
    rows, past = _spread(case)
    for r, p in zip(rows, past):
        keys += min(p + r, r - 1 + window) if window else p + r
        if window:
            short = max(0, min(r, window - p))          # rows that see less than a window
            pairs += short * p + short * (short + 1) // 2 + (r - short) * window
        else:
            pairs += r * p + r * (r + 1) // 2
    return keys, pairs


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "score":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * size + n * (4 + 8 + 8 * k), "flops": 6 * n * v}
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    held = hd * 9 // 16                                  # bytes of a key or a value of one head
    if case["kind"] == "write":
        n = case["rows"]
        return {"bytes": n * ((2 * nh + 2 * nkv) * hd * size + 4 * case["rot"] + 8 + 2 * nkv * (2 * held + 2 * hd)),
                "flops": n * (3 * (nh + nkv) * case["rot"] + 2 * 4 * nkv * hd)}
    keys, pairs = _visible(case)
    n = sum(_spread(case)[0])
    return {"bytes": keys * nkv * 2 * held + 2 * n * nh * hd * size, "flops": 4 * pairs * nh * hd}


# ------------------------------------------------------------------------------------------------ inputs
def _table(rot, longest, device):
    """cos and sin of every position's angles, [positions, rot / 2, 2]."""
    if not rot:
        return None
    inv = torch.pow(ROPE_BASE, -torch.arange(0, rot, 2, dtype=F64, device=device) / rot)
    angle = torch.arange(longest, dtype=F64, device=device)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float()


def _five_bits(x):
    """x rounded to five significant bits, ties to even."""
    mantissa, exponent = torch.frexp(x)
    return torch.ldexp((mantissa * 32).round(), exponent - 5)


def _to_codes(x):
    """Whole numbers -8 .. 7 and scales [..., G] of x [..., hd]."""
    g = x.unflatten(-1, (-1, GROUP))
    high, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    most = torch.where(high >= -low, high, low)
    scale = _five_bits(-most / 8)
    small = most.abs() < 2.0 ** -117
    scale = torch.where(small, torch.zeros_like(scale), scale)
    s = (g / torch.where(small, torch.ones_like(scale), scale)).round().clamp(-8, 7)
    s = torch.where(small, torch.zeros_like(s), s)
    return s.flatten(-2), scale.squeeze(-1)


def _nibble(hd, per, device):
    """channel -> its nibble in a row of codes; per: neighbouring channels that stay together (8 for keys, 4 for values)."""
    c = torch.arange(hd, device=device)
    return (c % GROUP // per * (hd // GROUP) + c // GROUP) * per + c % per


def _pack(x, per):
    """The cache's bytes [pages, heads, 9 hd * PAGE / 16] of numbers x [pages, heads, PAGE, hd]."""
    s, scale = _to_codes(x)
    hd = x.shape[-1]
    s = (s + 8).to(torch.uint8)
    placed = torch.empty_like(s)
    placed[..., _nibble(hd, per, x.device)] = s
    codes = (placed[..., 0::2] | placed[..., 1::2] << 4).unflatten(-2, (-1, TILE)).flatten(-2)
    scales = scale.to(torch.bfloat16).contiguous().view(torch.uint8).unflatten(-2, (-1, TILE)).flatten(-2)
    return torch.cat([codes, scales], dim=-1).flatten(-2).contiguous()


def _values(cache, hd, per):
    """What the bytes [pages, heads, bytes] stand for: codes (whole) and scales of [pages, heads, PAGE, hd], in float32."""
    tiles = cache.unflatten(-1, (-1, 9 * hd))
    codes = tiles[..., :8 * hd].unflatten(-1, (TILE, hd // 2))
    both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    s = both[..., _nibble(hd, per, cache.device)].flatten(-3, -2).float() - 8
    scale = tiles[..., 8 * hd:].contiguous().view(torch.bfloat16).unflatten(-1, (TILE, hd // GROUP)).flatten(-3, -2).float()
    return s, scale


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "score":
        n, v = case["rows"], case["vocab"]
        logits = torch.randn(n, v, generator=g, device=dev) * 2.5
        tokens = torch.randint(0, v, (n,), generator=g, device=dev, dtype=torch.int32)
        logits[torch.arange(n, device=dev), tokens.long()] += 6.0          # (a text's own tokens are likely ones)
        if case["masked"]:                                                 # (what a grammar rules out, never the whole row)
            out = torch.rand(n, v, generator=g, device=dev) < 0.6
            out[torch.arange(n, device=dev), tokens.long()] = False
            logits.masked_fill_(out, -math.inf)
        return dict(case=case, logits=logits.to(dtype), tokens=tokens)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    if case["kind"] == "write":
        n, rot = case["rows"], case["rot"]
        pages = -(-n // PAGE) + 2
        qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device=dev)
        # (some channels of the keys are much larger than the rest, as in trained models)
        qkv[:, nh * hd:(nh + nkv) * hd] *= torch.exp(torch.randn((nkv * hd), generator=g, device=dev) * 0.7)
        slots = torch.randperm(pages * PAGE, generator=g, device=dev)[:n].sort().values.to(torch.int32)
        first = int(torch.randint(0, 1000, (1,), generator=g, device=dev))
        return dict(case=case, qkv=qkv.to(dtype), table=_table(rot, first + n, dev), positions=torch.arange(first, first + n, dtype=torch.int32, device=dev),
                    slots=slots, k=torch.zeros(pages, nkv, 9 * hd * PAGE // TILE, dtype=torch.uint8, device=dev),
                    v=torch.zeros(pages, nkv, 9 * hd * PAGE // TILE, dtype=torch.uint8, device=dev), status=status)
    rows, past = _spread(case)
    need = [-(-(r + p) // PAGE) for r, p in zip(rows, past)]
    pages, width = sum(need) + 3, max(need) + 1
    ids = torch.randperm(pages, generator=g, device=dev)[:sum(need)].to(torch.int32)
    column = torch.arange(width, device=dev)[None, :]
    counts = torch.tensor(need, device=dev)[:, None]
    tables = torch.full((len(need), width), -1, dtype=torch.int32, device=dev)
    tables[column < counts] = ids
    spread = torch.exp(torch.randn(nkv, 1, hd, generator=g, device=dev) * 0.5)
    k = _pack(torch.randn(pages, nkv, PAGE, hd, generator=g, device=dev) * spread, 8)
    v = _pack(torch.randn(pages, nkv, PAGE, hd, generator=g, device=dev), 4)
    n = sum(rows)
    q = torch.randn(n, nh * hd, generator=g, device=dev).to(dtype)
    firsts = [0]
    for r in rows:
        firsts.append(firsts[-1] + r)
    row_seq = torch.repeat_interleave(torch.arange(len(rows), device=dev), torch.tensor(rows, device=dev)).to(torch.int32)
    first_row, start = _ints(firsts, dev), _ints(past, dev)
    positions = torch.arange(n, device=dev, dtype=torch.int32) - first_row[row_seq.long()] + start[row_seq.long()]
    return dict(case=case, q=q, k=k, v=v, tables=tables, row_seq=row_seq, positions=positions, first_row=first_row, start=start, most=max(rows),
                reach=max(r + p for r, p in zip(rows, past)), scale=1.0 / math.sqrt(hd), window=case["window"] or None, status=status, keep={})


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _OWN[state["case"]["kind"]](state)
    return _PLAIN[state["case"]["kind"]](state)


def _sizes(state):
    return state["case"]["nh"], state["case"]["nkv"], state["case"]["hd"]


def _own_write(s):
    from glassbox_b200 import kernels
    nh, nkv, hd = _sizes(s)
    qkv = s["qkv"]
    n, dev = qkv.shape[0], qkv.device
    q = torch.empty(n, nh * hd, dtype=qkv.dtype, device=dev)
    k, v = (torch.empty(n, nkv, hd, dtype=torch.bfloat16, device=dev) for _ in range(2))
    kernels.kv4_write(qkv, q, s["table"], s["positions"], s["slots"], s["k"], s["v"], nh, nkv, hd, s["case"]["rot"], PAGE, True, s["status"])
    kernels.kv4_read(s["k"], s["v"], s["slots"], k, v, PAGE, s["status"])
    return {"q": q, "k": k, "v": v}


def _own_decode(s):
    from glassbox_b200 import kernels
    nh, nkv, hd = _sizes(s)
    q, keep = s["q"], s["keep"]
    if not keep:                                         # (what a program keeps from call to call)
        keep["parts"] = kernels.kv4_decode_parts(q, nh, nkv, hd, s["reach"])
    out = torch.empty_like(q)
    kernels.kv4_attention_decode(q, out, s["k"], s["v"], s["tables"], s["row_seq"], s["positions"], nh, nkv, hd, PAGE, s["scale"], s["window"],
                                 s["reach"], keep["parts"], s["status"])
    return out


def _own_prompt(s):
    from glassbox_b200 import kernels
    nh, nkv, hd = _sizes(s)
    q, keep = s["q"], s["keep"]
    if not keep:
        keep["k"], keep["v"] = (torch.zeros(s["k"].shape[0], nkv, PAGE, hd, dtype=q.dtype, device=q.device) for _ in range(2))
    out = torch.empty_like(q)
    kernels.kv4_attention_prefill(q, out, s["k"], s["v"], s["tables"], s["row_seq"], s["positions"], s["first_row"], s["start"], s["most"],
                                  nh, nkv, hd, PAGE, s["scale"], s["window"], s["reach"], keep["k"], keep["v"], s["status"])
    return out


def _own_score(s):
    from glassbox_b200 import kernels
    logits, top = s["logits"], s["case"]["top"]
    n, dev = logits.shape[0], logits.device
    logprob, entropy = torch.empty(n, device=dev), torch.empty(n, device=dev)
    best = torch.empty(n, top, device=dev) if top else None
    ids = torch.empty(n, top, dtype=torch.int32, device=dev) if top else None
    kernels.token_logprobs(logits, s["tokens"], logprob, entropy, best, ids)
    return [logprob, entropy] + ([best, ids] if top else [])


def _turned(x, table, positions, rot):
    """x [rows, heads, hd] with channel i and channel i + rot / 2 of the first ``rot`` turned by their row's angle."""
    if not rot:
        return x
    turn = table[positions.long()][:, None].to(x.dtype)
    c, s = turn[..., 0], turn[..., 1]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], dim=-1)


def _plain_write(s):
    nh, nkv, hd = _sizes(s)
    qkv, rot = s["qkv"], s["case"]["rot"]
    q, k, v = qkv.float().unflatten(-1, (-1, hd)).split([nh, nkv, nkv], dim=1)
    q = _turned(q, s["table"], s["positions"], rot)
    k = _turned(k.double(), s["table"], s["positions"], rot)             # (a rounding to 4 bits: what lies next to a border is told in 64)
    held = []
    for x in (k, v.double()):
        codes, scale = _to_codes(x)
        held.append((codes.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2).to(torch.bfloat16))
    return {"q": q.flatten(1).to(qkv.dtype), "k": held[0], "v": held[1]}


def _gathered(s, cache, per):
    """What the pages of each sequence hold, [sequences, heads, tokens, hd], in float32 (pages that a sequence has not: zeros)."""
    nkv, hd = s["case"]["nkv"], s["case"]["hd"]
    tables = s["tables"].long()
    codes, scale = _values(cache, hd, per)
    x = (codes.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)
    x = x[tables.clamp(min=0)] * (tables >= 0)[..., None, None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    nh, nkv, hd = _sizes(s)
    q, first, most = s["q"], s["first_row"].long(), s["most"]
    k, v = _gathered(s, s["k"], 8), _gathered(s, s["v"], 4)
    seq = s["row_seq"].long()
    at = torch.arange(q.shape[0], device=q.device) - first[seq]
    grid = torch.zeros(k.shape[0], most, nh, hd, device=q.device)        # rows of a sequence side by side, shorter ones padded
    grid[seq, at] = q.float().unflatten(-1, (nh, hd))
    grid = grid.unflatten(2, (nkv, nh // nkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = grid @ k.transpose(-1, -2) * s["scale"]
    pos = s["start"].long()[:, None] + torch.arange(most, device=q.device)
    key = torch.arange(k.shape[2], device=q.device)
    seen = key <= pos[..., None]
    if s["window"]:
        seen &= key > pos[..., None] - s["window"]
    seen = seen[:, None, None].expand(-1, nkv, nh // nkv, -1, -1).flatten(2, 3)
    scores = scores.masked_fill(~seen, -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    out = (scores @ v) / scores.sum(-1, keepdim=True)
    out = out.unflatten(2, (nh // nkv, most)).permute(0, 3, 1, 2, 4).flatten(2, 4)
    return out[seq, at].to(q.dtype)


def _plain_score(s):
    logits, top = s["logits"].float(), s["case"]["top"]
    n, v = logits.shape
    most = logits.amax(-1, keepdim=True)
    shifted = logits - most
    e = shifted.exp()
    total = e.sum(-1, keepdim=True)
    norm = total.log()
    logprob = shifted.gather(1, s["tokens"].long()[:, None]) - norm
    entropy = norm - torch.where(e > 0, e * shifted, 0.0).sum(-1, keepdim=True) / total
    if not top:
        return [logprob[:, 0], entropy[:, 0]]
    # the largest, of equal ones those of the lowest index: one whole number orders them all
    bits = logits.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff)) * (1 << 20) + (v - 1 - torch.arange(v, device=logits.device))
    ids = order.topk(top, dim=-1).indices
    return [logprob[:, 0], entropy[:, 0], shifted.gather(1, ids) - norm, ids.to(torch.int32)]


_OWN = {"write": _own_write, "decode": _own_decode, "prompt": _own_prompt, "score": _own_score}
_PLAIN = {"write": _plain_write, "decode": _plain_attention, "prompt": _plain_attention, "score": _plain_score}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return _exact_write(s)
    if case["kind"] == "score":
        return _exact_score(s)
    return _exact_attention(s)


def _exact_write(s):
    nh, nkv, hd = _sizes(s)
    rot, half = s["case"]["rot"], s["case"]["rot"] // 2
    heads = s["qkv"].to(F64).view(-1, nh + 2 * nkv, hd)
    out = heads.clone()
    if rot:
        angle = s["table"].to(F64)[s["positions"].long()]
        z = torch.complex(heads[:, :nh + nkv, :half].contiguous(), heads[:, :nh + nkv, half:rot].contiguous())
        z = z * torch.complex(angle[..., 0].contiguous(), angle[..., 1].contiguous())[:, None]
        out[:, :nh + nkv, :half], out[:, :nh + nkv, half:rot] = z.real, z.imag
    g = out[:, nh:].reshape(-1, 2 * nkv, hd // GROUP, GROUP)
    size = g.abs().amax(-1, keepdim=True)
    positive = (g == size).any(-1, keepdim=True)
    d = torch.where(positive, -size, size) / 8
    unit = torch.exp2(torch.floor(torch.log2(size.clamp(min=1e-300) / 8)) - 4)          # the fifth bit of the scale
    d = (d / unit).round() * unit
    nearest = torch.where(size < 2.0 ** -117, 0.0, (g / d).round().clamp(-8, 7) * d).view(-1, 2 * nkv, hd)
    return {"q": out[:, :nh].reshape(-1, nh * hd), "k": nearest[:, :nkv].contiguous(), "v": nearest[:, nkv:].contiguous()}


def _exact_score(s):
    top, out = s["case"]["top"], []
    for a in range(0, s["logits"].shape[0], 256):
        x = s["logits"][a:a + 256].to(F64)
        z = torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(x - z)
        entropy = -(p * torch.where(p > 0, x - z, 0.0)).sum(-1)
        row = [torch.gather(x - z, 1, s["tokens"][a:a + 256].long()[:, None])[:, 0], entropy]
        if top:
            value, index = torch.sort(x, dim=-1, descending=True, stable=True)
            row += [value[:, :top] - z, index[:, :top].to(torch.int32)]
        out.append(row)
    return [torch.cat(parts) for parts in zip(*out)]


def _exact_attention(s):
    nh, nkv, hd = _sizes(s)
    groups, each = hd // GROUP, nh // nkv
    out = torch.empty(s["q"].shape[0], nh, hd, dtype=F64, device=s["q"].device)
    firsts, starts = s["first_row"].tolist(), s["start"].tolist()
    channel = torch.arange(hd, device=out.device)
    for i, start in enumerate(starts):
        a, b = firsts[i], firsts[i + 1]
        length = start + b - a
        pages = s["tables"][i, :-(-length // PAGE)].long()
        both = []
        for cache, per in ((s["k"], 8), (s["v"], 4)):
            tile = cache[pages].view(len(pages), nkv, PAGE // TILE, 9 * hd)
            place = (channel % GROUP // per * groups + channel // GROUP) * per + channel % per
            byte = tile[..., :8 * hd].reshape(len(pages), nkv, PAGE, hd // 2)[..., place // 2].int()
            code = (byte >> (4 * (place % 2)).int()) % 16 - 8
            scale = tile[..., 8 * hd:].contiguous().view(torch.bfloat16).reshape(len(pages), nkv, PAGE, groups).to(F64)
            x = code.to(F64) * scale[..., channel // GROUP]
            both.append(x.permute(1, 0, 2, 3).reshape(nkv, len(pages) * PAGE, hd)[:, :length])
        pos = torch.arange(start, length, device=out.device)[:, None]
        key = torch.arange(length, device=out.device)[None]
        hidden = (key > pos) | ((key <= pos - s["window"]) if s["window"] else False)
        q = s["q"][a:b].to(F64).view(b - a, nkv, each, hd)
        for h in range(nkv):
            score = torch.einsum("rec,kc->rek", q[:, h], both[0][h]) * s["scale"]
            p = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), dim=-1)
            out[a:b, h * each:(h + 1) * each] = torch.einsum("rek,kc->rec", p, both[1][h])
    return out.reshape(-1, nh * hd)
