"""The operators of drafted tokens, as cases that can be timed and compared.

A request brings a tree of drafted tokens to a step: row 0 is the token that it was given last, every other row a guess at what follows the
row that is its parent. One step runs all of them; then the part of the tree that the model would have written itself is kept. Three operators:

* ``tree``: softmax attention of a request's rows over its cache. A row sees every key before the tree (the last ``window`` positions of them), and of the
  tree the rows that its bits name: its ancestors and itself. All rows of a tree lie in the cache one behind the other, row i at place start + i, at
  position start + depth.
* ``verify``: which rows are kept, and the token that follows them. The walk begins at row 0. Without ``drafted``, a token is drawn at the row it has
  reached from softmax(logits / temperature), the first one, in the order of the ids, at which the sum of probabilities exceeds the row's second random
  number times the whole (at temperature 0 the largest logit, of equal ones the lowest id); where that is the token of one of the row's children,
  the walk goes on there (of equal tokens at the first), else it ends and that token follows. With ``drafted``, the children's tokens were drawn
  independently from the distribution q that a drafting model's logits give: with r = p at first, a child of token x is taken where its own first random number
  times q(x) sum(r) is below r(x), and where it is not, r becomes max(r - sum(r) q, 0) and the next child is looked at. Behind the last child the token that
  follows is drawn from r (from p where nothing is left of r).
* ``keep``: the keys and values of the kept rows move to the places directly behind the tokens that the cache held before, in every layer.

Sizes are those of the SmolLM2 shapes (9/3, 15/5 and 32/32 heads of 64; 49,152 tokens) and of wider layouts (32/8 heads of 128).
"""
import math
import random

import torch

own = False

PAGE = 16
WORD = 32                   # rows of a tree that a word of bits names
AGREE = 0.75                # how often a row's first child is what the model itself would have written
NOISE = 0.6                 # how far a drafting model's logits are from the model's: it agrees about as often
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
F64 = torch.float64


def listed():
    return [
        # one user's generation behind a short context, a few guesses: the smallest attention call there is
        dict(name="tree_135m_b1", kind="tree", dtype="bfloat16", seqs=1, nodes=8, width=3, past=1023, ragged=False, nh=9, nkv=3, hd=64, window=0),
        # a small service: unequal contexts and trees
        dict(name="tree_360m_b8", kind="tree", dtype="bfloat16", seqs=8, nodes=16, width=3, past=2500, ragged=True, nh=15, nkv=5, hd=64, window=0),
        # a full batch, every head with keys of its own
        dict(name="tree_1.7b_b16", kind="tree", dtype="bfloat16", seqs=16, nodes=32, width=4, past=4095, ragged=False, nh=32, nkv=32, hd=64, window=0),
        # large trees behind long contexts, four queries a key: as much arithmetic as there is memory traffic
        dict(name="tree_wide_b4", kind="tree", dtype="bfloat16", seqs=4, nodes=64, width=4, past=16001, ragged=True, nh=32, nkv=8, hd=128, window=0),
        # one request with a very long context: few rows, a long axis
        dict(name="tree_long_b1", kind="tree", dtype="bfloat16", seqs=1, nodes=26, width=3, past=131071, ragged=False, nh=32, nkv=8, hd=128, window=0),
        # the 32-bit path
        dict(name="tree_fp32_b4", kind="tree", dtype="float32", seqs=4, nodes=24, width=3, past=1500, ragged=True, nh=15, nkv=5, hd=64, window=0),
        # one greedy request: a few rows of logits, latency is all
        dict(name="verify_greedy_1", kind="verify", dtype="float32", seqs=1, nodes=8, width=3, ragged=False, vocab=49152, temperature=0.0, drafted=False, masked=False),
        # a full batch that samples
        dict(name="verify_sampled_64", kind="verify", dtype="float32", seqs=64, nodes=16, width=3, ragged=True, vocab=49152, temperature=0.8, drafted=False, masked=False),
        # bfloat16 logits of a large odd vocabulary, parts of which a grammar rules out; greedy requests beside others
        dict(name="verify_odd_16", kind="verify", dtype="bfloat16", seqs=16, nodes=32, width=4, ragged=True, vocab=100003, temperature=-0.7, drafted=False, masked=True),
        # chains of five tokens that a smaller model has drawn
        dict(name="verify_drafted_32", kind="verify", dtype="float32", seqs=32, nodes=6, width=1, ragged=False, vocab=49152, temperature=1.0, drafted=True, masked=False),
        # a few kept rows of the smallest model
        dict(name="keep_135m_1", kind="keep", dtype="bfloat16", seqs=1, nodes=8, width=3, layers=30, nkv=3, hd=64, past=1003),
        # a full batch of the largest
        dict(name="keep_1.7b_64", kind="keep", dtype="bfloat16", seqs=64, nodes=16, width=3, layers=24, nkv=32, hd=64, past=40),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "verify", "verify", "keep"])
    dtype = "bfloat16" if rng.random() < 0.75 else "float32"
    if kind == "verify":
        drafted, vocab = rng.random() < 0.4, _between(rng, 300, 150000)
        nodes = _between(rng, 1, 9 if drafted else 64)
        seqs = max(1, min(_between(rng, 1, 64), 1024 * 49152 // (vocab * nodes * (2 if drafted else 1))))
        return dict(kind="verify", dtype=dtype, seqs=seqs, nodes=nodes, width=rng.choice([1, 2, 4]), ragged=rng.random() < 0.5, vocab=vocab,
                    temperature=rng.choice([0.0, 0.6, 1.0, -0.9]), drafted=drafted, masked=rng.random() < 0.3)
    nh, nkv = rng.choice([(9, 3), (15, 5), (32, 32), (32, 8), (16, 2), (12, 1), (7, 7)])
    if kind == "keep":
        hd, layers, nodes = rng.choice([48, 64, 80, 128]), rng.randint(1, 32), _between(rng, 2, 64)
        seqs = max(1, min(_between(rng, 1, 64), 64 * 24 * 32 * 64 * 4 // (layers * nkv * hd * (nodes // PAGE + 3) * (2 if dtype == "float32" else 1))))
        return dict(kind="keep", dtype=dtype, seqs=seqs, nodes=nodes, width=rng.choice([1, 2, 4]), layers=layers, nkv=nkv, hd=hd, past=rng.randint(0, 60))
    hd, nodes, seqs = rng.choice([32, 64, 64, 96, 128, 128]), _between(rng, 1, 64), _between(rng, 1, 32)
    most = 16 * 4096 * 32 * 64 // (seqs * nkv * hd * (1 if dtype == "bfloat16" else 8))
    most = min(most, 64 * 4 * 12000 * 32 * 128 // (seqs * nodes * nh * hd * (1 if dtype == "bfloat16" else 30)))
    past = _between(rng, 1, max(2, min(most, 131071)))
    return dict(kind="tree", dtype=dtype, seqs=seqs, nodes=nodes, width=rng.choice([1, 2, 4]), past=past, ragged=rng.random() < 0.7, nh=nh, nkv=nkv, hd=hd,
                window=rng.choice([0, 0, _between(rng, 10, 2000)]))


# ------------------------------------------------------------------------------------------------ shapes of a batch
def _tree(nodes, width):
    """The parent of each row (-1 of the first): at most ``width`` children a row, a parent before its children."""
    rng = random.Random(1000 * nodes + width)
    parents, children = [-1], [0] * nodes
    for i in range(1, nodes):
        last = i - 1 if width == 1 or rng.random() < 0.4 else rng.choice([r for r in range(i) if children[r] < width])
        last = last if children[last] < width else next(r for r in range(i) if children[r] < width)
        children[last] += 1
        parents.append(last)
    return parents


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _counts(case):
    """Rows of each request's tree."""
    nodes = case["nodes"]
    return [max(1, nodes - (nodes // 4) * (i % 3)) if case.get("ragged") else nodes for i in range(case["seqs"])]


def _pasts(case):
    """Tokens in the cache before each request's tree: between half and all of ``past`` where they are unequal."""
    n, past = case["seqs"], case["past"]
    if case["kind"] == "keep":
        return [past + 5 * i % PAGE for i in range(n)]
    return [past - (past // 2) * i // max(n - 1, 1) if case["ragged"] else past for i in range(n)]


def _walks(case):
    """Of each request the rows that are kept (for ``keep``): from row 0 down to a leaf, another child here and there."""
    walks = []
    for i, nodes in enumerate(_counts(case)):
        parents, walk = _tree(nodes, case["width"]), [0]
        while True:
            children = [r for r, p in enumerate(parents) if p == walk[-1]]
            if not children:
                break
            walk.append(children[(i + len(walk)) % len(children)])
        walks.append(walk)
    return walks


def _visits(nodes, width):
    """How many rows a walk reaches, on the average: a row's first child is taken as often as ``AGREE`` says."""
    parents, at, chance, total = _tree(nodes, width), 0, 1.0, 1.0
    while at in parents:
        at = parents.index(at)
        chance *= AGREE
        total += chance
    return total


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "verify":
        rows = sum(_visits(n, case["width"]) for n in _counts(case)) * (2 if case["drafted"] and case["temperature"] else 1)
        return {"bytes": rows * case["vocab"] * size + 20 * sum(_counts(case)) + 16 * case["seqs"], "flops": 4 * rows * case["vocab"]}
    if case["kind"] == "keep":
        moved = sum(sum(r != j for j, r in enumerate(walk)) for walk in _walks(case))
        return {"bytes": 4 * moved * case["layers"] * case["nkv"] * case["hd"] * size + 4 * sum(_counts(case)), "flops": 0}
    nh, nkv, hd, window = case["nh"], case["nkv"], case["hd"], case["window"]
    keys, pairs, n = 0, 0, 0
    for nodes, past in zip(_counts(case), _pasts(case)):
        depth = _depths(_tree(nodes, case["width"]))
        keys += nodes + (min(past, window - 1) if window else past)
        pairs += sum(min(d + 1, window) + max(0, min(past, window - d - 1)) if window else d + 1 + past for d in depth)
        n += nodes
    return {"bytes": keys * nkv * 2 * hd * size + 2 * n * nh * hd * size, "flops": 4 * pairs * nh * hd}


# ------------------------------------------------------------------------------------------------ inputs
def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _trees(case, device):
    """What a step knows of its trees: the first row of each request, parents, depths, and of each row the bits of the rows that it sees."""
    counts = _counts(case)
    words = -(-max(counts) // WORD)
    known = {}
    firsts, parents, depths, bits = [0], [], [], []
    for nodes in counts:
        if nodes not in known:
            tree, sees = _tree(nodes, case["width"]), []
            for i, p in enumerate(tree):
                sees.append((sees[p] if p >= 0 else 0) | 1 << i)
            split = [[s >> WORD * w & 0xffffffff for w in range(words)] for s in sees]
            known[nodes] = tree, _depths(tree), [[w - (1 << 32) if w >> 31 else w for w in row] for row in split]
        tree, depth, row_bits = known[nodes]
        parents += tree
        depths += depth
        bits += row_bits
        firsts.append(firsts[-1] + nodes)
    return _ints(firsts, device), _ints(parents, device), _ints(depths, device), _ints(bits, device)


def _pages(need, g, device):
    """Block tables for requests of ``need`` pages each, in no order, and the number of pages of the pool."""
    pages, width = sum(need) + 3, max(need) + 1
    ids = torch.randperm(pages, generator=g, device=device)[:sum(need)].to(torch.int32)
    tables = torch.full((len(need), width), -1, dtype=torch.int32, device=device)
    tables[torch.arange(width, device=device)[None, :] < torch.tensor(need, device=device)[:, None]] = ids
    return tables, pages


def _first_children(case, device):
    """Of each row its first child (a row of the whole batch; -1: it has none)."""
    first, at = [], 0
    for nodes in _counts(case):
        tree = _tree(nodes, case["width"])
        first += [at + tree.index(i) if i in tree else -1 for i in range(nodes)]
        at += nodes
    return torch.tensor(first, device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    first_row, parents, depths, bits = _trees(case, dev)
    counts, n, most = _counts(case), sum(_counts(case)), max(_counts(case))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    state = dict(case=case, first_row=first_row, parents=parents, most=most, status=status, keep={})
    row_seq = torch.repeat_interleave(torch.arange(len(counts), device=dev), torch.tensor(counts, device=dev))
    if case["kind"] == "verify":
        v = case["vocab"]
        warm = abs(case["temperature"])
        heat = torch.full((case["seqs"],), warm, device=dev)
        if case["temperature"] < 0:                                        # (greedy requests beside others)
            heat[::2] = 0.0
        logits = torch.randn(n, v, generator=g, device=dev) * 2.5
        tokens = torch.randint(0, v, (n,), generator=g, device=dev, dtype=torch.int32)
        if case["masked"]:                                                 # (what a grammar rules out: never a whole row)
            logits.masked_fill_(torch.rand(n, v, generator=g, device=dev) < 0.6, -math.inf)
            logits[:, v // 2] = 0.0
        state.update(temperature=heat, uniform=torch.rand(n, 2, generator=g, device=dev), draft=None)
        row_heat = torch.where(heat > 0, heat, torch.ones_like(heat))[row_seq]
        if case["drafted"]:
            draft = (logits + NOISE * row_heat[:, None] * torch.randn(n, v, generator=g, device=dev)).to(dtype)
            q = torch.softmax(draft[first_row[:-1].long()[row_seq] + parents.clamp(min=0)].float() / row_heat[:, None], dim=-1)
            tokens = torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32)
            state["draft"] = draft
        else:
            # a row's first child has the probability AGREE, or is the largest as often
            child = _first_children(case, dev)
            rows = torch.nonzero(child >= 0)[:, 0]
            token, t = tokens[child[rows]].long(), row_heat[rows]
            logits[rows, token] = -math.inf
            rest = torch.logsumexp(logits[rows] / t[:, None], dim=-1)
            likely = torch.where(torch.rand(len(rows), generator=g, device=dev) < AGREE, logits[rows].amax(-1) + 0.5, torch.zeros_like(t))
            logits[rows, token] = torch.where(heat[row_seq[rows]] > 0, t * (rest + math.log(AGREE / (1 - AGREE))), likely)
        state.update(logits=logits.to(dtype), tokens=tokens)
        return state
    pasts, nkv, hd = _pasts(case), case["nkv"], case["hd"]
    tables, pages = _pages([-(-(c + p) // PAGE) for c, p in zip(counts, pasts)], g, dev)
    start = _ints(pasts, dev)
    state.update(tables=tables, start=start)
    if case["kind"] == "keep":
        walks = _walks(case)
        path = torch.full((n,), -1, dtype=torch.int32, device=dev)
        for a, walk in zip(first_row.tolist(), walks):
            path[a:a + len(walk)] = _ints(walk, dev)
        shape = (case["layers"], pages, nkv, PAGE, hd)
        k, v = (torch.randn(shape, generator=g, device=dev, dtype=dtype) for _ in range(2))
        state.update(k=k, v=v, path=path, accepted=_ints([len(w) for w in walks], dev))
        return state
    spread = torch.exp(torch.randn(nkv, 1, hd, generator=g, device=dev) * 0.5)
    k = (torch.randn(pages, nkv, PAGE, hd, generator=g, device=dev) * spread).to(dtype)
    v = torch.randn(pages, nkv, PAGE, hd, generator=g, device=dev).to(dtype)
    q = torch.randn(n, case["nh"] * hd, generator=g, device=dev).to(dtype)
    state.update(q=q, k=k, v=v, positions=start[row_seq] + depths, visible=bits, reach=max(c + p for c, p in zip(counts, pasts)),
                 scale=1.0 / math.sqrt(hd), window=case["window"] or None)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _OWN[state["case"]["kind"]](state)
    return _PLAIN[state["case"]["kind"]](state)


def _own_tree(s):
    from glassbox_b200 import kernels
    c, q, keep = s["case"], s["q"], s["keep"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    if not keep:                                         # (what a program keeps from call to call)
        keep["parts"] = kernels.tree_attention_parts(q, nh, nkv, hd, c["seqs"], s["most"], s["reach"], s["window"])
    out = torch.empty_like(q)
    kernels.tree_attention(q, out, s["k"], s["v"], s["tables"], s["first_row"], s["start"], s["positions"], s["visible"], s["most"], nh, nkv, hd, PAGE,
                           s["scale"], s["window"], s["reach"], keep["parts"], s["status"])
    return out


def _own_verify(s):
    from glassbox_b200 import kernels
    n, seqs, dev = s["logits"].shape[0], s["case"]["seqs"], s["logits"].device
    path = torch.empty(n, dtype=torch.int32, device=dev)
    accepted, following = (torch.empty(seqs, dtype=torch.int32, device=dev) for _ in range(2))
    kernels.verify_tree(s["logits"], s["tokens"], s["parents"], s["first_row"], s["uniform"], s["temperature"], path, accepted, following, s["draft"])
    return {"path": path, "accepted": accepted, "next": following}


def _own_keep(s):
    from glassbox_b200 import kernels
    kernels.keep_rows(s["k"], s["v"], s["tables"], s["first_row"], s["start"], s["path"], s["accepted"], PAGE, s["most"], s["status"])
    return {"k": s["k"], "v": s["v"]}


def _batch(s):
    """(request, row within it) of every row."""
    first = s["first_row"].long()
    seq = torch.repeat_interleave(torch.arange(len(first) - 1, device=first.device), first.diff())
    return seq, torch.arange(len(seq), device=first.device) - first[seq]


def _named(bits, most):
    """Truth values [rows, most] of words of bits."""
    at = torch.arange(most, device=bits.device)
    return bits.long()[:, at // WORD] >> at % WORD & 1 == 1


def _plain_tree(s):
    c, most = s["case"], s["most"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    seq, at = _batch(s)
    # keys and values of a request side by side, padded; what lies behind its rows is masked
    start, table = s["start"].long(), s["tables"].clamp(min=0).long()
    k, v = (x[table].float().transpose(1, 2).flatten(2, 3) for x in (s["k"], s["v"]))
    q = torch.zeros(len(start), most, nh, hd, device=k.device)
    q[seq, at] = s["q"].float().unflatten(-1, (nh, hd))
    q = q.unflatten(2, (nkv, nh // nkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = q @ k.transpose(-1, -2) * s["scale"]
    key = torch.arange(k.shape[2], device=k.device)
    place = key - start[:, None]                                           # of a key within its request's tree
    named = torch.zeros(len(start), most, most, dtype=torch.bool, device=k.device)
    named[seq, at] = _named(s["visible"], most)
    inside = (place >= 0) & (place < s["first_row"].long().diff()[:, None])
    seen = named.gather(2, place.clamp(0, most - 1)[:, None].expand(-1, most, -1)) & inside[:, None] | (place < 0)[:, None]
    if s["window"]:
        pos = torch.zeros(len(start), most, dtype=torch.long, device=k.device)
        pos[seq, at] = s["positions"].long()
        key_pos = torch.where(place < 0, key[None], pos.gather(1, place.clamp(0, most - 1)))
        seen &= pos[..., None] - key_pos[:, None] < s["window"]
    seen = seen[:, None, None].expand(-1, nkv, nh // nkv, -1, -1).flatten(2, 3)
    scores = scores.masked_fill(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    total = weights.sum(-1, keepdim=True)
    out = (weights @ v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.unflatten(2, (nh // nkv, most)).permute(0, 3, 1, 2, 4).flatten(2, 4)
    return out[seq, at].to(s["q"].dtype)


def _softmax(logits, heat):
    x = logits.to(F64)
    e = torch.exp((x - x.amax(-1, keepdim=True)) / heat.to(F64)[:, None])
    return e / e.sum(-1, keepdim=True)


def _drawn(weights, uniform):
    """The first place at which the sum exceeds the random number times the whole."""
    upto = weights.cumsum(-1)
    return torch.searchsorted(upto, uniform.to(F64)[:, None] * upto[:, -1:], right=True)[:, 0].clamp(max=weights.shape[-1] - 1)


def _plain_verify(s):
    logits, tokens, parents, uniform = s["logits"], s["tokens"].long(), s["parents"].long(), s["uniform"]
    seq, at = _batch(s)
    first, n, dev = s["first_row"].long(), len(seq), logits.device
    above = first[seq] + parents.clamp(min=0)                              # a row's parent, among all rows
    child = parents >= 0
    heat = s["temperature"][seq]
    warm = heat > 0
    safe = torch.where(warm, heat, torch.ones_like(heat))
    # what is drawn at every row, as if the walk came there
    top = logits.float()
    largest = (top == top.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1)
    p = _softmax(logits, safe)
    pick = torch.where(warm, _drawn(p, uniform[:, 1]), largest)
    index = torch.arange(n, device=dev)
    if s["draft"] is None:
        taken = child & (tokens == pick[above])
        twin = taken[:, None] & taken[None] & (above[:, None] == above[None]) & (index[:, None] > index[None])
        taken &= ~twin.any(-1)
    else:
        # the children of every row in their order: taken where the random number says so and no earlier one was; r = max(p - taken_away q, 0)
        q = _softmax(s["draft"], safe)
        sibling = (above[:, None] == above[None]) & child[:, None] & child[None] & (index[:, None] > index[None])
        rank = sibling.sum(-1)
        away, whole = torch.zeros(n, dtype=F64, device=dev), torch.ones(n, dtype=F64, device=dev)
        done, taken = torch.zeros(n, dtype=torch.bool, device=dev), torch.zeros(n, dtype=torch.bool, device=dev)
        for turn in range(int(rank.max()) + 1):
            now = index[child & (rank == turn)]
            up, x = above[now], tokens[now]
            r = (p[up, x] - away[up] * q[up, x]).clamp(min=0)
            fits = uniform[now, 0].to(F64) * q[up, x] * whole[up] < r
            fits = torch.where(warm[up], fits, x == largest[up])
            taken[now] = fits & ~done[up]
            done[up] |= fits
            away[up[~fits]] += whole[up[~fits]]
            whole[up] = (p[up] - away[up, None] * q[up]).clamp(min=0).sum(-1)
        r = (p - away[:, None] * q).clamp(min=0)
        r = torch.where((away > 0)[:, None] & (r.sum(-1, keepdim=True) > 0), r, p)
        pick = torch.where(warm, _drawn(r, uniform[:, 1]), largest)
    # a row is kept where it and all rows above it are taken
    good = taken | ~child & (at == 0)
    seen = torch.eye(n, dtype=torch.bool, device=dev)
    for _ in range(s["most"].bit_length()):                                # (paths of 1, 2, 4 ... steps)
        seen |= seen[above]
        above = above[above]
    kept = ~(seen & ~good[None]).any(-1)
    place = kept.to(torch.int64).cumsum(0) - 1
    accepted = torch.zeros(len(first) - 1, dtype=torch.int64, device=dev).index_add_(0, seq, kept.to(torch.int64))
    before = accepted.cumsum(0) - accepted
    path = torch.full((n,), -1, dtype=torch.int64, device=dev)
    path[(first[seq] + place - before[seq])[kept]] = at[kept]
    last = first[:-1] + path[first[:-1] + accepted - 1]
    return {"path": path.to(torch.int32), "accepted": accepted.to(torch.int32), "next": pick[last].to(torch.int32)}


def _plain_keep(s):
    seq, at = _batch(s)
    path, start, tables = s["path"].long(), s["start"].long(), s["tables"].long()
    moves = at < s["accepted"].long()[seq]
    seq, at, path = seq[moves], at[moves], path[moves]
    source, target = start[seq] + path, start[seq] + at
    for x in (s["k"], s["v"]):
        x[:, tables[seq, target // PAGE], :, target % PAGE] = x[:, tables[seq, source // PAGE], :, source % PAGE].clone()
    return {"k": s["k"], "v": s["v"]}


_OWN = {"tree": _own_tree, "verify": _own_verify, "keep": _own_keep}
_PLAIN = {"tree": _plain_tree, "verify": _plain_verify, "keep": _plain_keep}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["kind"] != "tree":
        return None                                                        # (whole numbers, and numbers that are copied)
    s = prepare(case, seed)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    each, window = nh // nkv, case["window"]
    out = torch.empty(s["q"].shape[0], nh, hd, dtype=F64, device=s["q"].device)
    firsts = s["first_row"].tolist()
    for i, start in enumerate(s["start"].tolist()):
        a, b = firsts[i], firsts[i + 1]
        length = start + b - a
        parents = s["parents"][a:b].tolist()
        pages = s["tables"][i, :-(-length // PAGE)].long()
        k, v = (x[pages].to(F64).permute(1, 0, 2, 3).reshape(nkv, len(pages) * PAGE, hd)[:, :length] for x in (s["k"], s["v"]))
        hidden, depth = torch.zeros(b - a, length, dtype=torch.bool), _depths(parents)
        for r in range(b - a):
            hidden[r, start:] = True
            up = r
            while up >= 0:
                if not window or depth[r] - depth[up] < window:
                    hidden[r, start + up] = False
                up = parents[up]
            if window:
                hidden[r, :max(0, min(start, start + depth[r] - window + 1))] = True
        hidden = hidden.to(out.device)
        q = s["q"][a:b].to(F64).view(b - a, nkv, each, hd)
        for h in range(nkv):
            score = torch.einsum("rec,kc->rek", q[:, h], k[h]) * s["scale"]
            p = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), dim=-1)
            out[a:b, h * each:(h + 1) * each] = torch.einsum("rek,kc->rec", p, v[h])
    return out.reshape(-1, nh * hd)
