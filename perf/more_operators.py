"""Cases and plain forms of the operators of a decoding step on drafted tokens: each sequence brings a tree
of tokens (node 0 the last one it emitted, the others guesses for what follows), the model runs over
all nodes at once, a token is drawn at every node, and the path that the draws confirm is kept.

Operators, each by its ``op`` name:
  reserve    blocks from the free list, block tables, slots and positions of the new tokens (and, for
             trees, each node's depth and its ancestors as bits)
  attention  every node's attention over its sequence's cached tokens and its own ancestors
  sample     a token per row of logits: temperature, top-k, top-p, min-p, from a given uniform number
  accept     follow the draws down each tree; K and V of the confirmed nodes move to the front

The cache is [layers, blocks, kv heads, 16, D] for K and for V; slot s is token s % 16 of block s // 16.
"""
import math

import torch

own = False

BLOCK = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


# ---- cases -------------------------------------------------------------------------------------
def listed():
    small = {"nh": 14, "kvh": 2, "d": 64, "dtype": "bf16"}
    return [
        # one decode step of a continuous batch: a token each, a sixteenth of the rows need a block
        dict(name="reserve-256x1", op="reserve", batch=256, lo=128, hi=2048, most=1, tree=False,
             spare=1.0),
        # drafted trees of up to 64 nodes behind ordinary contexts, with depths and ancestors
        dict(name="reserve-64x64-tree", op="reserve", batch=64, lo=128, hi=2048, most=64, tree=True,
             spare=1.0),
        # admission: new prompts of up to 16384 tokens, the pool short of what they all need
        dict(name="reserve-64x16384", op="reserve", batch=64, lo=0, hi=0, most=16384, tree=False,
             spare=0.9),
        # a short batch of small trees: latency counts
        dict(small, name="attention-4x8-512", op="attention", batch=4, nodes=8, lo=1, hi=512,
             tree=True, ragged=True),
        # speculative decoding of a batch behind long contexts
        dict(small, name="attention-32x64-8192", op="attention", batch=32, nodes=64, lo=2048, hi=8192,
             tree=True, ragged=False),
        # few sequences, very long contexts, wider heads; a chain of drafts instead of a tree
        dict(name="attention-8x16-32768-d128", op="attention", nh=32, kvh=8, d=128, dtype="fp16",
             batch=8, nodes=16, lo=16384, hi=32768, tree=False, ragged=True),
        # one request with the scheduler's default parameters
        dict(name="sample-1x151936", op="sample", rows=1, vocab=151936, dtype="bf16", kind="default"),
        # a batch whose requests all ask for something else
        dict(name="sample-256x151936-mixed", op="sample", rows=256, vocab=151936, dtype="bf16",
             kind="mixed"),
        # nothing but a temperature, or top-p alone: the whole vocabulary takes part
        dict(name="sample-256x151936-open", op="sample", rows=256, vocab=151936, dtype="fp32",
             kind="open"),
        # every node of 64 trees of 16, a smaller vocabulary
        dict(name="sample-1024x32000", op="sample", rows=1024, vocab=32000, dtype="bf16",
             kind="mixed"),
        # small trees, the cache of a 24-layer model: latency counts
        dict(small, name="accept-8x8", op="accept", layers=24, batch=8, nodes=8),
        # a whole batch of wide trees, more and wider heads
        dict(name="accept-256x64-d128", op="accept", layers=24, kvh=8, d=128, dtype="bf16", nh=32,
             batch=256, nodes=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["reserve", "attention", "attention", "sample", "sample", "accept"])
    if op == "reserve":
        tree = rng.random() < 0.5
        batch = _log(rng, 1, 256)
        hi = rng.choice([0, _log(rng, 1, 8000)])
        most = _log(rng, 1, 128) if tree else _log(rng, 1, max(1, min(16384, 500000 // batch)))
        return dict(op=op, batch=batch, lo=rng.choice([0, hi]), hi=hi, most=most, tree=tree,
                    spare=rng.choice([1.0, 1.0, 0.8]))
    if op == "sample":
        vocab = _log(rng, 100, 200000)
        rows = _log(rng, 1, max(1, min(1024, 38_000_000 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    kind=rng.choice(["default", "mixed", "mixed", "open"]))
    nh, kvh = rng.choice([(14, 2), (32, 8), (8, 8), (8, 1), (28, 4), (12, 2), (16, 1), (9, 3)])
    c = dict(op=op, nh=nh, kvh=kvh, d=rng.choice([64, 64, 128]), dtype=rng.choice(["bf16", "fp16"]))
    if op == "attention":
        batch, nodes = _log(rng, 1, 64), _log(rng, 1, 128)
        # no more products than the long listed case has, and no larger cache
        top = min(32768, int(1.4e8 / (batch * nodes * nh * (c["d"] // 64))), int(3.0e8 / (batch * kvh * c["d"])))
        hi = _log(rng, 1, max(1, top))
        c.update(batch=batch, nodes=nodes, lo=rng.choice([0, max(1, hi // 4), hi]), hi=hi,
                 tree=rng.random() < 0.7, ragged=rng.random() < 0.5)
    else:
        c.update(layers=rng.choice([1, 2, 24]), batch=_log(rng, 1, 128), nodes=_log(rng, 1, 128))
    return c


# ---- inputs ----------------------------------------------------------------------------------------
def _blocks(n):
    return -(-n // BLOCK)


def _randint(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen)


def _spread(gen, lo, hi, n):
    """n numbers from lo to hi, evenly spread and in random order: their sum does not go by the seed."""
    return torch.linspace(lo, hi, n).round().long()[torch.randperm(n, generator=gen)]


def _trees(counts, gen):
    """Parents (index within the tree, -1 for its root) of packed trees: drafts are wide near the root and
    thin out."""
    out = []
    for n in counts.tolist():
        j = torch.arange(1, n)
        up = (torch.rand(max(0, n - 1), generator=gen) ** 2 * torch.clamp(j, max=12)).long()
        out += [torch.full((min(1, n),), -1), torch.clamp(j - 1 - up, min=0)]
    return torch.cat(out).int()


def _place(lens, cols, extra, gen):
    """Block tables of sequences of these lengths over a shuffled pool, and the blocks that are left."""
    need = _blocks(lens.clone())
    order = torch.randperm(int(need.sum()) + extra, generator=gen).int()
    cell = torch.arange(cols) < need.view(-1, 1)
    t = torch.full((len(lens), cols), -1, dtype=torch.int32)
    t[cell] = order[:int(need.sum())]
    return t, order[int(need.sum()):]


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    make = {"reserve": _prepare_reserve, "attention": _prepare_attention, "sample": _prepare_sample,
            "accept": _prepare_accept}[case["op"]]
    make(case, st, cpu, gpu)
    return st


def _prepare_reserve(case, st, cpu, gpu):
    b, most = case["batch"], case["most"]
    lens = _randint(cpu, case["lo"], case["hi"], b)
    counts = _spread(cpu, max(1, most // 4), most, b)
    cols = _blocks(case["hi"] + most)
    need = int((_blocks(lens + counts) - _blocks(lens)).sum())
    tables, left = _place(lens, cols, need + 64, cpu)
    left = left[:max(1, int(need * case["spare"]))] if case["spare"] < 1 else left
    # the free list is a ring that has gone round: its first entry is somewhere in the middle
    size, head = int(tables.max()) + 1 + need + 64, 37 % (need + 64)
    ids = torch.zeros(size, dtype=torch.int32)
    ids[(head + torch.arange(len(left))) % size] = left
    # one buffer for all that a pass changes, so that a pass begins with one copy
    flat = torch.cat([torch.tensor([head, len(left)], dtype=torch.int32), ids, tables.flatten()])
    st["start"] = flat.cuda()
    st["flat"] = st["start"].clone()
    st["ring"] = st["flat"][:2 + size]
    st["tables"] = st["flat"][2 + size:].view(b, cols)
    st["lens"], st["counts"] = lens.int().cuda(), counts.int().cuda()
    # buffers of a fixed size, as a captured step keeps them: places behind the last token get slot -1
    total = int(counts.sum()) + 5
    st["slots"] = torch.zeros(total, dtype=torch.int64, device="cuda")
    st["positions"] = torch.zeros(total, dtype=torch.int32, device="cuda")
    st["cu"] = torch.zeros(b + 1, dtype=torch.int32, device="cuda")
    st["granted"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    st["parents"] = st["masks"] = None
    if case["tree"]:
        st["parents"] = torch.cat([_trees(counts, cpu), torch.zeros(5, dtype=torch.int32)]).cuda()
        st["masks"] = torch.zeros(total, -(-most // 32), dtype=torch.int32, device="cuda")


def _ancestor_bits(parents, counts):
    """Bits of each packed node's ancestors and itself, [T, words] int32, on the host."""
    most = max(1, int(counts.max()))
    rows, at = [], 0
    for n in counts.tolist():
        m = torch.zeros(n, most, dtype=torch.bool)
        for j, p in enumerate(parents[at:at + n].tolist()):
            if p >= 0:
                m[j] = m[p]
            m[j, j] = True
        rows.append(m)
        at += n
    m = torch.nn.functional.pad(torch.cat(rows), (0, -most % 32)).view(at, -1, 32)
    w = (m.long() << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _prepare_attention(case, st, cpu, gpu):
    b, nh, kvh, d, dt = case["batch"], case["nh"], case["kvh"], case["d"], DTYPES[case["dtype"]]
    lens = _randint(cpu, case["lo"], case["hi"], b)
    counts = _spread(cpu, 1 if case["ragged"] else case["nodes"], case["nodes"], b)
    tables, _ = _place(lens + counts, _blocks(case["hi"] + case["nodes"]), 8, cpu)
    blocks, total = int(tables.max()) + 9, int(counts.sum())
    # some dims of the keys are much larger than the others, as rotary keys with a bias have them
    spread = torch.exp(0.7 * torch.randn(d, generator=gpu, device="cuda")).to(dt)
    shape = (blocks, kvh, BLOCK, d)
    st["k"] = torch.randn(shape, generator=gpu, device="cuda", dtype=dt).mul_(spread)
    st["v"] = torch.randn(shape, generator=gpu, device="cuda", dtype=dt)
    # q as the fused projection leaves it: the front of [q | k | v] rows
    rows = torch.randn(total, (nh + 2 * kvh) * d, generator=gpu, device="cuda").to(dt)
    st["q"] = rows[:, :nh * d].view(total, nh, d)
    st["out"] = torch.zeros(total, nh, d, dtype=dt, device="cuda")
    st["lse"] = torch.zeros(total, nh, device="cuda")
    st["tables"], st["lens"] = tables.cuda(), lens.int().cuda()
    cu = torch.zeros(b + 1, dtype=torch.int32)
    cu[1:] = counts.cumsum(0)
    st["cu"] = cu.cuda()
    st["nodes"], st["length"] = int(counts.max()), int((lens + counts).max())
    st["masks"] = _ancestor_bits(_trees(counts, cpu), counts).cuda() if case["tree"] else None


def _prepare_sample(case, st, cpu, gpu):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gpu, device="cuda")
    # logits: some rows are sure of themselves, some are not, a few tokens stand out
    x = x * (0.5 + 2.5 * torch.rand(rows, 1, generator=gpu, device="cuda"))
    top = torch.randint(0, vocab, (rows, 8), generator=gpu, device="cuda")
    x.scatter_add_(1, top, 8 * torch.rand(rows, 8, generator=gpu, device="cuda"))
    st["logits"] = x.to(DTYPES[case["dtype"]])
    pick = torch.randint(0, 6, (rows,), generator=cpu)
    if case["kind"] == "default":
        t, k, p, m = (torch.full((rows,), v) for v in (0.7, 20, 0.9, 0.0))
    elif case["kind"] == "open":
        t = 0.6 + 0.8 * torch.rand(rows, generator=cpu)
        k, m = torch.zeros(rows), torch.zeros(rows)
        p = torch.where(pick < 3, torch.ones(rows), 0.5 + 0.49 * torch.rand(rows, generator=cpu))
    else:
        # greedy; defaults; top-p alone; min-p alone; a wide top-k; all of them
        at = lambda *v: torch.tensor(v)[pick]                                            # noqa: E731
        t = at(0.0, 0.7, 1.0, 1.2, 0.9, 1.0)
        k = at(0.0, 20.0, 0.0, 0.0, 200.0, 50.0)
        p = at(1.0, 0.9, 0.95, 1.0, 1.0, 0.97)
        m = at(0.0, 0.0, 0.0, 0.1, 0.0, 0.02)
    st["t"], st["k"], st["p"], st["m"] = (v.float().cuda() for v in (t, k, p, m))
    st["k"] = st["k"].int()
    st["u"] = torch.rand(rows, generator=cpu).cuda()
    st["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    st["logprobs"] = torch.zeros(rows, device="cuda")


def _prepare_accept(case, st, cpu, gpu):
    b, kvh, d, dt = case["batch"], case["kvh"], case["d"], DTYPES[case["dtype"]]
    lens = _randint(cpu, 100, 1000, b) % BLOCK               # (only the place within a block matters here)
    counts = _spread(cpu, max(1, case["nodes"] // 2), case["nodes"], b)
    cols = _blocks(BLOCK + case["nodes"])
    parents = _trees(counts, cpu)
    total = int(counts.sum())
    # the drafts' K and V sit in blocks of their own; the confirmed ones go to the sequences' blocks,
    # which are the first of the pool
    table = torch.arange(b * cols).view(b, cols)
    src = torch.randperm(b * cols, generator=cpu).view(b, cols) + b * cols
    node = torch.cat([torch.arange(n) for n in counts.tolist()])
    seq = torch.repeat_interleave(torch.arange(b), counts)
    pos = lens[seq] + node
    st["front"] = b * cols
    st["src"] = (src[seq, pos // BLOCK] * BLOCK + pos % BLOCK).cuda()
    st["dst"] = (table[seq, pos // BLOCK] * BLOCK + pos % BLOCK).cuda()
    shape = (case["layers"], 2 * b * cols, kvh, BLOCK, d)
    st["kc"] = torch.randn(shape, generator=gpu, device="cuda", dtype=dt)
    st["vc"] = torch.randn(shape, generator=gpu, device="cuda", dtype=dt)
    st["kc"][:, :st["front"]] = 0
    st["vc"][:, :st["front"]] = 0
    # draws that agree with one of a node's guesses more often than not
    tokens = torch.randint(0, 151936, (total,), generator=cpu).int()
    targets = torch.randint(0, 151936, (total,), generator=cpu).int()
    cu = torch.zeros(b + 1, dtype=torch.int32)
    cu[1:] = counts.cumsum(0)
    child = torch.flip(torch.arange(total), (0,))            # the first child of a node is written last
    up = parents[child].long()
    has = (up >= 0) & (torch.rand(total, generator=cpu) < 0.8)
    targets[cu[seq[child[has]]].long() + up[has]] = tokens[child[has]]
    st["tokens"], st["parents"], st["targets"] = tokens.cuda(), parents.cuda(), targets.cuda()
    st["cu"] = cu.cuda()
    st["deep"] = min(case["nodes"], 32)                      # room for the longest path
    st["nodes"] = case["nodes"]
    st["num"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    st["path"] = torch.zeros(b, st["deep"], dtype=torch.int32, device="cuda")
    st["new"] = torch.zeros(b, st["deep"], dtype=torch.int32, device="cuda")


# ---- plain forms -------------------------------------------------------------------------------------
def _packed(cu, total):
    """Sequence and index within it of each packed token; those behind the last one belong to none."""
    at = torch.arange(total, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], at, right=True)
    live = seq < len(cu) - 1
    seq = torch.where(live, seq, 0)
    return seq, torch.where(live, at - cu[seq], 0).long(), live


def _plain_reserve(st):
    tables, lens, counts = st["tables"], st["lens"].long(), st["counts"].long()
    ring, size = st["ring"][2:], st["ring"].numel() - 2
    head, have = st["ring"][0].long(), st["ring"][1].long()
    col = torch.arange(tables.shape[1], device="cuda")
    last = (lens + counts - 1) // BLOCK
    need = (col >= (lens // BLOCK).view(-1, 1)) & (col <= last.view(-1, 1)) & (tables < 0)
    need &= (counts > 0).view(-1, 1)
    each = need.sum(1)
    served = (each == 0) | (each.cumsum(0) <= have)          # in order, until one does not fit
    take = need & served.view(-1, 1)
    rank = take.flatten().cumsum(0).view_as(need) - 1
    tables.copy_(torch.where(take, ring[(head + rank) % size], tables))
    used = take.sum()
    st["ring"][0] = (head + used) % size
    st["ring"][1] = have - used
    st["granted"].copy_(torch.where(served, counts, 0))
    st["cu"][1:] = counts.cumsum(0)
    seq, node, live = _packed(st["cu"], st["slots"].numel())
    pos = lens[seq] + node
    live_slot = live & served[seq]
    blk = tables[seq, torch.where(live_slot, pos // BLOCK, 0)].long()
    st["slots"].copy_(torch.where(live_slot, blk * BLOCK + pos % BLOCK, -1))
    if st["parents"] is None:
        st["positions"].copy_(torch.where(live, pos, 0))
        return _reserved(st)
    # who is above whom: one step up, squared until no path is longer
    n, words = st["case"]["most"], st["masks"].shape[1]
    up = torch.zeros(len(lens), n, words * 32, device="cuda")
    flat = torch.where(live, (seq * n + node) * words * 32 + node, 0)
    up.view(-1).index_fill_(0, flat, 1.0)
    par = torch.where(live & (node > 0), flat - node + st["parents"].long(), flat)
    up.view(-1).index_fill_(0, par, 1.0)
    for _ in range(max(1, (n - 1).bit_length())):
        up = (torch.matmul(up[:, :, :n], up) > 0).float()
    above = torch.where(live.view(-1, 1), up[seq, node], 0.0)
    st["positions"].copy_(torch.where(live, lens[seq] + above.sum(1).long() - 1, 0))
    w = (above.view(-1, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    st["masks"].copy_(torch.where(w >= 1 << 31, w - (1 << 32), w))
    return _reserved(st)


def _reserved(st):
    out = dict(tables=st["tables"], slots=st["slots"], positions=st["positions"], cu=st["cu"],
               granted=st["granted"], left=st["ring"][:2])
    if st["masks"] is not None:
        out["masks"] = st["masks"]
    return out


def _plain_attention(st):
    case, q = st["case"], st["q"]
    kvh, d, n, length = case["kvh"], case["d"], st["nodes"], st["length"]
    b, g = case["batch"], case["nh"] // case["kvh"]
    seq, node, _ = _packed(st["cu"], q.shape[0])
    cols = _blocks(length)
    ids = st["tables"][:, :cols].long().clamp(min=0)
    gather = lambda x: x[ids].transpose(1, 2).reshape(b, kvh, cols * BLOCK, d)[:, :, :length].float()  # noqa: E731
    k, v = gather(st["k"]), gather(st["v"])
    padded = torch.zeros(b, n, kvh, g, d, device="cuda")
    padded[seq, node] = q.float().view(-1, kvh, g, d)
    s = torch.matmul(padded.permute(0, 2, 1, 3, 4).reshape(b, kvh, n * g, d), k.transpose(2, 3))
    s = (s / math.sqrt(d)).view(b, kvh, n, g, length)
    # the cached tokens, and of the drafts the ancestors (or all up to the token itself)
    key = torch.arange(length, device="cuda") - st["lens"].view(-1, 1)                  # [B, length]
    draft = key[seq].clamp(min=0)                                                       # [T, length]
    if st["masks"] is None:
        seen = draft <= node.view(-1, 1)
    else:
        word = (draft // 32).clamp(max=st["masks"].shape[1] - 1)
        seen = (st["masks"].gather(1, word) >> (draft % 32)) & 1 > 0
    seen &= draft < (st["cu"][1:] - st["cu"][:-1])[seq].view(-1, 1)
    allowed = torch.zeros(b, n, length, dtype=torch.bool, device="cuda")
    allowed[seq, node] = seen | (key[seq] < 0)
    s = torch.where(allowed.view(b, 1, n, 1, length), s, -INF)
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s - m)
    tot = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, kvh, n * g, length), v).view(b, kvh, n, g, d) / tot
    st["out"].copy_(o.permute(0, 2, 1, 3, 4)[seq, node].reshape(-1, kvh * g, d))
    st["lse"].copy_((m + tot.log()).squeeze(-1).permute(0, 2, 1, 3)[seq, node].reshape(-1, kvh * g))
    return st["out"], st["lse"]


def _plain_sample(st):
    """In 64 bits: a draw may fall next to the border of two tokens."""
    rows, vocab = st["logits"].shape
    x, idx = st["logits"].float().sort(dim=1, descending=True, stable=True)
    t, p, m, u = (st[i].double().view(-1, 1) for i in "tpmu")
    greedy = t <= 0
    z = x.double() / torch.where(greedy, 1.0, t)
    w = torch.exp(z - z[:, :1])
    k = st["k"].long().view(-1, 1)
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    kept = (x >= x.gather(1, k - 1)).sum(1, keepdim=True)                # equal values stay together
    place = torch.arange(vocab, device="cuda")
    w = torch.where(place < kept, w, 0.0)
    cum = w.cumsum(1)
    whole = cum[:, -1:]
    nucleus = ((cum <= p * whole) & (place < kept)).sum(1, keepdim=True) + 1
    kept = torch.where(p < 1, torch.minimum(kept, nucleus), kept)
    kept = torch.minimum(kept, (w >= m.clamp(max=1.0)).sum(1, keepdim=True))
    mass = cum.gather(1, kept - 1)
    at = ((cum <= u * mass) & (place < kept)).sum(1, keepdim=True)
    at = torch.where(greedy, 0, torch.minimum(at, kept - 1))
    st["tokens"].copy_(idx.gather(1, at).view(-1))
    logp = torch.log(w.gather(1, at) / mass)
    st["logprobs"].copy_(torch.where(greedy, 0.0, logp).view(-1))
    return st["tokens"], st["logprobs"]


def _plain_accept(st):
    b, deep, n = st["case"]["batch"], st["deep"], st["nodes"]
    cu = st["cu"].long()
    counts = cu[1:] - cu[:-1]
    node = torch.arange(n, device="cuda")
    at = (cu[:-1].view(-1, 1) + node).clamp(max=st["tokens"].numel() - 1)                # [B, n]
    live = node < counts.view(-1, 1)
    parents, tokens, targets = (st[i][at] for i in ("parents", "tokens", "targets"))
    parents = torch.where(live, parents, -2)
    cur = torch.zeros(b, 1, dtype=torch.long, device="cuda")
    on = counts.view(-1, 1) > 0
    st["path"].fill_(-1)
    st["new"].fill_(-1)
    st["num"].zero_()
    for j in range(deep):
        drawn = targets.gather(1, cur)
        st["path"][:, j:j + 1] = torch.where(on, cur, -1)
        st["new"][:, j:j + 1] = torch.where(on, drawn, -1)
        st["num"] += on.view(-1)
        hit = (parents == cur) & (tokens == drawn) & (node > cur)
        on = on & hit.any(1, keepdim=True)
        cur = hit.int().argmax(1, keepdim=True)
    path = st["path"].long()
    keep = path >= 0
    first = cu[:-1].view(-1, 1)
    src = st["src"][(first + path.clamp(min=0))[keep]]
    dst = st["dst"][(first + torch.arange(deep, device="cuda"))[keep]]
    for c in (st["kc"], st["vc"]):
        c[:, dst // BLOCK, :, dst % BLOCK] = c[:, src // BLOCK, :, src % BLOCK]
    return _accepted(st)


def _accepted(st):
    f = st["front"]
    return st["num"], st["path"], st["new"], st["kc"][:, :f], st["vc"][:, :f]


# ---- one pass ------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if op == "reserve":
        st["flat"].copy_(st["start"])                        # every pass begins with the same tables
    if not own:
        return {"reserve": _plain_reserve, "attention": _plain_attention, "sample": _plain_sample,
                "accept": _plain_accept}[op](st)
    if op == "reserve":
        from tiny_infra_b200 import paging
        paging.reserve(st["tables"], st["lens"], st["counts"], st["ring"], st["slots"],
                       st["positions"], st["cu"], granted=st["granted"], parents=st["parents"],
                       masks=st["masks"])
        return _reserved(st)
    if op == "sample":
        from tiny_infra_b200 import sampler
        sampler.sample(st["logits"], st["t"], st["u"], top_ks=st["k"], top_ps=st["p"],
                       min_ps=st["m"], out=st["tokens"], logprobs=st["logprobs"])
        return st["tokens"], st["logprobs"]
    from tiny_infra_b200 import tree
    if op == "attention":
        tree.attention(st["out"], st["q"], st["k"], st["v"], st["tables"], st["lens"], st["cu"],
                       masks=st["masks"], lse=st["lse"])
        return st["out"], st["lse"]
    tree.accept(st["kc"], st["vc"], st["tokens"], st["parents"], st["targets"], st["cu"], st["src"],
                st["num"], st["path"], st["new"], out_slots=st["dst"])
    return _accepted(st)


# ---- work ----------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "reserve":
        mean = (max(1, case["most"] // 4) + case["most"]) / 2
        total = case["batch"] * mean
        mask = total * (4 + -(-case["most"] // 32) * 4) if case["tree"] else 0
        return {"bytes": int(case["batch"] * 24 + total * 12 + total / BLOCK * 12 + mask), "flops": 0}
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * 28, "flops": 2 * n}
    kvh, d = case["kvh"], case["d"]
    if op == "attention":
        b, nh = case["batch"], case["nh"]
        n = (1 + case["nodes"]) / 2 if case["ragged"] else case["nodes"]
        length = (case["lo"] + case["hi"]) / 2 + n
        return {"bytes": int(b * (length * kvh * d * 4 + length / 4 + n * nh * (4 * d + 4))),
                "flops": int(4 * b * n * nh * d * length)}
    # a path of about three nodes a tree, moved in every layer, K and V, read and written
    n = case["batch"] * 0.75 * case["nodes"]
    moved = case["batch"] * min(3, case["nodes"])
    return {"bytes": int(n * 20 + moved * case["layers"] * kvh * d * 8), "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"reserve": _exact_reserve, "attention": _exact_attention, "sample": _exact_sample,
            "accept": _exact_accept}[case["op"]](case, st)


def _exact_reserve(case, st):
    """Token by token, on the host."""
    ring = st["ring"].tolist()
    head, have, ids = ring[0], ring[1], ring[2:]
    tables, lens, counts = st["tables"].tolist(), st["lens"].tolist(), st["counts"].tolist()
    slots, positions, granted, cu, bits = [], [], [], [0], []
    parents = None if st["parents"] is None else st["parents"].tolist()
    words = 0 if parents is None else st["masks"].shape[1]
    stopped = False
    for row, start, n in zip(tables, lens, counts):
        want = [j for j in range(start // BLOCK, (start + n - 1) // BLOCK + 1) if row[j] < 0]
        stopped = stopped or len(want) > have
        ok = not want or not stopped
        for j in want if ok else []:
            row[j] = ids[head]
            head, have = (head + 1) % len(ids), have - 1
        granted.append(n if ok else 0)
        seen, depth = [], []
        for j in range(n):
            at = start + j
            slots.append(row[at // BLOCK] * BLOCK + at % BLOCK if ok else -1)
            if parents is None:
                positions.append(at)
                continue
            p = parents[cu[-1] + j]
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
            depth.append(depth[p] + 1 if p >= 0 else 0)
            positions.append(start + depth[j])
        bits += seen
        cu.append(cu[-1] + n)
    pad = st["slots"].numel() - cu[-1]
    new = lambda v, like: torch.tensor(v, dtype=like.dtype, device="cuda")               # noqa: E731
    out = dict(tables=new(tables, st["tables"]), slots=new(slots + [-1] * pad, st["slots"]),
               positions=new(positions + [0] * pad, st["positions"]), cu=new(cu, st["cu"]),
               granted=new(granted, st["granted"]), left=new([head, have], st["ring"]))
    if parents is not None:
        signed = lambda w: w - (1 << 32) if w >> 31 else w                              # noqa: E731
        out["masks"] = new([[signed(b >> 32 * i & 0xFFFFFFFF) for i in range(words)]
                            for b in bits + [0] * pad], st["masks"])
    return out


def _exact_attention(case, st):
    nh, kvh, d = case["nh"], case["kvh"], case["d"]
    if case["batch"] * case["nodes"] * nh * case["hi"] * d > 1 << 39:
        return None
    outs, lses = [], []
    cu, lens = st["cu"].tolist(), st["lens"].tolist()
    for i, ctx in enumerate(lens):
        n = cu[i + 1] - cu[i]
        ids = st["tables"][i, :_blocks(ctx + n)].long()
        take = lambda c: c[ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :ctx + n].double()  # noqa: E731
        k, v = take(st["k"]), take(st["v"])
        q = st["q"][cu[i]:cu[i + 1]].double().unflatten(1, (kvh, nh // kvh))
        z = torch.einsum("nhgd,hld->hgnl", q, k) * d ** -0.5
        see = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        if st["masks"] is not None:
            w = st["masks"][cu[i]:cu[i + 1]].long().unsqueeze(-1)
            see = (torch.bitwise_right_shift(w, torch.arange(32, device="cuda")) % 2 == 1).flatten(1)[:, :n]
        z[..., ctx:] = z[..., ctx:].masked_fill(~see, -INF)
        outs.append(torch.einsum("hgnl,hld->nhgd", torch.softmax(z, -1), v).flatten(1, 2))
        lses.append(torch.logsumexp(z, -1).permute(2, 0, 1).flatten(1))
    return torch.cat(outs), torch.cat(lses)


def _exact_sample(case, st):
    """Row by row, on the host."""
    import numpy as np
    x = st["logits"].double().cpu().numpy()
    t, k, p, m, u = (st[i].cpu().numpy().astype(np.float64) for i in "tkpmu")
    tokens, logps = [], []
    for r in range(len(x)):
        if t[r] <= 0:
            tokens.append(int(np.argmax(x[r])))
            logps.append(0.0)
            continue
        order = np.argsort(-x[r], kind="stable")
        v = x[r][order]
        if 0 < k[r] < len(v):
            v = v[v >= v[int(k[r]) - 1]]
        w = np.exp((v - v[0]) / t[r])
        c = np.cumsum(w)
        n = len(v)
        if p[r] < 1:
            n = min(n, int(np.searchsorted(c, p[r] * c[-1], side="right")) + 1)
        n = min(n, int((w >= m[r]).sum()))
        j = min(n - 1, int(np.searchsorted(c[:n], u[r] * c[n - 1], side="right")))
        tokens.append(int(order[j]))
        logps.append(float(np.log(w[j]) - np.log(c[n - 1])))
    return (torch.tensor(tokens, dtype=torch.int32, device="cuda"),
            torch.tensor(logps, dtype=torch.float64, device="cuda"))


def _exact_accept(case, st):
    """Node by node, on the host; the moved values are what they were."""
    cu, parents, tokens, targets = (st[i].tolist() for i in ("cu", "parents", "tokens", "targets"))
    src, dst = st["src"].tolist(), st["dst"].tolist()
    num, paths, news, moves = [], [], [], []
    for i in range(case["batch"]):
        a, n = cu[i], cu[i + 1] - cu[i]
        path = [0] if n else []
        while path and len(path) < st["deep"]:
            cur = path[-1]
            nxt = [c for c in range(cur + 1, n) if parents[a + c] == cur and tokens[a + c] == targets[a + cur]]
            if not nxt:
                break
            path.append(nxt[0])
        pad = [-1] * (st["deep"] - len(path))
        num.append(len(path))
        paths.append(path + pad)
        news.append([targets[a + c] for c in path] + pad)
        moves += [(src[a + c], dst[a + j]) for j, c in enumerate(path)]
    s, e = torch.tensor(moves, device="cuda").T
    outs = []
    for c in (st["kc"], st["vc"]):
        out = c[:, :st["front"]].clone()
        out[:, e // BLOCK, :, e % BLOCK] = c[:, s // BLOCK, :, s % BLOCK]
        outs.append(out)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")                    # noqa: E731
    return i32(num), i32(paths), i32(news), outs[0], outs[1]
