"""Cases and plain forms of the operators on a KV cache held in 4 bits (``tiny_infra_b200.kv4``).

The cache: a paged pool [num_blocks, num_kv_heads, 18 * D] uint8 of blocks of 16 tokens.  One
(block, kv head) tile holds, in this order, the K codes [16, D/2], the V codes [16, D/2], the K
scales [D/16, 16] and the V scales [D/16, 16].  A code is 4 bits: sign and e2m1 magnitude
(0, .5, 1, 1.5, 2, 3, 4, 6), two per byte, the lower dim in the low half.  A scale byte b is the
half-precision number with the bits b << 7; it belongs to 16 consecutive dims of one token.

Operators, each by its ``op`` name:
  append    quantise new tokens' K and V into the pool (the result is read back as values)
  decode    one query token per sequence over the sequence's cached tokens, with log-sum-exp
  prefill   chunks of query tokens, causal, over the cached tokens
  weights   add each cached token's attention weight to its running total
  evict     keep the recent tokens and the heaviest older ones, moved to the front
"""
import math

import torch

own = False

BLOCK = 16
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------
def listed():
    small = {"nh": 14, "kvh": 2, "d": 64, "dtype": "bf16"}
    return [
        # one decode step's new tokens of 256 sequences (k and v are slices of the fused qkv rows)
        dict(small, name="append-256", op="append", tokens=256, run=1),
        # a packed prefill of 16384 tokens, wider heads
        dict(name="append-16384-d128", op="append", nh=32, kvh=8, d=128, dtype="fp16",
             tokens=16384, run=4096),
        # the attention op's small configuration: 8 short sequences, latency counts
        dict(small, name="decode-8x512", op="decode", batch=8, lo=1, hi=512),
        # a continuous batch at its ordinary lengths
        dict(small, name="decode-256x2048", op="decode", batch=256, lo=128, hi=2048),
        # long-context serving: bandwidth counts
        dict(small, name="decode-256x32768", op="decode", batch=256, lo=8192, hi=32768),
        # other head layout and type
        dict(name="decode-32x8192-d128", op="decode", nh=32, kvh=8, d=128, dtype="fp16",
             batch=32, lo=1024, hi=8192),
        # three short chunks, one of a single token behind a long prefix
        dict(small, name="prefill-3x130", op="prefill", counts="1,37,130", starts="511,0,100"),
        # chunked prefill of 4096 tokens behind long prefixes
        dict(small, name="prefill-4x1024", op="prefill", counts="1024,1024,1024,1024",
             starts="0,9001,20480,32767"),
        # per decode step, ordinary batch
        dict(small, name="weights-256x2048", op="weights", batch=256, lo=128, hi=2048),
        # per decode step, long contexts
        dict(small, name="weights-32x32768", op="weights", batch=32, lo=8192, hi=32768),
        # one sequence reaches its budget: all 24 layers at once
        dict(small, name="evict-1x2048", op="evict", layers=24, batch=1, lo=2048, hi=2048,
             keep=1024, recent=256),
        # a whole batch of ragged sequences brought down to its budget
        dict(small, name="evict-32x4096", op="evict", layers=24, batch=32, lo=600, hi=4096,
             keep=1000, recent=100),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "weights", "evict"])
    nh, kvh = rng.choice([(14, 2), (32, 8), (8, 8), (8, 1), (28, 4), (12, 2), (16, 1), (9, 3)])
    d = rng.choice([64, 64, 128])
    c = dict(op=op, nh=nh, kvh=kvh, d=d, dtype=rng.choice(["bf16", "fp16"]))
    if op == "append":
        c.update(tokens=_log(rng, 1, 16384), run=rng.choice([1, 7, 100, 4096]))
    elif op in ("decode", "weights"):
        batch = _log(rng, 1, 256)
        top = min(32768, int(3.0e8 / (batch * kvh * d)))     # the work of a long listed case at most
        hi = _log(rng, 1, max(1, top))
        c.update(batch=batch, lo=rng.choice([1, max(1, hi // 4), hi]), hi=hi)
    elif op == "prefill":
        n = rng.randint(1, 6)
        counts = [_log(rng, 1, 700) for _ in range(n)]
        starts = [rng.choice([0, _log(rng, 1, 8000)]) for _ in range(n)]
        c.update(counts=",".join(map(str, counts)), starts=",".join(map(str, starts)))
    else:
        hi = _log(rng, 20, 4096)
        keep = rng.randint(1, hi)
        c.update(layers=rng.choice([1, 2, 24]), batch=_log(rng, 1, 12), lo=rng.choice([1, hi]),
                 hi=hi, keep=keep, recent=rng.randint(0, keep))
        c.update(nh=kvh)
    return c


def _lens(case, gen):
    n = torch.randint(case["lo"], case["hi"] + 1, (case["batch"],), generator=gen)
    return [int(x) for x in n]


def _blocks(n):
    return -(-n // BLOCK)


# ---- the format, in 32 bits ----------------------------------------------------------------------
def _quantize(x):
    """x [..., D] float32 -> (codes uint8 [..., D], scale float32 [..., D/16])."""
    g = x.reshape(*x.shape[:-1], -1, 16)
    a = g.abs().amax(-1)
    a = a / torch.full_like(a, 6.0)          # a division: by a plain 6.0 it may be a product with 1/6
    e = torch.frexp(a)[1] - 1                                 # a in [2^e, 2^(e+1))
    step = ((e.clamp(min=-14) - 3 + 127) << 23).view(torch.float32)     # 2^(e - 3), exactly
    s = (torch.round(a / step) * step).clamp(max=10240.0)     # ties to even, 4 significant bits
    m, t = g.abs(), s.unsqueeze(-1)
    # midpoints between neighbouring magnitudes; a tie goes to the even code
    code = ((m > 0.25 * t).to(torch.uint8) + (m >= 0.75 * t).to(torch.uint8)
            + (m > 1.25 * t).to(torch.uint8) + (m >= 1.75 * t).to(torch.uint8)
            + (m > 2.5 * t).to(torch.uint8) + (m >= 3.5 * t).to(torch.uint8)
            + (m > 5.0 * t).to(torch.uint8))
    code = torch.where(t > 0, code, torch.zeros_like(code))
    code = torch.where((g < 0) & (code > 0), code | 8, code)
    return code.reshape(x.shape), s


def _value(code, scale, dtype=torch.float32):
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=code.device)
    v = table[code.long()].reshape(*scale.shape, 16) * scale.unsqueeze(-1)
    return v.reshape(code.shape).to(dtype)


def _tile(kcode, vcode, ks, vs):
    """Codes [N, 16, D] and scales [N, 16, D/16] of tiles -> bytes [N, 18 D]."""
    pack = lambda c: (c[..., 0::2] | (c[..., 1::2] << 4)).flatten(1)                 # noqa: E731
    byte = lambda s: ((s.to(torch.float16).view(torch.int16).int() >> 7)             # noqa: E731
                      .to(torch.uint8).transpose(1, 2).flatten(1))
    return torch.cat([pack(kcode), pack(vcode), byte(ks), byte(vs)], 1)


def _untile(tiles, d):
    """Bytes [N, 18 D] -> K, V float32 [N, 16, D]."""
    n, h = tiles.shape[0], 8 * d
    half = lambda b: torch.stack([b & 15, b >> 4], -1).reshape(n, BLOCK, d)          # noqa: E731
    scale = lambda b: ((b.int() << 7).to(torch.int16).view(torch.float16).float()    # noqa: E731
                       .reshape(n, d // 16, BLOCK).transpose(1, 2))
    k = _value(half(tiles[:, :h]), scale(tiles[:, 2 * h:2 * h + d]))
    v = _value(half(tiles[:, h:2 * h]), scale(tiles[:, 2 * h + d:]))
    return k, v


def _cached(pool, table, n, d):
    """K, V float32 [KVH, n, D] of the first n tokens of a block table row."""
    nb, kvh = _blocks(n), pool.shape[1]
    k, v = _untile(pool[table[:nb].long()].reshape(nb * kvh, -1), d)
    shape = lambda x: x.reshape(nb, kvh, BLOCK, d).transpose(0, 1).reshape(          # noqa: E731
        kvh, nb * BLOCK, d)[:, :n]
    return shape(k), shape(v)


# ---- inputs ----------------------------------------------------------------------------------------
def _random_pool(shape, d, gen):
    """A pool of quantised keys (some dims much larger than the others, as rotary keys with a
    bias have) and values, its tiles drawn from a bank of 2048."""
    spread = torch.exp(0.7 * torch.randn(d, generator=gen, device="cuda"))
    k = torch.randn(2048, BLOCK, d, generator=gen, device="cuda") * spread
    v = torch.randn(2048, BLOCK, d, generator=gen, device="cuda")
    (kc, ks), (vc, vs) = _quantize(k), _quantize(v)
    bank = _tile(kc, vc, ks, vs)
    flat = torch.empty((math.prod(shape), 18 * d), dtype=torch.uint8, device="cuda")
    for i in range(0, flat.shape[0], 1 << 20):
        part = flat[i:i + (1 << 20)]
        part.copy_(bank[torch.randint(0, 2048, (part.shape[0],), generator=gen, device="cuda")])
    return flat.reshape(*shape, 18 * d)


def _tables(lens, gen, width):
    """Block tables of the sequences over a shuffled pool that could hold all of them at their
    longest; (int32 [B, width], pool blocks)."""
    need = [_blocks(n) for n in lens]
    total = len(lens) * width + 8
    order = torch.randperm(total, generator=gen)
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n].int()
        at += n
    return t.cuda(), total


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    op, nh, kvh, d = case["op"], case["nh"], case["kvh"], case["d"]
    dt = DTYPES[case["dtype"]]
    st = dict(case=case, dt=dt)

    def rnd(*shape):
        return torch.randn(*shape, generator=gpu, device="cuda").to(dt)

    if op == "append":
        t, run = case["tokens"], case["run"]
        runs = [run] * (t // run) + ([t % run] if t % run else [])
        before = [int(x) for x in torch.randint(0, 200, (len(runs),), generator=cpu)]
        lens = [b + r for b, r in zip(before, runs)]
        tables, total = _tables(lens, cpu, _blocks(run + 200))
        st["pool"] = _random_pool((total, kvh), d, gpu)
        # K and V as the fused projection leaves them: slices of [q | k | v] rows
        spread = torch.exp(0.7 * torch.randn(d, generator=gpu, device="cuda"))
        row = rnd(t, (nh + 2 * kvh) * d).view(t, nh + 2 * kvh, d)
        row[:, nh:nh + kvh] = (row[:, nh:nh + kvh].float() * spread).to(dt)
        st["k"], st["v"] = row[:, nh:nh + kvh], row[:, nh + kvh:]
        th = tables.cpu().long()
        pos = [torch.arange(b, n) for b, n in zip(before, lens)]
        slots = torch.cat([th[i][p // BLOCK] * BLOCK + p % BLOCK for i, p in enumerate(pos)])
        st["slots"] = slots.cuda()
        # read back: the blocks that took new tokens, up to each sequence's length
        first = [b // BLOCK for b in before]
        n_out = [_blocks(n) - f for n, f in zip(lens, first)]
        most = _blocks(run + BLOCK - 1)
        src = torch.full((len(runs), most), -1, dtype=torch.int32)
        dst = torch.full_like(src, -1)
        for i, (f, n) in enumerate(zip(first, n_out)):
            src[i, :n] = th[i, f:f + n].int()
            dst[i, :n] = torch.arange(i * most, i * most + n, dtype=torch.int32)
        st["tables"], st["out_tables"] = src.cuda(), dst.cuda()
        st["host_lens"] = [n - BLOCK * f for n, f in zip(lens, first)]
        st["lens"] = torch.tensor(st["host_lens"], dtype=torch.int32, device="cuda")
        st["k_out"] = torch.zeros(len(runs) * most, kvh, BLOCK, d, dtype=dt, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
    elif op in ("decode", "weights"):
        lens = _lens(case, cpu)
        st["tables"], total = _tables(lens, cpu, _blocks(case["hi"]))
        st["pool"] = _random_pool((total, kvh), d, gpu)
        st["host_lens"] = lens
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = rnd(len(lens), nh, d)
        if op == "decode":
            st["out"] = torch.empty_like(st["q"])
            st["lse"] = torch.empty(len(lens), nh, device="cuda")
        else:
            # the log-sum-exp that the step's attention gave
            st["lse"] = torch.stack([_lse(st["q"][i].float(), _cached(
                st["pool"], st["tables"][i], n, d)[0]) for i, n in enumerate(lens)])
            st["weights"] = torch.rand(total, kvh, BLOCK, generator=gpu, device="cuda")
            st["new"] = st["weights"].clone()
    elif op == "prefill":
        counts = [int(x) for x in case["counts"].split(",")]
        starts = [int(x) for x in case["starts"].split(",")]
        lens = [s + n for s, n in zip(starts, counts)]
        st["tables"], total = _tables(lens, cpu, _blocks(max(lens)))
        st["pool"] = _random_pool((total, kvh), d, gpu)
        st["q"] = rnd(sum(counts), nh, d)
        st["out"] = torch.empty_like(st["q"])
        st["counts"], st["starts"], st["host_lens"] = counts, starts, lens
        if own:
            from tiny_infra_b200 import kv4
            st["plan"] = kv4.PrefillPlan(starts, counts, device="cuda")
    else:
        layers, keep = case["layers"], case["keep"]
        lens = _lens(case, cpu)
        new = [min(n, keep) for n in lens]
        # the survivors go to blocks of their own at the front of the pool
        most = _blocks(keep)
        at = len(lens) * most
        tables, total = _tables(lens, cpu, _blocks(case["hi"]))
        tables = torch.where(tables >= 0, tables + at, tables)
        total += at
        dst = torch.full((len(lens), most), -1, dtype=torch.int32)
        for i, n in enumerate(new):
            dst[i, :_blocks(n)] = torch.arange(i * most, i * most + _blocks(n), dtype=torch.int32)
        st["tables"], st["dst"], st["front"] = tables, dst.cuda(), at
        st["pool"] = _random_pool((layers, total, kvh), d, gpu)
        # totals of attention weight: most tokens little, a few much; some exactly zero
        w = torch.rand(layers, total, kvh, BLOCK, generator=gpu, device="cuda")
        st["weights"] = torch.where(w < 0.05, torch.zeros_like(w), w ** 6 * 30.0)
        st["weights"][:, :at] = 0
        st["host_lens"], st["new"] = lens, new
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["kept"] = torch.full((layers, len(lens), kvh, keep), -1, dtype=torch.int32,
                                device="cuda")
        # read back: the survivors of every layer through one table over the flattened pool
        off = torch.arange(layers, dtype=torch.int32, device="cuda").view(-1, 1, 1)
        at_l = torch.where(st["dst"] >= 0, st["dst"] + off * total, st["dst"].expand(layers, -1, -1))
        to_l = torch.where(st["dst"] >= 0, st["dst"] + off * at, st["dst"].expand(layers, -1, -1))
        st["read"] = at_l.reshape(-1, dst.shape[1]).contiguous()
        st["read_to"] = to_l.reshape(-1, dst.shape[1]).contiguous()
        st["read_lens"] = torch.tensor(new * layers, dtype=torch.int32, device="cuda")
        st["k_out"] = torch.zeros(layers * at, kvh, BLOCK, d, dtype=dt, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
    return st


# ---- plain forms -------------------------------------------------------------------------------------
def _lse(q, k):
    """q [NH, D], k [KVH, n, D] -> log-sum-exp of the scaled scores [NH]."""
    return _scores(q, k).logsumexp(-1).flatten()


def _scores(q, k):
    kvh, _, d = k.shape
    return torch.matmul(q.reshape(kvh, -1, d), k.transpose(1, 2)) / math.sqrt(d)


def _read_back(st, k, v, tables, to, lens):
    """Values of the cached tokens, zero behind each sequence's last one."""
    d = st["case"]["d"]
    src, dst = tables.flatten(), to.flatten()
    left = (lens.view(-1, 1) - BLOCK * torch.arange(tables.shape[1], device="cuda")).flatten()
    ok = (dst >= 0) & (left > 0)
    src, dst, left = src[ok].long(), dst[ok].long(), left[ok]
    pool = st["pool"].reshape(-1, st["pool"].shape[-2], 18 * d)
    kvh = pool.shape[1]
    for i in range(0, src.numel(), 65536):
        s = slice(i, i + 65536)
        kk, vv = _untile(pool[src[s]].reshape(-1, 18 * d), d)
        live = (torch.arange(BLOCK, device="cuda") < left[s].view(-1, 1)).view(-1, 1, BLOCK, 1)
        k[dst[s]] = torch.where(live, kk.view(-1, kvh, BLOCK, d), 0.0).to(k.dtype)
        v[dst[s]] = torch.where(live, vv.view(-1, kvh, BLOCK, d), 0.0).to(v.dtype)


def _plain_append(st):
    pool, d = st["pool"], st["case"]["d"]
    kvh, h = pool.shape[1], 8 * d
    blk, off = st["slots"] // BLOCK, st["slots"] % BLOCK
    ar = torch.arange
    for x, code_at, scale_at in ((st["k"], 0, 2 * h), (st["v"], h, 2 * h + d)):
        code, s = _quantize(x.float())
        pack = code[..., 0::2] | (code[..., 1::2] << 4)                    # [T, KVH, D/2]
        byte = (s.to(torch.float16).view(torch.int16).int() >> 7).to(torch.uint8)
        b, hd = blk.view(-1, 1, 1), ar(kvh, device="cuda").view(1, -1, 1)
        o = off.view(-1, 1, 1)
        pool[b, hd, code_at + o * (d // 2) + ar(d // 2, device="cuda")] = pack
        pool[b, hd, scale_at + o + BLOCK * ar(d // 16, device="cuda")] = byte
    _read_back(st, st["k_out"], st["v_out"], st["tables"], st["out_tables"], st["lens"])
    return st["k_out"], st["v_out"]


def _plain_decode(st):
    d = st["case"]["d"]
    for i, n in enumerate(st["host_lens"]):
        k, v = _cached(st["pool"], st["tables"][i], n, d)
        s = _scores(st["q"][i].float(), k)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        tot = p.sum(-1, keepdim=True)
        st["out"][i] = (torch.matmul(p, v) / tot).reshape(-1, d).to(st["dt"])
        st["lse"][i] = (s.amax(-1, keepdim=True) + tot.log()).flatten()
    return st["out"], st["lse"]


def _plain_prefill(st):
    d, kvh = st["case"]["d"], st["case"]["kvh"]
    at = 0
    for i, (start, cnt) in enumerate(zip(st["starts"], st["counts"])):
        n = start + cnt
        k, v = _cached(st["pool"], st["tables"][i], n, d)
        q = st["q"][at:at + cnt].float()
        g = q.shape[1] // kvh
        hide = (torch.arange(n, device="cuda") > torch.arange(start, n, device="cuda").view(-1, 1))
        for h in range(q.shape[1]):
            s = torch.matmul(q[:, h], k[h // g].T) / math.sqrt(d)
            s = s.masked_fill(hide, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            st["out"][at:at + cnt, h] = (torch.matmul(p, v[h // g]) /
                                         p.sum(-1, keepdim=True)).to(st["dt"])
        at += cnt
    return st["out"]


def _plain_weights(st):
    d, kvh = st["case"]["d"], st["case"]["kvh"]
    for i, n in enumerate(st["host_lens"]):
        k, _ = _cached(st["pool"], st["tables"][i], n, d)
        s = _scores(st["q"][i].float(), k)
        p = torch.exp(s - st["lse"][i].view(kvh, -1, 1)).sum(1)            # [KVH, n]
        pos = torch.arange(n, device="cuda")
        b = st["tables"][i][pos // BLOCK].long()
        hd = torch.arange(kvh, device="cuda").view(-1, 1)
        st["new"][b, hd, pos % BLOCK] = st["weights"][b, hd, pos % BLOCK] + p
    return st["new"]


def _plain_evict(st):
    case, pool, w = st["case"], st["pool"], st["weights"]
    layers, kvh, d, keep, recent = (case["layers"], case["kvh"], case["d"], case["keep"],
                                    case["recent"])
    h = 8 * d
    la = torch.arange(layers, device="cuda").view(-1, 1, 1)
    hd = torch.arange(kvh, device="cuda").view(1, -1, 1)
    for i, (n, m) in enumerate(zip(st["host_lens"], st["new"])):
        pos = torch.arange(n, device="cuda")
        if n > keep:
            old = n - recent
            b = st["tables"][i][pos[:old] // BLOCK].long()
            score = w[la, b, hd, pos[:old] % BLOCK]                        # [L, KVH, old]
            top = score.sort(dim=-1, descending=True, stable=True)[1][..., :keep - recent]
            idx = torch.cat([top.sort(-1)[0], pos[old:].expand(layers, kvh, -1)], -1)
        else:
            idx = pos.expand(layers, kvh, -1)
        st["kept"][:, i, :, :m] = idx.int()
        to = torch.arange(m, device="cuda")
        sb, so = st["tables"][i][idx // BLOCK].long(), idx % BLOCK
        db, do = st["dst"][i][to // BLOCK].long().view(1, 1, -1), (to % BLOCK).view(1, 1, -1)
        w[la, db, hd, do] = w[la, sb, hd, so]
        for base in (0, h):
            j = torch.arange(d // 2, device="cuda")
            pool[la[..., None], db[..., None], hd[..., None], base + do[..., None] * (d // 2) + j] = \
                pool[la[..., None], sb[..., None], hd[..., None], base + so[..., None] * (d // 2) + j]
        j = BLOCK * torch.arange(d // 8, device="cuda")
        pool[la[..., None], db[..., None], hd[..., None], 2 * h + do[..., None] + j] = \
            pool[la[..., None], sb[..., None], hd[..., None], 2 * h + so[..., None] + j]
    _read_back(st, st["k_out"], st["v_out"], st["read"], st["read_to"], st["read_lens"])
    return st["kept"], w[:, :st["front"]], st["k_out"], st["v_out"]


# ---- one pass ------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
                "weights": _plain_weights, "evict": _plain_evict}[op](st)
    from tiny_infra_b200 import kv4
    if op == "append":
        kv4.append(st["pool"], st["k"], st["v"], st["slots"])
        kv4.dequantize(st["pool"], st["tables"], st["lens"], st["out_tables"], st["k_out"],
                       st["v_out"])
        return st["k_out"], st["v_out"]
    if op == "decode":
        kv4.decode_attention(st["out"], st["q"], st["pool"], st["tables"], st["lens"],
                             lse=st["lse"])
        return st["out"], st["lse"]
    if op == "prefill":
        kv4.prefill_attention(st["out"], st["q"], st["pool"], st["tables"], st["plan"])
        return st["out"]
    if op == "weights":
        kv4.accumulate_weights(st["weights"], st["q"], st["lse"], st["pool"], st["tables"],
                               st["lens"], out=st["new"])
        return st["new"]
    kv4.evict(st["pool"], st["weights"], st["tables"], st["lens"], st["case"]["keep"],
              st["case"]["recent"], out_block_tables=st["dst"], kept=st["kept"])
    kv4.dequantize(st["pool"], st["read"], st["read_lens"], st["read_to"], st["k_out"],
                   st["v_out"])
    return st["kept"], st["weights"][:, :st["front"]], st["k_out"], st["v_out"]


# ---- work ----------------------------------------------------------------------------------------------
def work(case):
    op, nh, kvh, d = case["op"], case["nh"], case["kvh"], case["d"]
    tok = kvh * d * 9 // 8                       # bytes of a cached token: codes and scales of K and V
    if op == "append":
        t = case["tokens"]
        return {"bytes": t * kvh * d * 4 + t * 8 + 2 * t * tok + t * kvh * d * 4,
                "flops": t * kvh * d * 4}
    if op in ("decode", "weights"):
        n = case["batch"] * (case["lo"] + case["hi"]) // 2
        if op == "decode":
            return {"bytes": n * tok + case["batch"] * nh * (4 * d + 4) + n // 4,
                    "flops": 4 * n * nh * d}
        return {"bytes": n * (tok // 2 + 8 * kvh) + case["batch"] * nh * (2 * d + 4) + n // 4,
                "flops": 2 * n * nh * d}
    if op == "prefill":
        counts = [int(x) for x in case["counts"].split(",")]
        starts = [int(x) for x in case["starts"].split(",")]
        seen = sum(s * n + n * (n + 1) // 2 for s, n in zip(starts, counts))
        return {"bytes": sum(s + n for s, n in zip(starts, counts)) * tok + sum(counts) * nh * d * 4,
                "flops": 4 * seen * nh * d}
    mean = (case["lo"] + case["hi"]) / 2
    kept = min(mean, case["keep"])
    units = case["layers"] * case["batch"]
    return {"bytes": int(units * (mean * kvh * 4 + kept * (2 * tok + 12 * kvh)
                                  + kept * (tok + kvh * d * 4))),
            "flops": int(units * kvh * mean)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _two_to(n):
    """2^n in 64 bits, from its bits (a power function may be off by a rounding)."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _values64(tiles, d):
    """Tiles [N, 18 D] of bytes -> K, V [N, 16, D] in 64 bits, from the bits of codes and scales."""
    t = tiles.long()

    def codes(b):
        c = torch.empty(b.shape[0], b.shape[1] * 2, dtype=torch.long, device=b.device)
        c[:, 0::2], c[:, 1::2] = b % 16, b // 16
        exp, man, sign = (c // 2) % 4, c % 2, 1 - 2 * (c // 8)
        mag = torch.where(exp == 0, 0.5 * man, (1.0 + 0.5 * man) * _two_to(exp - 1))
        return (mag * sign).reshape(-1, BLOCK, d)

    def scales(b):
        exp, man = b // 8, b % 8
        s = torch.where(exp == 0, man * 2.0 ** -17, (8 + man) * _two_to(exp - 18))
        return s.reshape(-1, d // 16, BLOCK).permute(0, 2, 1).repeat_interleave(16, 2)

    n = 8 * d
    return (codes(t[:, :n]) * scales(t[:, 2 * n:2 * n + d]),
            codes(t[:, n:2 * n]) * scales(t[:, 2 * n + d:]))


def _sequence64(st, i, n):
    d = st["case"]["d"]
    ids = st["tables"][i, :_blocks(n)].long()
    kvh = st["pool"].shape[1]
    k, v = _values64(st["pool"][ids].flatten(0, 1), d)
    order = lambda x: x.reshape(-1, kvh, BLOCK, d).permute(1, 0, 2, 3).flatten(1, 2)[:, :n]  # noqa: E731
    return order(k), order(v)


def _nearest64(x):
    """x [..., D] in 64 bits -> the values that the format holds for it."""
    g = x.unflatten(-1, (-1, 16))
    a = g.abs().max(-1, keepdim=True)[0]
    a = torch.div(a, torch.full_like(a, 6))
    e = (a.view(torch.long) >> 52) - 1023                    # the exponent's bits
    e = e.clamp(min=-14)
    s = (torch.round(a * _two_to(3 - e)) * _two_to(e - 3)).clamp(max=10240)
    mags = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    best, err = torch.zeros_like(g), (g.abs() / s).abs()
    for i in (2, 4, 6, 1, 3, 5, 7):              # even codes first: they win a tie
        m = mags[i]
        e2 = (g.abs() / s - m).abs()
        best, err = torch.where(e2 < err, m, best), torch.minimum(err, e2)
    out = torch.where(s > 0, best * s * g.sign(), torch.zeros_like(g))
    return out.flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    op, d, kvh = case["op"], case["d"], case["kvh"]
    if op in ("decode", "weights") and case["batch"] * case["hi"] * kvh * d > 1 << 31:
        return None
    if op == "append":
        outs = []
        b, o = st["slots"] // BLOCK, st["slots"] % BLOCK
        for new, which in ((st["k"], 0), (st["v"], 1)):
            ids = torch.unique(torch.cat([st["tables"].flatten().long().clamp(min=0), b]))
            at = torch.full((st["pool"].shape[0],), -1, dtype=torch.long, device="cuda")
            at[ids] = torch.arange(ids.numel(), device="cuda")
            vals = _values64(st["pool"][ids].flatten(0, 1), d)[which].reshape(-1, kvh, BLOCK, d)
            vals[at[b], :, o] = _nearest64(new.double())
            out = torch.zeros(st["k_out"].shape, dtype=torch.float64, device="cuda")
            for j in range(st["tables"].shape[1]):
                ok = st["out_tables"][:, j] >= 0
                live = (torch.arange(BLOCK, device="cuda") <
                        (st["lens"][ok] - BLOCK * j).view(-1, 1)).view(-1, 1, BLOCK, 1)
                out[st["out_tables"][ok, j].long()] = vals[at[st["tables"][ok, j].long()]] * live
            outs.append(out)
        return tuple(outs)
    if op == "decode":
        outs, lses = [], []
        for i, n in enumerate(st["host_lens"]):
            k, v = _sequence64(st, i, n)
            z = torch.einsum("hgd,hnd->hgn", st["q"][i].double().unflatten(0, (kvh, -1)), k)
            z = z * d ** -0.5
            outs.append(torch.einsum("hgn,hnd->hgd", torch.softmax(z, -1), v).flatten(0, 1))
            lses.append(torch.logsumexp(z, -1).flatten())
        return torch.stack(outs), torch.stack(lses)
    if op == "weights":
        new = st["weights"].double()
        for i, n in enumerate(st["host_lens"]):
            k, _ = _sequence64(st, i, n)
            z = torch.einsum("hgd,hnd->hgn", st["q"][i].double().unflatten(0, (kvh, -1)), k)
            p = (z * d ** -0.5 - st["lse"][i].double().view(kvh, -1, 1)).exp().sum(1)
            p = torch.nn.functional.pad(p, (0, -n % BLOCK)).unflatten(1, (-1, BLOCK))
            new[st["tables"][i, :_blocks(n)].long()] += p.permute(1, 0, 2)
        return new
    if op == "prefill":
        rows = []
        for i, (start, cnt) in enumerate(zip(st["starts"], st["counts"])):
            k, v = _sequence64(st, i, start + cnt)
            q = st["q"][len(rows):len(rows) + cnt].double()
            res = torch.empty_like(q)
            causal = torch.ones(cnt, start + cnt, dtype=torch.bool, device="cuda").tril(start)
            for hq in range(q.shape[1]):
                hk = hq * kvh // q.shape[1]
                z = (q[:, hq] @ k[hk].T) * d ** -0.5
                z = torch.where(causal, z, -torch.inf)
                res[:, hq] = torch.softmax(z, -1) @ v[hk]
            rows.extend(res)
        return torch.stack(rows)
    kept, w_out = st["kept"].clone(), st["weights"].double()[:, :st["front"]].clone()
    k_out = torch.zeros(st["k_out"].shape, dtype=torch.float64, device="cuda")
    v_out = torch.zeros_like(k_out)
    for la in range(case["layers"]):
        for i, (n, m) in enumerate(zip(st["host_lens"], st["new"])):
            ids = st["tables"][i, :_blocks(n)].long()
            w = st["weights"][la, ids].permute(1, 0, 2).flatten(1)[:, :n]          # [KVH, n]
            rank = w.double().clone()
            rank[:, n - case["recent"]:] = torch.inf
            # a heavier token before a lighter one, an earlier before a later one of the same weight
            order = torch.argsort(rank, dim=1, descending=True, stable=True)[:, :m]
            idx = order.sort(1)[0] if n > case["keep"] else torch.arange(n, device="cuda").expand(kvh, -1)
            kept[la, i, :, :m] = idx.int()
            k, v = _values64(st["pool"][la, ids].flatten(0, 1), d)
            to = st["dst"][i, :_blocks(m)].long()
            full = torch.nn.functional.pad(w.double().gather(1, idx), (0, -m % BLOCK))
            live = torch.arange(full.shape[1], device="cuda").view(-1, BLOCK) < m
            cur = w_out[la, to]
            w_out[la, to] = torch.where(live.unsqueeze(1), full.unflatten(1, (-1, BLOCK))
                                        .permute(1, 0, 2), cur)
            for x, out in ((k, k_out), (v, v_out)):
                x = x.reshape(-1, kvh, BLOCK, d).permute(1, 0, 2, 3).flatten(1, 2)
                x = x.gather(1, idx.unsqueeze(-1).expand(-1, -1, d))
                x = torch.nn.functional.pad(x, (0, 0, 0, -m % BLOCK)).unflatten(1, (-1, BLOCK))
                out[la * st["front"] + to] = x.permute(1, 0, 2, 3)
    return kept, w_out, k_out, v_out
