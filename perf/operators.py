"""Cases and plain forms of the paged key/value cache operators.

Three operators of ``ttl_moe.KvCache`` are measured:

``append``  K and V rows of new tokens go into a paged cache with their rotary
            position rotation applied on the way, and Q is rotated in the same
            call; a pass then reads the rows back as the cache holds them
            (``read``), so that the cache's contents are among the outputs.
``attend``  attention of the batch's Q rows over the paged cache, the cache
            held in the rows' own type: causal, with a sliding window, sinks, a
            tanh cap, a distance bias, a document mask or a prefix mask.
``attend`` over a cache held in 4 bits (``cache: mxfp4``): E2M1 codes with one
            E8M0 scale per 32 values of a head, the format of the framework's
            expert weights.

``step`` runs a serving step's calls one after another: the append of the new
tokens and the attention over them.  Every pass of every operator begins with
the batch's plan, as a new batch does; a program with many layers makes it once
for all of them.

With ``own`` false, ``run`` computes in elementary torch operations.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _case(name, kind, rows, cache, heads, kv_heads, dim, page, seqs, new, ctx, ragged=False, window=0, sinks=False,
          cap=0.0, slopes=False, docs=False, prefix=False, rope=0, interleaved=False, layout=0):
    c = dict(kind=kind, rows=rows, cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs,
             new=new, ctx=ctx, ragged=ragged, window=window, sinks=sinks, cap=cap, slopes=slopes, docs=docs,
             prefix=prefix, rope=rope, interleaved=interleaved, layout=layout)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the framework's own decode: one token of one sequence, f32 rows, gpt-oss heads; latency counts
        _case("append one f32 token", "append", "f32", "f32", 64, 8, 64, 64, 1, 1, 1040, rope=64),
        # a scheduler's mixed step: chunks of three prompts of unequal length, an odd group of heads
        _case("append ragged bf16 chunks", "append", "bf16", "bf16", 40, 8, 128, 32, 3, 701, 5000, ragged=True,
              rope=128),
        # a long prompt's cache written in 4 bits
        _case("append 16384 rows in 4 bits", "append", "bf16", "mxfp4", 64, 8, 64, 64, 4, 4096, 4096, rope=64),
        # the framework's own decode length, one sequence in f32
        _case("attend f32 token at 1040", "attend", "f32", "f32", 64, 8, 64, 64, 1, 1, 1040, sinks=True),
        # a full serving batch, every sequence at another length
        _case("attend 128 bf16 tokens", "attend", "bf16", "bf16", 64, 8, 64, 64, 128, 1, 8192, ragged=True, sinks=True),
        # a sliding-window layer of a large batch: little cache per token
        _case("attend 256 windowed tokens", "attend", "bf16", "bf16", 64, 8, 64, 64, 256, 1, 4096, ragged=True,
              sinks=True, window=128),
        # one user with a long context: the work has to be split over the keys
        _case("attend one token at 131072", "attend", "bf16", "bf16", 64, 8, 64, 64, 1, 1, 131072, sinks=True),
        # a whole prompt
        _case("attend a 4096 prompt", "attend", "bf16", "bf16", 64, 8, 64, 64, 1, 4096, 4096, sinks=True),
        # chunked prompts over earlier context, capped scores, packed documents, f16 and wider heads
        _case("attend f16 chunks with cap", "attend", "f16", "f16", 32, 8, 128, 16, 6, 509, 6144, ragged=True,
              cap=30.0, docs=True),
        # a serving batch over a 4-bit cache
        _case("attend 64 tokens, 4 bits", "attend", "bf16", "mxfp4", 64, 8, 64, 64, 64, 1, 16384, ragged=True,
              sinks=True),
        # a prompt over a 4-bit cache, part of it a prefix that sees itself whole, with a distance bias
        _case("attend a 1500 prompt, 4 bits", "attend", "bf16", "mxfp4", 32, 4, 64, 64, 2, 1500, 2000, ragged=True,
              prefix=True, slopes=True),
        # a serving step: plan, append and attention
        _case("step of 32 bf16 tokens", "step", "bf16", "bf16", 64, 8, 64, 64, 32, 1, 2048, ragged=True, sinks=True,
              rope=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "step"])
    rows = rng.choice(["bf16", "bf16", "f16", "f32"])
    cache = rng.choice([rows, rows, "mxfp4"])
    heads, kv_heads = rng.choice([(64, 8), (32, 8), (40, 8), (28, 4), (16, 16), (16, 1), (24, 3)])
    dim = rng.choice([64, 64, 128])
    page = rng.choice([16, 32, 64, 128])
    prompt = rng.random() < 0.4
    common = dict(ragged=rng.random() < 0.7, layout=rng.randrange(1 << 20))
    if kind != "attend":
        common.update(rope=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3)
    if kind != "append":
        common.update(window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.5,
                      cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, docs=rng.random() < 0.3,
                      prefix=rng.random() < 0.2)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.3 else _log(rng, 2, 8192 // seqs + 2)
        ctx = new + _log(rng, 1, 4096)
    elif prompt:
        heads, kv_heads = min(heads, 32), min(kv_heads, 8)
        seqs = rng.randrange(1, 5)
        new = _log(rng, 2, 500 if rows == "f32" else 1400)
        ctx = new + _log(rng, 1, 500 if rows == "f32" else 2500)
    else:
        seqs = _log(rng, 1, 96)
        new = rng.choice([1, 1, 1, 2, 3])
        ctx = new + _log(rng, 1, max(2, min(100000, 400000 // seqs)))
    return _case(None, kind, rows, cache, heads, kv_heads, dim, page, seqs, new, ctx, **common)


def _layout(case):
    """New rows and length after them of each sequence: the case's own, the same for every seed."""
    r = random.Random(1000003 * case["layout"] + 31 * case["seqs"] + case["ctx"])
    new, length = [], []
    for s in range(case["seqs"]):
        if not case["ragged"] or s == 0:
            n, l = case["new"], case["ctx"]
        elif s == 3:
            n, l = 0, 0  # a slot of the batch without a sequence
        else:
            n = r.randint(1, case["new"])
            l = r.randint(n, case["ctx"])
        new.append(n)
        length.append(l)
    return new, length


def _masks(case):
    """Lowest visible position of each row and prefix length of each sequence, or None."""
    new, length = _layout(case)
    r = random.Random(77 + case["layout"])
    first = prefix = None
    if case["docs"]:
        first = []
        for n, l in zip(new, length):
            cuts = sorted(r.randrange(l + 1) for _ in range(3)) if l else []
            first += [max([c for c in cuts if c <= p], default=0) for p in range(l - n, l)]
        first[-1 if case["seqs"] < 4 else new[0] - 1] = 1 << 30  # a padding row: it sees nothing
    if case["prefix"]:
        prefix = [r.randint(0, l) for l in length]
    return first, prefix


def _freq(case):
    """Rotation in radians per position of each pair: base 150000, as the framework's attention block."""
    n = case["rope"] // 2
    return 150000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))


# ---- what a program has in hand ----

def _to_mxfp4(x):
    """Codes (one per byte) and scale bytes of x [..., D]: blocks of 32, scale 2^(floor(log2 max) - 2)."""
    x = x.double()
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax)[1].double() - 3  # floor(log2(amax)) - 2
    e = torch.where(amax > 0, e.clamp(-127, 127), torch.full_like(e, -127))
    a = b.abs() * torch.exp2(-e)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))  # spacing of the codes at a
    a = (torch.round(a / step) * step).clamp(max=6)  # round() takes ties to even, as the codes' last bit does
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4))
    code = code + torch.where(torch.signbit(b), 8.0, 0.0)
    return code.to(torch.uint8).reshape(x.shape), (e + 127).to(torch.uint8).squeeze(-1)


def _from_mxfp4(code, scale):
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float32, device=code.device)
    mag = table[(code & 7).long()]
    v = torch.where(code >= 8, -mag, mag).reshape(*code.shape[:-1], -1, 32)
    return (v * torch.exp2(scale.float() - 127)[..., None]).reshape(code.shape)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, dev = TYPES[case["rows"]], "cuda"
    H, KV, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    new, length = _layout(case)
    S, rows = case["seqs"], sum(new)
    per = max(1, max(-(-l // page) for l in length))
    used = sum(-(-l // page) for l in length)
    pages = used + 3

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    # one projection's output, of which Q, K and V are views
    qkv = rand(rows, (H + 2 * KV) * D)
    q = qkv[:, :H * D].unflatten(1, (H, D))
    k = qkv[:, H * D:(H + KV) * D].unflatten(1, (KV, D))
    v = qkv[:, (H + KV) * D:].unflatten(1, (KV, D))
    table = torch.zeros(S, per, dtype=torch.int32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))[:used].to(torch.int32)
    at = 0
    for s, l in enumerate(length):
        n = -(-l // page)
        table[s, :n] = order[at:at + n]
        at += n
    start = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    first, prefix = _masks(case)
    st = dict(case=case, q=q, k=k, v=v, table=table.to(dev), start=start.to(dev),
              length=torch.tensor(length, dtype=torch.int32, device=dev), new=new, lengths=length, pages=pages,
              first=None if first is None else torch.tensor(first, dtype=torch.int32, device=dev),
              prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=dev),
              sinks=torch.randn(H, generator=g, device=dev) if case["sinks"] else None,
              slopes=torch.exp2(-8.0 * (torch.arange(H, device=dev) + 1) / H) if case["slopes"] else None,
              freq=_freq(case), scale=1.0 / math.sqrt(D))
    # what the cache holds of earlier tokens (attend: of all of them), each at its page and slot
    kind = case["kind"]
    total = sum(length)
    hist_k = rand(total, KV, D) if kind != "append" else None
    hist_v = rand(total, KV, D) if kind != "append" else None
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(length))
    off = torch.tensor([0] + length).cumsum(0)
    pos = torch.arange(total) - off[seq]
    slot = (table[seq, pos // page].long() * page + pos % page).to(dev)
    rseq = torch.repeat_interleave(torch.arange(S), torch.tensor(new))
    rpos = torch.arange(rows) - start[rseq].long() + torch.tensor(length)[rseq] - torch.tensor(new)[rseq]
    st["row_slot"] = (table[rseq, rpos // page].long() * page + rpos % page).to(dev)
    st["row_pos"], st["row_seq"] = rpos.to(dev), rseq.to(dev)
    if case["cache"] == "mxfp4":
        pool = {n: (torch.zeros(pages * page, KV, D, dtype=torch.uint8, device=dev),
                    torch.zeros(pages * page, KV, D // 32, dtype=torch.uint8, device=dev)) for n in "kv"}
        if hist_k is not None:
            for n, x in (("k", hist_k), ("v", hist_v)):
                code, scale = _to_mxfp4(x)
                pool[n][0][slot], pool[n][1][slot] = code, scale
            hist_k, hist_v = (_from_mxfp4(pool[n][0][slot], pool[n][1][slot]).to(dt) for n in "kv")
    else:
        pool = {n: torch.zeros(pages * page, KV, D, dtype=dt, device=dev) for n in "kv"}
        if hist_k is not None:
            pool["k"][slot], pool["v"][slot] = hist_k, hist_v
    st["pool"] = pool
    st["hist"] = (hist_k, hist_v)  # exact() reads these
    if own:
        _open(st, hist_k, hist_v)
    return st


def _open(st, hist_k, hist_v):
    """The framework's cache with the same contents, and the outputs."""
    import sys
    if "tt-lab_b200/python" not in sys.path:
        sys.path.insert(0, "tt-lab_b200/python")
    import ttl_moe
    case = st["case"]
    new, length = st["new"], st["lengths"]
    make = dict(layers=1, pages=st["pages"], page_tokens=case["page"], q_heads=case["heads"],
                kv_heads=case["kv_heads"], head_dim=case["dim"], rows=case["rows"], cache=case["cache"],
                max_seqs=case["seqs"], max_rows=max(sum(length), 1), window=case["window"],
                stream=torch.cuda.current_stream())
    st["cache"] = cache = ttl_moe.KvCache(rope_freq=st["freq"].numpy() if case["rope"] else None,
                                          rope_interleaved=case["interleaved"], **make)
    if hist_k is not None:
        # the earlier tokens, unrotated: their rows are what the cache holds
        off = torch.tensor([0] + length).cumsum(0).to(torch.int32).cuda()
        cache.batch_async(off, st["length"], st["table"], rows=sum(length), max_new=max(length))
        cache.append_async(0, hist_k, hist_v, rotate=False)
    st["out"] = torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda")
    st["q_out"] = torch.empty_like(st["out"])
    st["k_out"] = torch.empty(st["k"].shape, dtype=st["k"].dtype, device="cuda")
    st["v_out"] = torch.empty_like(st["k_out"])


def _plan(st):
    st["cache"].batch_async(st["start"], st["length"], st["table"], rows=sum(st["new"]), max_new=max(st["new"]),
                            first=st["first"], prefix=st["prefix"])


# ---- one pass ----

def run(st):
    kind = st["case"]["kind"]
    if own:
        c = st["cache"]
        _plan(st)  # a new batch's rows, lengths, masks and pages are part of every pass, as in the plain form
        if kind == "append":
            c.append_async(0, st["k"], st["v"], q=st["q"], q_out=st["q_out"])
            c.read_async(0, st["k_out"], st["v_out"])
            return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"]}
        q = st["q"]
        if kind == "step":
            c.append_async(0, st["k"], st["v"], q=st["q"], q_out=st["q_out"])
            q = st["q_out"]
        c.attend_async(0, q, st["out"], sinks=st["sinks"], slopes=st["slopes"], cap=st["case"]["cap"],
                       sliding=st["case"]["window"] > 0)
        return {"out": st["out"]}
    if kind == "append":
        q = _plain_append(st)
        k, v = (_plain_read(st, st["row_slot"], n).to(st["k"].dtype) for n in "kv")
        return {"q": q, "k": k, "v": v}
    q = _plain_append(st) if kind == "step" else st["q"]
    return {"out": _plain_attend(st, q)}


def _plain_rotate(st, x, keep64):
    """x [rows, heads, D] rotated by its rows' positions; the angles in 64 bits."""
    n = st["case"]["rope"] // 2
    if n == 0:
        return x.double() if keep64 else x.float()
    angle = st["row_pos"].double()[:, None] * st["freq"].to(x.device)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    y = x.double() if keep64 else x.float()
    if not keep64:
        cos, sin = cos.float(), sin.float()
    if st["case"]["interleaved"]:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :n], y[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, y[..., 2 * n:]], -1)


def _plain_append(st):
    """K and V into the pool, K rotated; returns Q rotated."""
    four = st["case"]["cache"] == "mxfp4"
    k = _plain_rotate(st, st["k"], four)  # in 64 bits before 4-bit rounding: a value next to a border
    pool, slot = st["pool"], st["row_slot"]
    if four:
        for n, x in (("k", k), ("v", st["v"])):
            pool[n][0][slot], pool[n][1][slot] = _to_mxfp4(x)
    else:
        pool["k"][slot] = k.to(st["k"].dtype)
        pool["v"][slot] = st["v"]
    return _plain_rotate(st, st["q"], False).to(st["q"].dtype)


def _plain_read(st, slot, n):
    p = st["pool"][n]
    return _from_mxfp4(p[0][slot], p[1][slot]) if st["case"]["cache"] == "mxfp4" else p[slot].float()


def _plain_attend(st, q):
    """The batch padded to its longest sequence, the scores whole in 32 bits."""
    case = st["case"]
    S, N, L, page = case["seqs"], max(st["new"]), max(st["lengths"]), case["page"]
    H, KV, D, dev = case["heads"], case["kv_heads"], case["dim"], q.device
    G = H // KV
    seq, pos = st["row_seq"], st["row_pos"]
    col = pos - (st["length"].long() - st["start"].long().diff())[seq]
    j = torch.arange(L, device=dev)
    slot = st["table"].long()[:, j // page] * page + j % page  # [S, L]
    inside = j < st["length"][:, None]
    k = torch.where(inside[..., None, None], _plain_read(st, slot, "k"), 0.0)
    v = torch.where(inside[..., None, None], _plain_read(st, slot, "v"), 0.0)
    x = torch.zeros(S, N, H, D, device=dev)
    x[seq, col] = q.float() * st["scale"]
    x = x.unflatten(2, (KV, G)).permute(0, 2, 3, 1, 4).reshape(S, KV, G * N, D)
    s = torch.matmul(x, k.permute(0, 2, 3, 1)).reshape(S, KV, G, N, L)
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    # lowest visible position and the one after the highest, of each row
    p = torch.zeros(S, N, dtype=torch.long, device=dev)
    lo, hi = torch.zeros_like(p), torch.zeros_like(p)
    p[seq, col] = pos
    hi[seq, col] = torch.maximum(pos + 1, st["prefix"].long()[seq]) if st["prefix"] is not None else pos + 1
    if st["first"] is not None:
        lo[seq, col] = st["first"].long()
    if case["window"]:
        lo = torch.maximum(lo, p - case["window"] + 1)
    if case["slopes"]:
        s = s - st["slopes"].reshape(1, KV, G, 1, 1) * (j - p[..., None]).abs()[:, None, None]
    see = ((j >= lo[..., None]) & (j < hi[..., None]))[:, None, None]
    s = s.masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].reshape(1, KV, G, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul(w.reshape(S, KV, G * N, L), v.permute(0, 2, 1, 3)).reshape(S, KV, G, N, D)
    o = torch.where(see.any(-1, keepdim=True), o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, N, H, D)
    return o[seq, col].to(q.dtype)


# ---- what a pass cannot do without ----

def work(case):
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    new, length = _layout(case)
    rows, size = sum(new), SIZE[case["rows"]]
    cached = KV * (D * size if case["cache"] != "mxfp4" else D // 2 + D // 32)  # K or V of a token
    out = {"bytes": 0.0, "flops": 0.0}
    if case["kind"] != "attend":
        read = case["kind"] == "append"
        out["bytes"] += rows * ((2 * H + 2 * KV) * D * size + 2 * cached + (2 * cached + 2 * KV * D * size if read else 0))
        out["flops"] += 3.0 * rows * (H + KV) * case["rope"]
    if case["kind"] != "append":
        first, prefix = _masks(case)
        at = pairs = keys = 0
        for s, (n, l) in enumerate(zip(new, length)):
            low, high = l, 0
            for i in range(n):
                p = l - n + i
                lo = first[at + i] if first else 0
                lo = max(lo, p - case["window"] + 1, 0) if case["window"] else lo
                hi = max(p + 1, prefix[s]) if prefix else p + 1
                if lo < hi:
                    pairs += hi - lo
                    low, high = min(low, lo), max(high, hi)
            at += n
            keys += max(0, high - low)
        out["bytes"] += 2.0 * rows * H * D * size + 2.0 * keys * cached
        out["flops"] += 4.0 * pairs * H * D
    return out


# ---- the definition in 64 bits ----

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    new, length = st["new"], st["lengths"]
    H, KV, D, n = case["heads"], case["kv_heads"], case["dim"], case["rope"] // 2

    def turned(x):
        """Each pair of a head as a complex number times exp(i angle)."""
        y = x.double().clone()
        if n:
            z = torch.polar(torch.ones(len(x), n, dtype=torch.float64, device=x.device),
                            st["row_pos"].double()[:, None] * st["freq"].to(x.device))[:, None]
            a = slice(0, 2 * n, 2) if case["interleaved"] else slice(0, n)
            b = slice(1, 2 * n, 2) if case["interleaved"] else slice(n, 2 * n)
            z = z * torch.complex(y[..., a].clone(), y[..., b].clone())
            y[..., a], y[..., b] = z.real, z.imag
        return y

    def held(x):
        """x as the cache holds it."""
        if case["cache"] != "mxfp4":
            return x.to(TYPES[case["rows"]]).double()
        b = x.reshape(*x.shape[:-1], D // 32, 32)
        amax = b.abs().amax(-1, keepdim=True)
        unit = torch.exp2((torch.floor(torch.log2(amax)) - 2).clamp(-127, 127))
        unit = torch.where(amax > 0, unit, 1.0)
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        low = torch.bucketize((b / unit).abs().clamp(max=6), table, right=True).clamp(1, 7) - 1
        a, c = table[low], table[low + 1]
        m = (b / unit).abs().clamp(max=6)
        up = (m - a > c - m) | ((m - a == c - m) & (low % 2 == 1))  # ties go to the even code
        return (torch.where(up, c, a) * unit * torch.sign(b)).reshape(x.shape)

    k = turned(st["k"])
    if case["kind"] == "append":
        four = case["cache"] == "mxfp4"
        return {"q": turned(st["q"]), "k": held(k) if four else k, "v": held(st["v"].double())}
    q = st["q"].double()
    if case["kind"] == "step":
        q = turned(st["q"])
    kept_k, kept_v = (x.double() for x in st["hist"])
    out = torch.zeros(len(q), H, D, dtype=torch.float64, device=q.device)
    row = tok = 0
    for s, (m, l) in enumerate(zip(new, length)):
        K, V = kept_k[tok:tok + l].clone(), kept_v[tok:tok + l].clone()
        if case["kind"] == "step" and m:
            K[l - m:], V[l - m:] = held(k[row:row + m]), held(st["v"][row:row + m].double())
        for i in range(0, m, 512):
            p = torch.arange(l - m + i, l - m + min(m, i + 512), device=q.device)[:, None]
            Q = q[row + i:row + i + len(p)]
            j = torch.arange(l, device=q.device)
            see = j <= p if st["prefix"] is None else (j <= p) | (j < st["prefix"][s])
            if st["first"] is not None:
                see = see & (j >= st["first"][row + i:row + i + len(p), None])
            if case["window"]:
                see = see & (j > p - case["window"])
            for h in range(H):
                z = Q[:, h] @ K[:, h * KV // H].T / math.sqrt(D)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if case["slopes"]:
                    z = z - st["slopes"][h].double() * (p - j).abs()
                z = torch.where(see, z, -math.inf)
                if st["sinks"] is not None:
                    z = torch.cat([z, st["sinks"][h].double().expand(len(p), 1)], 1)
                z = torch.softmax(z, 1)[:, :l]
                z = torch.where(see, z, 0.0)
                out[row + i:row + i + len(p), h] = z @ V[:, h * KV // H]
        row, tok = row + m, tok + l
    return {"out": out}
