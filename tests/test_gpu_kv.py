"""The paged key/value cache on the GPU (ttl_kv_*) against plain 64-bit forms
(kv_plain): append with rotation, read, and attention over a cache in the rows'
type or in 4 bits, over the shapes and masks where they can go wrong.
Tolerances are the ones kv_plain derives."""
import math

import numpy as np
import pytest
import torch

import kv_plain
from kv_plain import TYPES, unit

pytestmark = pytest.mark.gpu

COMBOS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "mxfp4"), ("f16", "mxfp4"), ("bf16", "mxfp4")]


class Setup:
    """A cache, a batch over randomly placed pages, and the rows of whole
    sequences: of sequence s the last new[s] are this batch's."""

    def __init__(self, rows="bf16", cache=None, H=8, KV=2, D=64, page=16, new=(1,), length=(5,), seed=0, window=0,
                 freq=None, rope_scale=1.0, interleaved=False, pad=0, extra_pages=2, first=None, prefix=None,
                 stream=None, scale_values=1.0, max_new=None, layers=1, layer=0):
        import ttl_moe
        self.rows_type, self.cache_type = rows, cache or rows
        self.H, self.KV, self.D, self.page = H, KV, D, page
        self.new, self.length = list(new), list(length)
        self.freq, self.rope_scale, self.interleaved, self.window = freq, rope_scale, interleaved, window
        self.layer = layer
        g = torch.Generator().manual_seed(seed)
        self.dt = TYPES[rows]
        S, total, n = len(new), sum(length), sum(new)
        self.rows = n + pad
        per = max(1, max(-(-l // page) for l in length))
        used = sum(-(-l // page) for l in length)
        pages = used + extra_pages
        order = torch.randperm(pages, generator=g)[:used].to(torch.int32)
        self.table = torch.full((S, per), -1, dtype=torch.int32)  # unused entries are never read
        at = 0
        for s, l in enumerate(length):
            m = -(-l // page)
            self.table[s, :m] = order[at:at + m]
            at += m
        self.start = torch.tensor([0] + self.new).cumsum(0).to(torch.int32)
        self.first, self.prefix = first, prefix

        def rand(*shape):
            return (torch.randn(*shape, generator=g) * scale_values).to(self.dt)

        self.k, self.v = rand(total, KV, D), rand(total, KV, D)   # every token, sequence by sequence
        self.q = rand(self.rows, H, D)
        self.tok0 = [0] + list(np.cumsum(length))
        self.cache = ttl_moe.KvCache(layers=layers, pages=pages, page_tokens=page, q_heads=H, kv_heads=KV, head_dim=D,
                                     rows=rows, cache=self.cache_type, max_seqs=S, max_rows=max(total, self.rows, 1),
                                     window=window, rope_freq=freq, rope_scale=rope_scale, rope_interleaved=interleaved,
                                     device=0, stream=stream or torch.cuda.current_stream())
        self.dev = {n: getattr(self, n).cuda() for n in ("table", "start", "k", "v", "q")}
        self.dev["length"] = torch.tensor(self.length, dtype=torch.int32).cuda()
        self.dev["first"] = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
        self.dev["prefix"] = None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda()
        self.max_new = max(self.new) if max_new is None else max_new

    def fill(self, rotate=False):
        """Puts every token of every sequence in the cache."""
        off = torch.tensor(self.tok0, dtype=torch.int32).cuda()
        self.cache.batch_async(off, self.dev["length"], self.dev["table"], rows=sum(self.length))
        self.cache.append_async(self.layer, self.dev["k"], self.dev["v"], rotate=rotate)
        torch.cuda.synchronize()
        return self

    def plan(self):
        d = self.dev
        self.cache.batch_async(d["start"], d["length"], d["table"], rows=self.rows, max_new=self.max_new, first=d["first"],
                               prefix=d["prefix"])
        return self

    def attend(self, fill=7.0, **kw):
        out = torch.full_like(self.dev["q"], fill)
        self.cache.attend_async(self.layer, self.dev["q"], out, **kw)
        self.cache.sync()
        return out.cpu()

    def reference(self, sliding=False, k=None, v=None, **kw):
        outs, tols = [], []
        k = kv_plain.held(self.k.double(), self.cache_type) if k is None else k
        v = kv_plain.held(self.v.double(), self.cache_type) if v is None else v
        at = 0
        for s, (n, l) in enumerate(zip(self.new, self.length)):
            a, b = self.tok0[s], self.tok0[s] + l
            o, t = kv_plain.attend(self.q[at:at + n].double(), k[a:b], v[a:b], torch.arange(l - n, l), self.rows_type,
                                   self.cache_type, window=self.window if sliding else 0,
                                   first=None if self.first is None else torch.tensor(self.first[at:at + n]),
                                   prefix=0 if self.prefix is None else min(self.prefix[s], l), **kw)
            outs.append(o)
            tols.append(t)
            at += n
        return torch.cat(outs), torch.cat(tols)

    def check(self, sliding=False, **kw):
        self.fill().plan()
        dev = {n: (x.cuda() if isinstance(x, torch.Tensor) else x) for n, x in kw.items()}
        out = self.attend(sliding=sliding, **dev)
        ref, tol = self.reference(sliding=sliding, **kw)
        n = sum(self.new)
        off = (out[:n].double() - ref).abs()
        assert (off <= tol).all(), (float((off / tol).max()), float(off.max()))
        assert (out[n:] == 7.0).all()  # rows behind the last sequence
        return out


# ---- append and read ----

def append_and_read(s, **kw):
    n = sum(s.new)
    rows = [torch.full((s.rows, h, s.D), 3.0, dtype=s.dt, device="cuda") for h in (s.H, s.KV, s.KV)]
    idx = torch.cat([torch.arange(a + l - m, a + l) for a, l, m in zip(s.tok0, s.length, s.new)])
    k = torch.full((s.rows, s.KV, s.D), 9.0, dtype=s.dt)
    v = k.clone()
    k[:n], v[:n] = s.k[idx], s.v[idx]
    s.plan()
    s.cache.append_async(s.layer, k.cuda(), v.cuda(), q=s.dev["q"], q_out=rows[0], **kw)
    s.cache.read_async(s.layer, rows[1], rows[2])
    s.cache.sync()
    pos = torch.cat([torch.arange(l - m, l) for l, m in zip(s.length, s.new)])
    for r in rows:
        assert (r[n:] == 3.0).all()
    return [r[:n].cpu() for r in rows], s.q[:n].double(), k[:n].double(), v[:n].double(), pos


def check_rotated(got, x, pos, s, exact_turns=2.0 ** -23):
    """Rotation: cosine and sine to 2 steps of f32 each (the angle cut to its
    fraction in 64 bits), two products and a sum: 4 steps of |x cos| + |y sin|
    <= |x| + |y|; then one rounding to the rows' type."""
    ref = kv_plain.rotate(x, pos, s.freq if s.freq is not None else [], s.rope_scale, s.interleaved)
    n = 0 if s.freq is None else len(s.freq)
    pair = torch.zeros_like(x)
    if n:
        a = slice(0, 2 * n, 2) if s.interleaved else slice(0, n)
        b = slice(1, 2 * n, 2) if s.interleaved else slice(n, 2 * n)
        pair[..., a] = pair[..., b] = x[..., a].abs() + x[..., b].abs()
    tol = unit(s.rows_type) * ref.abs() * (1 + 1e-6) + 6 * exact_turns * abs(s.rope_scale) * pair
    off = (got.double() - ref).abs()
    assert (off <= tol).all(), float((off - tol).max())
    return ref


@pytest.mark.parametrize("rows,cache", COMBOS)
@pytest.mark.parametrize("D,pairs,interleaved", [(64, 32, False), (64, 32, True), (128, 64, False), (128, 32, True), (64, 8, False), (128, 24, False)])
def test_append_rotates_and_stores(rows, cache, D, pairs, interleaved):
    freq = 150000.0 ** (-np.arange(pairs) / pairs)
    s = Setup(rows, cache, H=6, KV=2, D=D, page=16, new=(1, 7, 0, 33), length=(40, 7, 0, 50), freq=freq,
              rope_scale=1.25, interleaved=interleaved, pad=3)
    (q, k, v), q0, k0, v0, pos = append_and_read(s)
    check_rotated(q, q0, pos, s)
    if cache != "mxfp4":
        check_rotated(k, k0, pos, s)
        assert torch.equal(v.double(), v0)
    else:
        turned = kv_plain.rotate(k0, pos, freq, 1.25, interleaved)
        assert torch.equal(k.double(), kv_plain.mxfp4(turned).to(s.dt).double())
        assert torch.equal(v.double(), kv_plain.mxfp4(v0).to(s.dt).double())


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_far_positions(page):
    """Positions past 2^20: the angle has lost 20 bits of an f32's fraction."""
    L = 1_100_003
    freq = 10000.0 ** (-np.arange(32) / 32)
    import ttl_moe
    n = 19
    need = -(-L // page)
    table = torch.zeros(1, need, dtype=torch.int32)
    table[0, -3:] = torch.tensor([4, 2, 1])
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(n, h, 64, generator=g) for h in (4, 1, 1)]
    with ttl_moe.KvCache(pages=5, page_tokens=page, q_heads=4, kv_heads=1, rows="f32", max_rows=n, rope_freq=freq,
                         device=0, stream=torch.cuda.current_stream()) as c:
        c.batch_async(torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([L], dtype=torch.int32).cuda(),
                      table.cuda(), rows=n)
        q, k, v = (t.cuda() for t in x)
        out = [torch.empty_like(t) for t in (q, k, v)]
        c.append_async(0, k, v, q=q, q_out=out[0])
        c.read_async(0, out[1], out[2])
        c.sync()
    pos = torch.arange(L - n, L)
    for got, was in zip(out[:2], x[:2]):
        ref = kv_plain.rotate(was.double(), pos, freq)
        assert (got.cpu().double() - ref).abs().max() <= 8 * 2.0 ** -23 * 2 * was.abs().max()
    assert torch.equal(out[2].cpu(), x[2])


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
def test_append_in_place_views_of_one_projection_and_no_rotation(rows):
    freq = 1000.0 ** (-np.arange(32) / 32)
    H, KV, D, n = 5, 1, 64, 21
    s = Setup(rows, H=H, KV=KV, D=D, new=(n,), length=(n + 9,), freq=freq)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(n, (H + 2 * KV) * D, generator=g).to(s.dt).cuda()
    before = qkv.cpu().double()
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, KV * D, KV * D], 1))
    s.plan()
    s.cache.append_async(0, k, v, q=q, q_out=q)   # in place
    k2, v2 = torch.empty(n, KV, D, dtype=s.dt, device="cuda"), torch.empty(n, KV, D, dtype=s.dt, device="cuda")
    s.cache.read_async(0, k2, v2)
    s.cache.sync()
    pos = torch.arange(9, n + 9)
    check_rotated(q.cpu(), before[:, :H * D].unflatten(1, (H, D)), pos, s)
    check_rotated(k2.cpu(), before[:, H * D:(H + 1) * D].unflatten(1, (KV, D)), pos, s)
    assert torch.equal(qkv[:, H * D:].cpu().double(), before[:, H * D:])  # K and V as they were
    s.cache.append_async(0, k, v, rotate=False)
    s.cache.read_async(0, k2, v2)
    s.cache.sync()
    assert torch.equal(k2, k) and torch.equal(v2, v)


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
def test_append_4_bits_at_borders_and_extremes(rows):
    """Ties between codes, saturation, zero blocks, the type's largest and
    smallest values, infinities and NaN (their block of 32 becomes NaN)."""
    n, D = 12, 64
    s = Setup(rows, "mxfp4", H=2, KV=1, D=D, new=(n,), length=(n,))
    fi = torch.finfo(s.dt)
    v = torch.zeros(n, 1, D, dtype=s.dt)
    v[0, 0, :12] = torch.tensor([4, 0.25, -0.25, 0.75, 1.25, 1.75, 2.5, -2.5, 3.5, 5, 7, -7])
    v[1] = fi.max
    v[2, 0, :3] = torch.tensor([fi.tiny, -fi.tiny, fi.smallest_normal * 0.5])
    v[3, 0, 5], v[3, 0, 40] = math.inf, 1.0
    v[4, 0, 50], v[4, 0, 3] = math.nan, 1.5
    v[5, 0, ::2] = -math.inf
    v[6] = torch.linspace(-6, 6, D)
    v[7, 0, 1] = -0.0
    v[8] = torch.linspace(-1, 1, D) * 2.0 ** -10
    v[9] = 6
    v[10, 0, 0], v[10, 0, 1] = fi.max, fi.tiny
    k = v.flip(0).contiguous()
    s.plan()
    s.cache.append_async(0, k.cuda(), v.cuda())
    k2, v2 = torch.empty_like(k).cuda(), torch.empty_like(v).cuda()
    s.cache.read_async(0, k2, v2)
    s.cache.sync()
    for got, x in ((k2, k), (v2, v)):
        want = kv_plain.mxfp4(x.double()).to(s.dt)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu().nan_to_num(0.0), want.nan_to_num(0.0))


def test_append_leaves_other_slots_alone():
    s = Setup("bf16", new=(3, 2), length=(20, 31)).fill()
    total = sum(s.length)
    s.dev["q"] = s.dev["q"][:5]
    (q, k, v), *_ = append_and_read(s)
    off = torch.tensor(s.tok0, dtype=torch.int32).cuda()
    s.cache.batch_async(off, s.dev["length"], s.dev["table"], rows=total)
    k2, v2 = torch.empty_like(s.dev["k"]), torch.empty_like(s.dev["v"])
    s.cache.read_async(0, k2, v2)
    s.cache.sync()
    assert torch.equal(k2, s.dev["k"]) and torch.equal(v2, s.dev["v"])  # the same rows were written again


# ---- attention ----

@pytest.mark.parametrize("rows,cache", COMBOS)
@pytest.mark.parametrize("H,KV,D,page", [(8, 8, 64, 16), (8, 1, 64, 64), (7, 1, 128, 32), (10, 2, 64, 128), (48, 2, 128, 16)])
def test_attend_tokens(rows, cache, H, KV, D, page):
    """One token per sequence (and a slot without one), lengths from one on."""
    Setup(rows, cache, H, KV, D, page, new=(1, 1, 0, 1, 1, 1), length=(1, 2, 0, 64, 129, 333), pad=2).check()


@pytest.mark.parametrize("rows,cache", COMBOS)
@pytest.mark.parametrize("H,KV,D,page,new,length", [
    (8, 2, 64, 16, (3, 2, 5), (3, 70, 200)),            # a few rows
    (8, 1, 64, 64, (40, 1, 0, 17), (40, 300, 0, 145)),  # chunks and a token
    (6, 2, 128, 32, (150,), (150,)),                    # a prompt
    (5, 1, 64, 128, (70, 33), (200, 33)),               # a group that divides no tile
    (64, 1, 64, 16, (5,), (77,)),                       # one KV head of 64 query heads
    (4, 4, 128, 16, (300, 2), (301, 260)),
])
def test_attend_rows(rows, cache, H, KV, D, page, new, length):
    Setup(rows, cache, H, KV, D, page, new=new, length=length, pad=1).check()


MASKS = [
    dict(window=20, sliding=True),
    dict(window=1, sliding=True),
    dict(sinks=True),
    dict(sinks=True, window=70, sliding=True),
    dict(cap=5.0),
    dict(cap=30.0, slopes=True, sinks=True),
    dict(slopes=True),
    dict(docs=True),
    dict(docs=True, window=50, sliding=True, sinks=True),
    dict(prefix=True),
    dict(prefix=True, docs=True, slopes=True),
    dict(scale=0.37),
    dict(scale=-0.1),
]


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "mxfp4")])
@pytest.mark.parametrize("new,length", [((1, 1, 1), (1, 100, 260)), ((2, 90, 1), (50, 130, 200)), ((200,), (290,))])
@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "-".join(m))
def test_attend_masks(rows, cache, new, length, mask):
    m = dict(mask)
    r = np.random.default_rng(5)
    first = prefix = None
    if m.pop("docs", False):
        first = []
        for n, l in zip(new, length):
            cuts = [0] + sorted(int(c) for c in r.integers(0, l, 2))
            first += [max(c for c in cuts if c <= p) for p in range(l - n, l)]
        first[-1] = 1 << 30                   # a row that sees nothing
        first[0] = -5                         # below the first position: sees everything
        if len(first) > 40:
            first[30:34] = [10 ** 6] * 4
    if m.pop("prefix", False):
        prefix = [int(r.integers(0, l + 40)) for l in length]
    H = 8
    g = torch.Generator().manual_seed(9)
    if m.pop("sinks", False):
        m["sinks"] = torch.randn(H, generator=g) * 2
    if m.pop("slopes", False):
        m["slopes"] = torch.rand(H, generator=g) * 0.1
    s = Setup(rows, cache, H, 2, 64, 16, new=new, length=length, window=m.pop("window", 0), first=first, prefix=prefix)
    out = s.check(**m)
    if first is not None and (prefix is None):
        assert (out[sum(new) - 1] == 0).all()


@pytest.mark.parametrize("rows,cache,D", [("f16", "f16", 64), ("f16", "f16", 128), ("bf16", "bf16", 128), ("bf16", "mxfp4", 64),
                                         ("bf16", "mxfp4", 128)])
@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "-".join(m))
def test_attend_masks_of_prompts(rows, cache, D, mask):
    """Prompts over earlier tokens in every type; biases that rise or fall with
    the distance, before, across and behind the rows' own keys."""
    m = dict(mask)
    new, length, H = (90, 2, 33), (330, 200, 200), 8
    r = np.random.default_rng(6)
    first = prefix = None
    if m.pop("docs", False):
        first = []
        for n, l in zip(new, length):
            cuts = [0] + sorted(int(c) for c in r.integers(0, l, 2))
            first += [max(c for c in cuts if c <= p) for p in range(l - n, l)]
        first[7] = first[100] = 1 << 30       # rows that see nothing
    if m.pop("prefix", False):
        prefix = [320, 0, 190]
    if m.pop("sinks", False):
        m["sinks"] = torch.linspace(-2, 3, H)
    if m.pop("slopes", False):
        m["slopes"] = torch.linspace(-0.05, 1.2, H)
    Setup(rows, cache, H, 2, D, 32, new=new, length=length, window=m.pop("window", 0), first=first, prefix=prefix,
          pad=0 if first else 3).check(**m)


@pytest.mark.parametrize("rows,cache,D", [("bf16", "bf16", 64), ("f16", "f16", 128), ("bf16", "mxfp4", 64)])
def test_tokens_of_many_sequences_beside_a_prompt(rows, cache, D):
    """Enough cache behind single tokens that they stay with their own kernel,
    and a prompt in the same batch."""
    new, length = (1,) * 20 + (90,) + (3,) * 20, (2600,) * 20 + (500,) + (2500,) * 20
    Setup(rows, cache, 4, 2, D, 64, new=new, length=length, seed=3).check(sinks=torch.linspace(-1, 1, 4))


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4"), ("f16", "mxfp4")])
@pytest.mark.parametrize("new", [1, 70])
def test_caps_far_from_the_scores(rows, cache, new):
    """A cap far above the scores changes nothing, one far below leaves the
    signs."""
    s = Setup(rows, cache, 8, 2, 64, 16, new=(new,), length=(new + 60,))
    s.fill().plan()
    ref, tol = s.reference()
    for cap in (1e5, 1e12, 1e30):
        assert ((s.attend(cap=cap).double() - ref).abs() <= tol).all()
    s.check(cap=1e-3)


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4"), ("f16", "mxfp4")])
@pytest.mark.parametrize("kw", [{}, dict(scale=-0.2), dict(cap=9.0), dict(slopes=0.1)], ids=lambda k: "-".join(k) or "plain")
def test_a_seen_nan_key_wherever_it_lies(rows, cache, kw):
    """A row that sees a key of NaN is NaN whole, at any place of the key in
    its tile; the rows before it are as without it."""
    n, extra = 70, 16
    kw = {k: torch.full((4,), v) if k == "slopes" else v for k, v in kw.items()}
    s = Setup(rows, cache, 4, 1, 64, 16, new=(n,) * extra, length=(n + 64,) * extra)
    for i in range(extra):
        s.dev["k"][s.tok0[i] + 70 + i] = math.nan
    s.fill().plan()
    out = s.attend(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}).reshape(extra, n, 4, 64)
    ref, tol = (x.reshape(extra, n, 4, 64) for x in s.reference(**kw))
    for i in range(extra):
        sees = 70 + i - 64  # the first of the sequence's rows that does
        assert torch.isnan(out[i, sees:]).all()
        assert ((out[i, :sees].double() - ref[i, :sees]).abs() <= tol[i, :sees]).all()


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("bf16", "mxfp4")])
def test_the_longest_sequence(rows, cache):
    """One token at the last position there is: every page is page 0, so the
    result is the attention over its 128 keys, each as often as the others.
    Where 2^29 weights are summed one after the other, a part's sums lose up to
    2^-23 per step of 16 keys, the part being at most 2^29 / 148 keys of which a
    warp takes a quarter."""
    n = 2 ** 29 - 128
    s = Setup(rows, cache, 4, 1, 64, 128, new=(1,), length=(128,), extra_pages=0)
    s.fill()
    ref, tol = s.reference()
    table = torch.zeros(1, 2 ** 22, dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 1], dtype=torch.int32).cuda()
    out = torch.full_like(s.dev["q"], 7.0)
    s.cache.batch_async(start, torch.tensor([n], dtype=torch.int32).cuda(), table, rows=1)
    s.cache.attend_async(0, s.dev["q"], out)
    s.cache.sync()
    k, v = (kv_plain.held(x.double(), cache) for x in (s.k, s.v))
    most = float(v.abs().max())
    steps = 2 ** 29 / 148 / 4 / 16
    assert ((out.cpu().double() - ref).abs() <= tol + 2 * steps * 2.0 ** -23 * most).all()
    s.cache.batch_async(start, torch.tensor([n + 1], dtype=torch.int32).cuda(), table, rows=1)
    out.fill_(7.0)
    s.cache.attend_async(0, s.dev["q"], out)
    with pytest.raises(Exception, match="length"):
        s.cache.sync()
    assert (out == 7).all()


def test_pieces_of_more_than_two_seconds():
    """A prompt of 40 rows of 256 heads behind 2^29 keys of 64 KV heads: a CTA's part
    of one head takes longer than the two seconds after which a wait gives up, and the
    next head's tile waits for its end.  (What 2^29 weights sum to in 32 bits is
    another matter: the values are one, so the result is at most a part's lost
    fraction from it.)"""
    import ttl_moe
    H, KV, n, new = 256, 64, 2 ** 29 - 128, 40
    with ttl_moe.KvCache(pages=1, page_tokens=128, q_heads=H, kv_heads=KV, max_rows=128, device=0,
                         stream=torch.cuda.current_stream()) as c:
        one = torch.ones(128, H, 64, dtype=torch.bfloat16, device="cuda")
        i32 = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        c.batch_async(i32(0, 128), i32(128), i32(0)[None], rows=128)
        c.append_async(0, one[:, :KV].contiguous(), one[:, :KV].contiguous())
        table = torch.zeros(1, 2 ** 22, dtype=torch.int32, device="cuda")
        c.batch_async(i32(0, new), i32(n), table, rows=new)
        out = torch.full((new, H, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        c.attend_async(0, one[:new], out)
        c.sync()
        assert (out != 7).all() and torch.isfinite(out).all()


def test_more_work_than_a_plan_counts_is_refused():
    """257 sequences of the greatest length are 2^31 granules of keys."""
    import ttl_moe
    S, n = 257, 2 ** 29 - 128
    with ttl_moe.KvCache(pages=1, page_tokens=128, q_heads=1, kv_heads=1, rows="f32", max_seqs=S, max_rows=S, device=0,
                         stream=torch.cuda.current_stream()) as c:
        table = torch.zeros(S, 2 ** 22, dtype=torch.int32, device="cuda")
        c.batch_async(torch.arange(S + 1, dtype=torch.int32).cuda(), torch.full((S,), n, dtype=torch.int32).cuda(), table, rows=S)
        q = torch.zeros(S, 1, 64, device="cuda")
        out = torch.full_like(q, 7.0)
        c.attend_async(0, q, out)
        with pytest.raises(Exception, match="range"):
            c.sync()
        assert (out == 7).all()


@pytest.mark.parametrize("rows,cache", COMBOS)
def test_attend_long_sequence_is_split_and_merged(rows, cache):
    """One token over 20011 keys: the work is cut into many parts; the same
    bits on every call."""
    s = Setup(rows, cache, 8, 2, 64, 64, new=(1, 2), length=(20011, 4097), seed=4)
    a = s.check(sinks=torch.linspace(-1, 1, 8))
    for _ in range(3):
        assert torch.equal(a, s.attend(sinks=torch.linspace(-1, 1, 8).cuda()))


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4")])
@pytest.mark.parametrize("new", [1, 3, 60])
def test_unseen_infinities_and_nan_do_not_reach_a_row(rows, cache, new):
    """Infinities and NaN in K and V at positions outside a row's window,
    before its document, after it, and in stale slots of its last page."""
    L = 150
    first = [100 if i % 2 else 90 for i in range(new)]
    s = Setup(rows, cache, 8, 2, 64, 16, new=(new,), length=(L,), first=first, window=30)
    poisoned = [5, 89, 3, 88]
    clean_k, clean_v = s.k.clone(), s.v.clone()
    for i, p in enumerate(poisoned):
        s.dev["k"][p] = [math.inf, math.nan, -math.inf, math.nan][i]
        s.dev["v"][p] = [math.nan, math.inf, -math.inf, math.nan][i]
    # stale slots: the sequence was longer once
    import copy
    longer = copy.copy(s)
    longer.fill()
    tail = torch.full((10, 2, 64), math.nan, dtype=s.dt, device="cuda")
    s.cache.batch_async(torch.tensor([0, 10], dtype=torch.int32).cuda(), torch.tensor([160], dtype=torch.int32).cuda(),
                        s.dev["table"], rows=10)
    s.cache.append_async(0, tail, tail)
    s.plan()
    for sliding in (False, True):
        out = s.attend(sliding=sliding)
        s.k, s.v = clean_k, clean_v
        ref, tol = s.reference(sliding=sliding)
        assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("rows,cache", COMBOS)
@pytest.mark.parametrize("D,new,length", [(64, (1,), (9000,)), (128, (3, 2), (5003, 700)), (64, (60,), (6000,)), (128, (40, 1), (4100, 300))])
def test_infinities_and_nan_in_work_that_is_cut(rows, cache, D, new, length):
    """Sequences that several CTAs share: a NaN key that no row sees, an infinite
    value that every other row sees, and NaN behind the end of the last page.  The
    rows that see the value have it in its place (4 bits: in its block of 32), and
    nothing else has."""
    H, KV, at = 8, 2, length[0] // 2
    first = [(at + 1 if i % 2 else at - 300) if i < new[0] else 0 for i in range(sum(new))]
    s = Setup(rows, cache, H, KV, D, 16, new=new, length=length, first=first, seed=5)
    s.v[at] = 0
    s.dev["v"] = s.v.cuda()
    ref, tol = s.reference()
    s.dev["k"][100] = math.nan
    s.dev["v"][at, :, 5] = math.inf
    s.dev["v"][50] = math.nan
    s.fill()
    tail = -length[0] % 16
    if tail:  # the last page's stale slots
        nan = torch.full((tail, KV, D), math.nan, dtype=s.dt, device="cuda")
        s.cache.batch_async(torch.tensor([0, tail], dtype=torch.int32).cuda(),
                            torch.tensor([length[0] + tail], dtype=torch.int32).cuda(), s.dev["table"][:1].contiguous(), rows=tail)
        s.cache.append_async(0, nan, nan)
    s.plan()
    for _ in range(2):
        out = s.attend()
        sees = torch.tensor([i < new[0] and i % 2 == 0 for i in range(sum(new))])
        place = torch.zeros(D, dtype=torch.bool)
        place[0:32 if cache == "mxfp4" else 6] = True
        place[0:0 if cache == "mxfp4" else 5] = False
        good = ~(sees[:, None, None] & place).expand_as(out)
        assert ((out.double() - ref).abs() <= tol)[good].all()
        assert (~torch.isfinite(out))[~good].all()


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4"), ("f16", "mxfp4")])
@pytest.mark.parametrize("where", ["unseen", "seen"])
def test_a_nan_in_a_long_prompt_stays_small(rows, cache, where):
    """320 columns over 65536 keys, every one of which has to be computed again,
    beside a short sequence: the call ends in time (one column after the other by
    one warp takes seconds, and a wait then gave the others up), the short
    sequence is right, and the long one is where it does not see the NaN."""
    n, new = 65536, 40
    s = Setup(rows, cache, 8, 1, 64, 64, new=(new, 3), length=(n, 90), first=[1000] * new + [0] * 3, seed=6)
    s.dev["v"][999 if where == "unseen" else 1000, 0, 40] = math.nan
    s.fill().plan()
    s.attend()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    out = torch.full_like(s.dev["q"], 7.0)
    begin.record()
    s.cache.attend_async(0, s.dev["q"], out)
    end.record()
    s.cache.sync()
    assert begin.elapsed_time(end) < 100.0
    out = out.cpu()
    ref, tol = s.reference()
    bad = slice(32, 64) if cache == "mxfp4" else slice(40, 41)
    if where == "seen":
        assert torch.isnan(out[:new, :, bad]).all()
        out[:new, :, bad] = ref[:new, :, bad].to(out.dtype)
    assert ((out.double() - ref).abs() <= tol).all()


def fastest(s, n=5, **kw):
    """Milliseconds of an attend, the least of a few, and its result."""
    out, best = torch.full_like(s.dev["q"], 7.0), math.inf
    for _ in range(n):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        s.cache.attend_async(0, s.dev["q"], out, **kw)
        b.record()
        s.cache.sync()
        best = min(best, a.elapsed_time(b))
    return best, out.cpu()


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4"), ("f16", "mxfp4")])
@pytest.mark.parametrize("D,page,new,length", [(64, 64, (1,) * 40, 2100), (128, 32, (1, 2) * 16, 1500), (64, 128, (300, 200), 1700),
                                              (128, 16, (90, 200), 1801), (64, 16, (130, 3), 129)])
def test_stale_slots_cost_nothing(rows, cache, D, page, new, length):
    """NaN in the last pages' slots behind the sequences' ends, left there by
    others: nothing is computed again for them (that takes 40 times as long and
    more)."""
    length = [max(length + 7 * i, n) for i, n in enumerate(new)]
    s = Setup(rows, cache, 8, 1, D, page, new=new, length=length, seed=7)
    s.fill().plan()
    clean, _ = fastest(s)
    tails = [-l % page for l in length]
    full = torch.tensor([l + t for l, t in zip(length, tails)], dtype=torch.int32).cuda()
    start = torch.tensor([0] + list(np.cumsum(tails)), dtype=torch.int32).cuda()
    nan = torch.full((sum(tails), 1, D), math.nan, dtype=s.dt, device="cuda")
    assert sum(tails) > 0
    s.cache.batch_async(start, full, s.dev["table"], rows=sum(tails))
    s.cache.append_async(0, nan, nan)
    s.plan()
    stale, out = fastest(s)
    ref, tol = s.reference()
    assert ((out.double() - ref).abs() <= tol).all()
    assert stale < 3 * clean, (stale, clean)


@pytest.mark.parametrize("rows,cache", [("bf16", "mxfp4"), ("f16", "mxfp4")])
@pytest.mark.parametrize("D,new", [(64, 2), (64, 4), (128, 2)])
def test_large_values_in_4_bits_cost_nothing(rows, cache, D, new):
    """Values whose scales pass 4 at keys that some of a tile's columns do not see
    while they have seen none: nothing is computed again for them."""
    times = []
    for size in (1.0, 30.0, 30000.0):
        first = [0 if i == 0 else 100 for i in range(new)] * 64
        s = Setup(rows, cache, 8, 1, D, 64, new=(new,) * 64, length=(1500,) * 64, first=first, seed=8)
        s.v = (s.v.clamp(-2, 2).double() * size).to(s.dt)
        s.dev["v"] = s.v.cuda()
        s.fill().plan()
        t, out = fastest(s)
        times.append(t)
        rows_checked = slice(0, 2 * new)
        s.new, s.length = s.new[:2], s.length[:2]
        ref, tol = s.reference()
        assert ((out[rows_checked].double() - ref).abs() <= tol).all()
    assert max(times) < 3 * times[0], times


@pytest.mark.parametrize("rows,cache", COMBOS)
@pytest.mark.parametrize("new", [1, 50])
def test_infinite_sinks(rows, cache, new):
    """A sink of infinity takes all the weight, one of minus infinity none."""
    s = Setup(rows, cache, 8, 2, 64, 16, new=(new,), length=(3000,))
    sinks = torch.tensor([math.inf, -math.inf] * 4)
    s.fill().plan()
    out = s.attend(sinks=sinks.cuda())
    ref, tol = s.reference()
    assert (out[:, 0::2] == 0).all()
    assert ((out.double() - ref).abs() <= tol)[:, 1::2].all()


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "mxfp4")])
def test_seen_infinities_and_nan_do(rows, cache):
    """A row that sees a NaN or infinite value has it in its result, as the
    sum has; a row before it has not."""
    n = 40
    s = Setup(rows, cache, 4, 1, 64, 16, new=(n,), length=(n,))
    s.dev["v"][20, 0, 7] = math.nan
    s.dev["v"][30, 0, 40] = math.inf
    s.fill().plan()
    out = s.attend()
    assert torch.isfinite(out[:20]).all()
    assert torch.isnan(out[20:, :, 7]).all()
    if cache == "mxfp4":
        assert torch.isnan(out[20:, :, :32]).all() and torch.isnan(out[30:, :, 32:]).all()
        assert torch.isfinite(out[20:30, :, 32:]).all()
    else:
        assert (out[30:, :, 40] == math.inf).all()
        keep = torch.ones(64, dtype=torch.bool)
        keep[[7, 40]] = False
        assert torch.isfinite(out[:, :, keep]).all()


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "mxfp4"), ("bf16", "mxfp4")])
def test_large_and_small_values(rows, cache):
    """Scores of hundreds (one key takes all the weight) and values near the
    ends of the type's range."""
    s = Setup(rows, cache, 8, 2, 64, 16, new=(1, 50), length=(90, 130), scale_values=12.0)
    s.check()
    s = Setup(rows, cache, 8, 2, 64, 16, new=(1, 50), length=(90, 130))
    big = 3e4 if rows == "f16" else 1e30
    s.v = (s.v.double() * big / 8).to(s.dt)
    s.dev["v"] = s.v.cuda()
    s.check()
    tiny = 2.0 ** -12 if rows == "f16" else 1e-30
    s.v = (s.v.double() / big * 8 * tiny).to(s.dt)
    s.dev["v"] = s.v.cuda()
    s.check()


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f16", "mxfp4"), ("f32", "f32")])
def test_values_of_very_different_size(rows, cache):
    """V rows whose sizes span the type: the small ones keep their part."""
    s = Setup(rows, cache, 4, 1, 64, 16, new=(3,), length=(200,))
    span = torch.exp2(torch.randint(-9, 9, (200, 1, 1), generator=torch.Generator().manual_seed(2)).double())
    s.v = (s.v.double() * span).to(s.dt)
    s.dev["v"] = s.v.cuda()
    s.check()


def test_strided_rows_and_layers():
    """Q and out as views of wider rows; a layer other than the first."""
    s = Setup("bf16", None, 8, 2, 64, 16, new=(4, 1), length=(60, 31), layers=3, layer=2)
    s.fill().plan()
    wide = torch.zeros(5, 16, 64, dtype=s.dt, device="cuda")
    wide[:, 4:12] = s.dev["q"]
    out = torch.full((5, 12, 64), 7.0, dtype=s.dt, device="cuda")
    s.cache.attend_async(2, wide[:, 4:12], out[:, 1:9])
    s.cache.sync()
    ref, tol = s.reference()
    assert ((out[:, 1:9].cpu().double() - ref).abs() <= tol).all()
    assert (out[:, 0] == 7).all() and (out[:, 9:] == 7).all()
    other = s.cache
    other.attend_async(0, s.dev["q"], out[:, :8])  # layer 0 holds nothing: K = 0 and V = 0
    other.sync()
    assert (out[:, :8] == 0).all()


def test_offsets_past_32_bits():
    """A pool of over 4 GiB, the pages at its end."""
    import ttl_moe
    pages = 40000
    with ttl_moe.KvCache(pages=pages, page_tokens=64, rows="bf16", max_rows=200, device=0,
                         stream=torch.cuda.current_stream()) as c:
        assert pages * c.page_bytes() > 2 ** 32
        g = torch.Generator(device="cuda").manual_seed(0)
        n = 200
        q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda").bfloat16() for h in (64, 8, 8))
        table = torch.tensor([[39999, 0, 32768, 39998]], dtype=torch.int32).cuda()
        for new in (n, 1):
            c.batch_async(torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda(),
                          table, rows=new)
            if new == n:
                c.append_async(0, k, v)
                k2, v2 = torch.empty_like(k), torch.empty_like(v)
                c.read_async(0, k2, v2)
                c.sync()
                assert torch.equal(k2, k) and torch.equal(v2, v)
            out = torch.empty(new, 64, 64, dtype=q.dtype, device="cuda")
            c.attend_async(0, q[n - new:], out)
            c.sync()
            ref, tol = kv_plain.attend(q[n - 2:].cpu().double(), k.cpu().double(), v.cpu().double(), torch.arange(n - 2, n),
                                       "bf16", "bf16")
            assert ((out[-1].cpu().double() - ref[-1]).abs() <= tol[-1]).all()


@pytest.mark.parametrize("new", [1, 40])
def test_leading_columns_of_a_wide_page_table(new):
    """A server's table has room for the longest sequence; a batch takes the
    columns that it needs."""
    s = Setup("bf16", None, 8, 2, 64, 16, new=(new, 1, 3), length=(90, 33, 150))
    s.fill()
    wide = torch.full((5, 64), -1, dtype=torch.int32)
    wide[:3, :s.table.shape[1]] = s.table
    s.dev["table"] = wide.cuda()[:, :s.table.shape[1]]
    s.plan()
    out = s.attend()
    ref, tol = s.reference()
    assert ((out.double() - ref).abs() <= tol).all()


def test_pages_shared_by_sequences():
    """Two sequences over the same first pages."""
    s = Setup("bf16", None, 8, 2, 64, 16, new=(1, 1), length=(40, 40))
    s.table[1, :2] = s.table[0, :2]
    s.dev["table"] = s.table.cuda()
    s.k[40:72], s.v[40:72] = s.k[:32], s.v[:32]
    s.dev["k"], s.dev["v"] = s.k.cuda(), s.v.cuda()
    s.check()


# ---- together, as a program uses them ----

@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "mxfp4")])
def test_prompt_then_tokens(rows, cache):
    """Two prompts of unequal length in chunks, then tokens one by one, against
    attention over the whole sequences."""
    import ttl_moe
    H, KV, D, page = 8, 2, 64, 16
    freq, scale = ttl_moe.gptoss_rope()
    L = [75, 41]
    g = torch.Generator().manual_seed(11)
    dt = TYPES[rows]
    qkv = [[torch.randn(l, h, D, generator=g).to(dt) for h in (H, KV, KV)] for l in L]
    table = torch.arange(12, dtype=torch.int32).flip(0).reshape(2, 6).contiguous().cuda()
    steps = [((32, 20), (32, 20)), ((30, 18), (62, 38))] + [((1, 1), (63 + i, 39 + i)) for i in range(3)] + \
            [((1, 0), (66 + i, 41)) for i in range(10)]
    got = [[], []]
    with ttl_moe.KvCache(pages=12, page_tokens=page, q_heads=H, kv_heads=KV, rows=rows, cache=cache, max_seqs=2,
                         max_rows=116, window=40, rope_freq=freq, rope_scale=scale, layers=2, device=0) as c:
        st = torch.cuda.ExternalStream(c.stream())
        with torch.cuda.stream(st):
            for new, length in steps:
                rowsn = sum(new)
                cat = [torch.cat([qkv[s][i][length[s] - new[s]:length[s]] for s in (0, 1)]).cuda() for i in range(3)]
                start = torch.tensor([0, new[0], rowsn], dtype=torch.int32).cuda()
                ln = torch.tensor(length, dtype=torch.int32).cuda()
                c.batch_async(start, ln, table, rows=rowsn, max_new=max(new))
                outs = []
                for layer in (0, 1):
                    qr, out = torch.empty_like(cat[0]), torch.empty_like(cat[0])
                    c.append_async(layer, cat[1], cat[2], q=cat[0], q_out=qr)
                    c.attend_async(layer, qr, out, sliding=layer == 0)
                    outs.append(out)
                c.sync()
                for s in (0, 1):
                    a = 0 if s == 0 else new[0]
                    got[s].append([o[a:a + new[s]].cpu() for o in outs + [qr]])
        # what the cache holds of both, and the rotated rows that were attended with
        c.batch_async(torch.tensor([0, 75, 116], dtype=torch.int32).cuda(), torch.tensor(L, dtype=torch.int32).cuda(), table,
                      rows=116)
        kv = [[torch.empty(116, KV, D, dtype=dt, device="cuda") for _ in "kv"] for _ in (0, 1)]
        torch.cuda.synchronize()
        for layer in (0, 1):
            c.read_async(layer, *kv[layer])
        c.sync()
    kv = [[t.cpu().double() for t in x] for x in kv]
    for s, l in enumerate(L):
        pos = torch.arange(l)
        a = 75 * s
        q = torch.cat([x[2] for x in got[s]])
        turned = kv_plain.rotate(qkv[s][0].double(), pos, freq, scale)
        assert ((q.double() - turned).abs() <= 8 * 2.0 ** -23 * 2 * 5 + unit(rows) * turned.abs()).all()
        for layer in (0, 1):
            ref, tol = kv_plain.attend(q, kv[layer][0][a:a + l], kv[layer][1][a:a + l], pos, rows, cache,
                                       window=40 if layer == 0 else 0)
            out = torch.cat([x[layer] for x in got[s]])
            assert ((out.double() - ref).abs() <= tol).all()


def test_paged_path_equals_the_attention_block():
    """ttl_attn's attended rows (the oracle's attention_steps) from the same
    weights: projections in numpy, then append and attend over the paged
    cache, a sliding and a full layer, as a prompt and token by token."""
    import oracle
    import ttl_moe
    from ttl_moe import synth
    P = 140
    freq, scale = ttl_moe.gptoss_rope()

    def weights(w, rows):
        b = w.reshape(rows, 90, 34)
        d = np.ascontiguousarray(b[:, :, :2]).view(np.float16).astype(np.float64)
        return (b[:, :, 2:].view(np.int8) * d).reshape(rows, 2880)

    for layer in (0, 1):
        t = synth.attention_layer_host(5, layer)
        x = synth.inputs_host(90 + layer, P)
        _, want = oracle.attention_steps(t, layer, x, impl="ref" if oracle.ref_available() else "port")
        xn = x.astype(np.float64)
        xn = xn / np.sqrt((xn ** 2).mean(1, keepdims=True) + 1e-5) * t["attn_norm"]
        q, k, v = (torch.from_numpy((xn @ weights(t[n + "_w"], r).T + t[n + "_b"]).astype(np.float32)).reshape(P, -1, 64).cuda()
                   for n, r in (("q", 4096), ("k", 512), ("v", 512)))
        table = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
        sinks = torch.from_numpy(t["sinks"]).cuda()
        for chunks in ([P], [100] + [1] * 40):
            got, at = [], 0
            with ttl_moe.KvCache(pages=3, rows="f32", max_rows=P, window=128, rope_freq=freq, rope_scale=scale, device=0,
                                 stream=torch.cuda.current_stream()) as c:
                for n in chunks:
                    c.batch_async(torch.tensor([0, n], dtype=torch.int32).cuda(),
                                  torch.tensor([at + n], dtype=torch.int32).cuda(), table, rows=n)
                    rot, out = torch.empty_like(q[:n]), torch.empty_like(q[:n])
                    c.append_async(0, k[at:at + n], v[at:at + n], q=q[at:at + n], q_out=rot)
                    c.attend_async(0, rot, out, sinks=sinks, sliding=layer % 2 == 0)
                    c.sync()
                    got.append(out.cpu())
                    at += n
            a = torch.cat(got).reshape(P, 4096).numpy()
            worst = max(float(np.max(np.abs(a[p] - want[p])) / np.max(np.abs(want[p]))) for p in range(P))
            assert worst <= 1e-3, (layer, len(chunks), worst)  # the attention block's own bar


def test_graph_replays_follow_the_batch():
    """Plan, append and attend captured once; replays with other lengths, rows
    and pages in the same arrays."""
    import ttl_moe
    H, KV, D, page, n, L = 8, 2, 64, 16, 3, 70
    st = torch.cuda.Stream()
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, L, KV, D, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(L, 2, H, D, generator=g).bfloat16()
    dev = dict(start=torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), length=torch.zeros(2, dtype=torch.int32).cuda(),
               table=torch.arange(10, dtype=torch.int32).reshape(2, 5).contiguous().cuda(),
               q=torch.zeros(2, H, D).bfloat16().cuda(), k=torch.zeros(2, KV, D).bfloat16().cuda(),
               v=torch.zeros(2, KV, D).bfloat16().cuda())
    out = torch.zeros_like(dev["q"])
    torch.cuda.synchronize()
    with ttl_moe.KvCache(pages=10, page_tokens=page, q_heads=H, kv_heads=KV, rows="bf16", max_seqs=2, max_rows=2, device=0,
                         stream=st) as c:
        def step():
            c.batch_async(dev["start"], dev["length"], dev["table"], rows=2, max_new=1)
            c.append_async(0, dev["k"], dev["v"])
            c.attend_async(0, dev["q"], out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step()
        for p in range(L):
            lens = [p + 1, max(0, p - 20) + 1]
            with torch.cuda.stream(st):
                dev["length"].copy_(torch.tensor(lens, dtype=torch.int32))
                for s in (0, 1):
                    for name, src in (("k", k), ("v", v)):
                        dev[name][s].copy_(src[s, lens[s] - 1])
                dev["q"].copy_(q[p])
                graph.replay()
            if p % 23 == 0 or p == L - 1:
                c.sync()
                for s in (0, 1):
                    ref, tol = kv_plain.attend(q[p, s:s + 1].double(), k[s, :lens[s]].double(), v[s, :lens[s]].double(),
                                               torch.tensor([lens[s] - 1]), "bf16", "bf16")
                    assert ((out[s:s + 1].cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4")])
def test_two_graphs_of_one_handle_replayed_in_turn(rows, cache):
    """Two graphs share the handle's plan and workspace: one of many tokens and a
    prompt, whose short sequences go with the prompt or by themselves as their
    lengths on the device ask, one of a prompt alone.  Replayed in turn, each
    gives what its calls give without a graph, bit for bit."""
    new, length = (1,) * 20 + (90,) + (3,) * 20, (2600,) * 20 + (500,) + (2500,) * 20
    st = torch.cuda.Stream()
    s = Setup(rows, cache, 4, 2, 64, 64, new=new, length=length, seed=3, stream=st)
    s.fill()
    d = s.dev
    short = torch.tensor([7 if n < 90 else l for n, l in zip(new, length)], dtype=torch.int32).cuda()
    full, now = d["length"].clone(), d["length"]
    one = dict(start=torch.tensor([0, 90], dtype=torch.int32).cuda(), length=torch.tensor([500], dtype=torch.int32).cuda(),
               table=d["table"][20:21].contiguous(), q=d["q"][20:110].contiguous())
    out, out1 = torch.zeros_like(d["q"]), torch.zeros_like(one["q"])

    def many():
        s.cache.batch_async(d["start"], now, d["table"], rows=s.rows, max_new=90)
        s.cache.attend_async(0, d["q"], out)

    def single():
        s.cache.batch_async(one["start"], one["length"], one["table"], rows=90, max_new=90)
        s.cache.attend_async(0, one["q"], out1)

    want = {}
    for name, lens in (("full", full), ("short", short)):
        torch.cuda.synchronize()
        now.copy_(lens)
        torch.cuda.synchronize()
        many()
        s.cache.sync()
        want[name] = out.clone()
    single()
    s.cache.sync()
    want["one"] = out1.clone()
    graphs = []
    for f in (many, single):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            f()
    for name, lens in (("full", full), ("short", short), ("full", full), ("short", short)):
        torch.cuda.synchronize()
        out.fill_(0), out1.fill_(0), now.copy_(lens)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graphs[0].replay()
            graphs[1].replay()
        s.cache.sync()
        assert torch.equal(out, want[name]) and torch.equal(out1, want["one"])
    assert not torch.equal(want["full"], want["short"])


def test_two_handles_on_two_streams_at_once():
    a = Setup("bf16", None, 8, 2, 64, 16, new=(1,), length=(9000,), seed=1, stream=torch.cuda.Stream())
    b = Setup("bf16", None, 8, 2, 64, 16, new=(1,), length=(8000,), seed=2, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    for s in (a, b):
        s.fill().plan()
    outs = [[torch.zeros_like(s.dev["q"]) for _ in range(20)] for s in (a, b)]
    torch.cuda.synchronize()
    for i in range(20):
        for s, o in zip((a, b), outs):
            s.cache.attend_async(0, s.dev["q"], o[i])
    for s, o in zip((a, b), outs):
        s.cache.sync()
        ref, tol = s.reference()
        for x in o:
            assert torch.equal(x, o[0])
        assert ((o[0].cpu().double() - ref).abs() <= tol).all()


# ---- what is refused, and what only the device can see ----

def test_bad_numbers_are_reported_and_skipped():
    s = Setup("bf16", None, 8, 2, 64, 16, new=(1, 2, 1), length=(30, 40, 50)).fill()
    ref, tol = s.reference()
    d = s.dev

    def go(start=None, length=None, table=None, max_new=2):
        s.cache.batch_async(d["start"] if start is None else start, d["length"] if length is None else length,
                            d["table"] if table is None else table, rows=4, max_new=max_new)
        out = torch.full_like(d["q"], 7.0)
        s.cache.attend_async(0, d["q"], out)
        return out

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    # (row_start, length, max_new) and the sequences that stay good
    for kw, good in ((dict(length=i32(30, 1, 50)), (0, 2)), (dict(length=i32(30, -7, 50)), (0, 2)),
                     (dict(length=i32(30, 40, 10 ** 6)), (0, 1)), (dict(length=i32(30, 40, 2 ** 31 - 1)), (0, 1)),
                     (dict(start=i32(0, 1, 3, 900)), (0, 1)), (dict(start=i32(0, 1, 3, -4)), (0, 1)),
                     (dict(start=i32(0, 2 ** 31 - 1, 3, 4)), (2,)), (dict(max_new=1), (0, 2))):
        out = go(**kw)
        with pytest.raises(RuntimeError, match="row_start or length"):
            s.cache.sync()
        rows = {0: [0], 1: [1, 2], 2: [3]}
        for q in range(3):
            for r in rows[q]:
                o = out[r].cpu().double()
                if q in good:
                    assert ((o - ref[r]).abs() <= tol[r]).all(), (kw, q)
                else:
                    assert (o == 7).all(), (kw, q)
    bad = s.table.clone()
    bad[1, 1] = 10 ** 6
    out = go(table=bad.cuda())
    with pytest.raises(RuntimeError, match="page id"):
        s.cache.sync()
    for r in (0, 3):
        assert ((out[r].cpu().double() - ref[r]).abs() <= tol[r]).all()
    # append and read skip it: sequence 1's rows are in its third page
    bad = s.table.clone()
    bad[1, 2] = -1
    s.cache.batch_async(d["start"], d["length"], bad.cuda(), rows=4, max_new=2)
    k = torch.full((4, 2, 64), 2.0, dtype=s.dt, device="cuda")
    s.cache.append_async(0, k, k)
    a, b = torch.zeros_like(k), torch.zeros_like(k)
    s.cache.read_async(0, a, b)
    with pytest.raises(RuntimeError, match="page id"):
        s.cache.sync()
    assert (a[[0, 3]] == 2).all() and (a[[1, 2]] == 0).all()
    s.plan()
    s.cache.sync()  # reported once; the handle stays usable


@pytest.mark.parametrize("rows,cache", COMBOS)
@pytest.mark.parametrize("new", [1, 3, 60])
def test_pages_below_the_window_may_be_gone(rows, cache, new):
    """A server frees the pages that a window has passed and leaves -1 in the
    table: a sliding call says nothing, a full one does, and so does a sliding
    one where a page that it sees is gone."""
    page, window, n = 16, 40, 391
    s = Setup(rows, cache, 8, 2, 64, page, new=(new, 1), length=(n, 50), window=window)
    s.fill()
    gone = (n - new - window + 1) // page  # pages below the lowest visible position
    for more, bad in ((0, False), (1, True)):
        table = s.table.clone()
        table[0, :gone + more] = torch.tensor([-1, 10 ** 6])[torch.arange(gone + more) % 2].to(torch.int32)
        s.dev["table"] = table.cuda()
        s.plan()
        out = torch.full_like(s.dev["q"], 7.0)
        s.cache.attend_async(0, s.dev["q"], out, sliding=True)
        if bad:
            with pytest.raises(RuntimeError, match="page id"):
                s.cache.sync()
            continue
        s.cache.sync()
        ref, tol = s.reference(sliding=True)
        assert ((out.cpu().double() - ref).abs() <= tol).all()
        s.cache.attend_async(0, s.dev["q"], out)
        with pytest.raises(RuntimeError, match="page id"):
            s.cache.sync()


def test_rows_that_see_nothing_ask_for_no_page():
    s = Setup("bf16", None, 8, 2, 64, 16, new=(40, 1), length=(100, 60), first=[1 << 30] * 41)
    s.fill()
    s.dev["table"] = torch.full_like(s.dev["table"], -1)
    s.plan()
    assert (s.attend() == 0).all()


def test_a_plan_of_another_shape_is_reported():
    """A captured attend whose plan was replaced by one of another shape."""
    st = torch.cuda.Stream()
    s = Setup("bf16", None, 8, 1, 64, 16, new=(1,), length=(50,), stream=st)
    big = Setup("bf16", None, 8, 1, 64, 16, new=(40,), length=(50,), stream=st)
    torch.cuda.synchronize()
    big.fill()
    d = big.dev
    big.cache.batch_async(s.dev["start"], d["length"], d["table"], rows=1, max_new=1)
    out = torch.full_like(d["q"], 7.0)
    big.cache.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        big.cache.attend_async(0, d["q"], out)
    big.plan()
    with torch.cuda.stream(st):
        g.replay()
    with pytest.raises(RuntimeError, match="another shape"):
        big.cache.sync()
    assert (out == 7).all()
    s.cache.close()


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f32", "mxfp4"), ("bf16", "mxfp4")])
@pytest.mark.parametrize("small", [((0, 8), (24,)), ((0, 3), (3,)), ((0, 40, 44), (60, 9))])
def test_a_graph_of_appends_after_a_batch_of_other_rows(rows, cache, small):
    """Append and read captured with 32 rows of four sequences, replayed after a
    batch of fewer or more rows and sequences whose page table is shorter: the
    rows that both have are stored, no other slot changes, and the difference is
    reported."""
    st = torch.cuda.Stream()
    s = Setup(rows, cache, 4, 2, 64, 16, new=(8, 8, 8, 8), length=(40, 24, 60, 33), stream=st)
    torch.cuda.synchronize()
    s.fill()
    c, d, total = s.cache, s.dev, sum(s.length)

    def whole():
        """Every token of every sequence, as the cache holds it."""
        off = torch.tensor(s.tok0, dtype=torch.int32).cuda()
        kv = [torch.zeros_like(d["k"]), torch.zeros_like(d["v"])]
        torch.cuda.synchronize()
        c.batch_async(off, d["length"], d["table"], rows=total)
        c.read_async(0, *kv)
        c.sync()
        return kv

    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(32, 2, 64, generator=g).to(s.dt).cuda() for _ in range(2))
    q, q_out = torch.ones_like(d["q"]), torch.full_like(d["q"], 7.0)
    k2, v2 = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    before = whole()
    s.plan()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        c.append_async(0, k, v, q=q, q_out=q_out)
        c.read_async(0, k2, v2)
    start, length = (torch.tensor(x, dtype=torch.int32).cuda() for x in small)
    table = d["table"][2:2 + len(small[1])].contiguous()  # the third sequence's pages (and the fourth's)
    torch.cuda.synchronize()
    n = min(32, small[0][-1])
    c.batch_async(start, length, table, rows=small[0][-1])
    with torch.cuda.stream(st):
        graph.replay()
    with pytest.raises(RuntimeError, match="another shape"):
        c.sync()
    c.sync()  # once
    held = [kv_plain.held(x.cpu().double(), cache).to(s.dt) for x in (k, v)]
    for got, want in zip((k2, v2), held):
        assert torch.equal(got[:n].cpu(), want[:n]) and (got[n:] == 7).all()
    assert (q_out[:n] == 1).all() and (q_out[n:] == 7).all()
    at = s.tok0[2] + torch.arange(n) + small[1][0] - (small[0][1] - small[0][0])
    for now, was, want in zip(whole(), before, held):
        was[at] = want[:n].cuda()
        assert torch.equal(now, was)


@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "mxfp4")])
@pytest.mark.parametrize("sliding", [False, True])
def test_a_graph_of_tokens_after_a_batch_with_a_prompt(rows, cache, sliding):
    """Beside a prompt, tokens have tiles as wide as without one: a graph that
    launches their kernel alone would leave the prompt out."""
    st = torch.cuda.Stream()
    s = Setup(rows, cache, 8, 1, 64, 16, new=(1, 90, 1), length=(150, 140, 200), window=30, stream=st)
    one = torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    s.fill()
    d, out = s.dev, torch.full_like(s.dev["q"], 7.0)
    torch.cuda.synchronize()
    s.cache.batch_async(one, d["length"], d["table"], rows=s.rows, max_new=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s.cache.attend_async(0, d["q"], out, sliding=sliding)
    with torch.cuda.stream(st):
        graph.replay()
    s.cache.sync()  # its own plan
    assert (out[:3] != 7).any() and (out[3:] == 7).all()
    out.fill_(7.0)
    torch.cuda.synchronize()
    s.plan()
    with torch.cuda.stream(st):
        graph.replay()
    with pytest.raises(RuntimeError, match="another shape"):
        s.cache.sync()
    assert (out == 7).all()
    # and the other way round
    mixed = torch.cuda.CUDAGraph()
    with torch.cuda.graph(mixed, stream=st):
        s.cache.attend_async(0, d["q"], out, sliding=sliding)
    s.cache.batch_async(one, d["length"], d["table"], rows=s.rows, max_new=1)
    with torch.cuda.stream(st):
        mixed.replay()
    with pytest.raises(RuntimeError, match="another shape"):
        s.cache.sync()
    assert (out == 7).all()


@pytest.mark.parametrize("rows", ["bf16", "f32"])
def test_a_graph_of_attention_after_a_batch_of_other_rows(rows):
    """The same kernels, another number of rows: those that both have are
    written, and the difference is reported."""
    st = torch.cuda.Stream()
    s = Setup(rows, None, 8, 2, 64, 16, new=(1,) * 6, length=(30, 41, 52, 3, 64, 75), stream=st)
    torch.cuda.synchronize()
    s.fill()
    d, out = s.dev, torch.full_like(s.dev["q"], 7.0)
    ref, tol = s.reference()
    torch.cuda.synchronize()

    def batch(n):
        s.cache.batch_async(d["start"][:n + 1].contiguous(), d["length"][:n].contiguous(), d["table"], rows=n, max_new=1)

    batch(4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s.cache.attend_async(0, d["q"], out)
    for n in (6, 2, 4):
        out.fill_(7.0)
        torch.cuda.synchronize()
        batch(n)
        with torch.cuda.stream(st):
            graph.replay()
        if n == 4:
            s.cache.sync()
        else:
            with pytest.raises(RuntimeError, match="another shape"):
                s.cache.sync()
        m = min(n, 4)
        assert ((out[:m].cpu().double() - ref[:m]).abs() <= tol[:m]).all()
        assert (out[m:] == 7).all()


def test_calls_after_a_batch_that_was_only_captured():
    """A batch call inside a capture runs nothing: append, read and attend after
    it meet the plan of the batch before, or none, and say so."""
    st = torch.cuda.Stream()
    s = Setup("bf16", None, 4, 2, 64, 16, new=(6,), length=(20,), stream=st)
    k, v = s.dev["k"][:6].contiguous(), s.dev["v"][:6].contiguous()
    outs = [torch.full_like(x, 7.0) for x in (s.dev["q"], s.dev["q"], k, v)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s.plan()
    for earlier in (False, True):
        for call in (lambda: s.cache.append_async(0, k, v, q=s.dev["q"], q_out=outs[0]),
                     lambda: s.cache.read_async(0, outs[2], outs[3]),
                     lambda: s.cache.attend_async(0, s.dev["q"], outs[1])):
            call()
            with pytest.raises(RuntimeError, match="another shape"):
                s.cache.sync()
        n = 2 if earlier else 0
        assert (outs[1] == 7).all()  # two rows make narrower tiles: other kernels
        for o in (outs[0], outs[2], outs[3]):
            assert (o[n:] == 7).all() and (o[:n] != 7).all()
        if earlier:
            break
        s.cache.batch_async(torch.tensor([0, 2], dtype=torch.int32).cuda(), s.dev["length"], s.dev["table"], rows=2)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=st):
            s.plan()
    # the captured batch, once it has run, is the plan
    with torch.cuda.stream(st):
        graph.replay()
    s.cache.append_async(0, k, v, q=s.dev["q"], q_out=outs[0])
    s.cache.read_async(0, outs[2], outs[3])
    s.cache.sync()
    assert torch.equal(outs[0], s.dev["q"]) and torch.equal(outs[2], k) and torch.equal(outs[3], v)


def test_overlapping_rows_are_refused():
    """What a call writes and what it reads lie apart; views of one array side by
    side do."""
    n, H, KV, D = 5, 4, 2, 64
    s = Setup("bf16", None, H, KV, D, 16, new=(n,), length=(20,), freq=100.0 ** (-np.arange(32) / 32))
    s.fill().plan()
    c = s.cache
    flat = torch.randn(4 * n * (H + 2 * KV) * D, device="cuda").bfloat16()

    def rows(start, heads, stride, count=n):
        return flat[start:].as_strided((count, heads, D), (stride, D, 1), start)

    S = (H + 2 * KV) * D
    q, k, v = rows(0, H, S), rows(H * D, KV, S), rows((H + KV) * D, KV, S)
    kw, other = dict(k=k, v=v, q=q), torch.empty(n, H, D, dtype=s.dt, device="cuda")
    for q_out, what in ((rows(D, H, S), "q"), (rows(2 * S, H, S), "q"), (rows(KV * D, H, S), "q"), (rows(S - D, H, S), "q"),
                        (rows(8, H, H * D), "q"), (rows(H * D + 8, H, S), "q"), (rows(H * D, H, S), "k")):
        with pytest.raises(RuntimeError, match=f"q_out overlaps {what}"):
            c.append_async(0, **kw, q_out=q_out)
    with pytest.raises(RuntimeError, match="q_out overlaps v"):
        c.append_async(0, k, rows(10 * S, KV, S), q=other, q_out=rows(10 * S, H, S))
    for out in (rows(D, H, S), rows(S, H, S), rows(8, H, H * D)):
        with pytest.raises(RuntimeError, match="out overlaps q"):
            c.attend_async(0, q, out)
    for v_out in (k, rows(H * D + 8, KV, S), rows(H * D + S, KV, S)):
        with pytest.raises(RuntimeError, match="v overlaps k"):
            c.read_async(0, k, v_out)
    # apart: in place, side by side, behind one another
    c.append_async(0, **kw, q_out=q)
    c.attend_async(0, rows(2 * KV * D, H, S), rows(n * S + 2 * KV * D, H, S))
    c.attend_async(0, rows(0, H, 2 * H * D), rows(H * D, H, 2 * H * D))
    c.attend_async(0, rows(H * D, H, 2 * H * D), rows(0, H, 2 * H * D))
    c.read_async(0, rows(0, KV, 2 * KV * D), rows(KV * D, KV, 2 * KV * D))
    c.read_async(0, rows(0, KV, KV * D), rows(n * KV * D, KV, KV * D))
    c.sync()


def test_refusals():
    import ttl_moe
    s = Setup("bf16", None, 8, 2, 64, 16, new=(2,), length=(5,))
    c, d = s.cache, s.dev
    L, h = ttl_moe.lib(), s.cache.h
    k = d["k"][:2].contiguous()
    out = torch.empty_like(d["q"])

    def refused(rc, code, match):
        assert rc == code, rc
        assert match in L.ttl_kv_last_error(h).decode(), L.ttl_kv_last_error(h)

    with pytest.raises(RuntimeError, match="no batch"):
        c.attend_async(0, d["q"], out)
    with pytest.raises(RuntimeError, match="seqs must be"):
        c.batch_async(d["start"].new_zeros(4), d["start"].new_zeros(3), d["table"].new_zeros(3, 1), rows=2)
    with pytest.raises(RuntimeError, match="rows exceed"):
        c.batch_async(d["start"], d["length"], d["table"], rows=100)
    host = d["start"].cpu()
    refused(L.ttl_kv_batch_async(h, 1, 2, 2, host.data_ptr(), d["length"].data_ptr(), d["table"].data_ptr(), 1, None, None),
            ttl_moe.TTL_ERR_ARGUMENT, "row_start is not")
    refused(L.ttl_kv_batch_async(h, 1, 2, 2, d["start"].data_ptr(), None, d["table"].data_ptr(), 1, None, None),
            ttl_moe.TTL_ERR_ARGUMENT, "null length")
    refused(L.ttl_kv_batch_async(h, 1, 2, 2, d["start"].data_ptr(), d["length"].data_ptr(), d["table"].data_ptr(), 0, None, None),
            ttl_moe.TTL_ERR_ARGUMENT, "page_stride")
    s.plan()
    for layer in (-1, 1):
        with pytest.raises(RuntimeError, match="out of range"):
            c.attend_async(layer, d["q"], out)
    with pytest.raises(RuntimeError, match="without a window"):
        c.attend_async(0, d["q"], out, sliding=True)
    with pytest.raises(RuntimeError, match="cap finite"):
        c.attend_async(0, d["q"], out, cap=-1.0)
    with pytest.raises(RuntimeError, match="scale must be finite"):
        c.attend_async(0, d["q"], out, scale=math.nan)
    with pytest.raises(RuntimeError, match="out must not be q"):
        c.attend_async(0, d["q"], d["q"])
    with pytest.raises(RuntimeError, match="q and q_out"):
        c.append_async(0, k, k, q=d["q"])
    q, o = d["q"].data_ptr(), out.data_ptr()
    A = ttl_moe.TTL_ERR_ARGUMENT
    refused(L.ttl_kv_attend_async(h, 0, 2, q, 512, o, 512, 0.0, 0.0, None, None), A, "unknown flags")
    refused(L.ttl_kv_attend_async(h, 0, 0, q + 2, 512, o, 512, 0.0, 0.0, None, None), A, "not aligned")
    refused(L.ttl_kv_attend_async(h, 0, 0, q, 500, o, 512, 0.0, 0.0, None, None), A, "row stride")
    refused(L.ttl_kv_attend_async(h, 0, 0, q, 513, o, 512, 0.0, 0.0, None, None), A, "row stride")
    refused(L.ttl_kv_attend_async(h, 0, 0, None, 512, o, 512, 0.0, 0.0, None, None), A, "null q")
    refused(L.ttl_kv_attend_async(h, 0, 0, q, 512, torch.empty(2, 512).data_ptr(), 512, 0.0, 0.0, None, None), A, "out is not")
    refused(L.ttl_kv_append_async(h, 0, 1, k.data_ptr(), 64, k.data_ptr(), 128, None, 0, None, 0), A, "row stride")
    refused(L.ttl_kv_append_async(h, 0, 1, k.data_ptr(), 128, k.data_ptr(), 128, q, 512, q, 1024), A, "one stride")
    with pytest.raises(ValueError, match="heads of a row"):
        c.attend_async(0, d["q"].transpose(1, 2).contiguous().transpose(1, 2), out)
    with pytest.raises(ValueError, match="q must be"):
        c.attend_async(0, d["q"].float(), out)
    with pytest.raises(ValueError, match="q must be"):
        c.attend_async(0, d["q"][:1], out)
    with pytest.raises(ValueError, match="sinks must be"):
        c.attend_async(0, d["q"], out, sinks=torch.zeros(3).cuda())
    c.attend_async(0, d["q"], out)
    c.sync()
    # a batch of no rows does nothing
    c.batch_async(d["start"].new_zeros(2), d["length"], d["table"], rows=0)
    e = torch.empty(0, 8, 64, dtype=s.dt, device="cuda")
    c.append_async(0, e[:, :2], e[:, :2])
    c.attend_async(0, e, e.clone())
    c.sync()
