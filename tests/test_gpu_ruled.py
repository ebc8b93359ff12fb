"""Attention over the paged cache with caps, distance biases and masks, over 4-bit pages too, for single rows
and runs of rows, against the definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
POOL = {"i4": torch.uint8, "i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step, relative


@pytest.fixture(scope="module")
def jy():
    import jieyu_amd
    if jieyu_amd.device_count() < 1:
        pytest.fail("no HIP device visible")
    return jieyu_amd


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Cache:
    """Sequences written into a pool in random page order, everything outside them what must never be read: NaN
    scales and words, NaN values.  k, v: what it holds, float64 [n][kv heads][hd] of each sequence; ka, va: bounds of the
    terms that make them up (4 bits: number times step, and low)."""

    def __init__(self, jy, lens, nkv, hd, page, pool, seed=1, layers=2, layer=1):
        g = gen(seed)
        self.lens, self.nkv, self.hd, self.page, self.kind, self.layer = lens, nkv, hd, page, pool, layer
        need = [-(-max(n, 0) // page) for n in lens]
        npages = sum(need) + 2
        order = torch.randperm(npages, generator=g)
        self.tables = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n].int()
            at += n
        self.pool = p = jy.PagePool.empty(layers, npages, page, nkv, hd, dtype=POOL[pool], device=DEV)
        for t in (p.k, p.v):
            t.fill_(-128 if pool == "i8" else 255 if pool == "i4" else math.nan)
        for t in (p.k_scale, p.v_scale):
            if t is not None:
                t.fill_(math.nan)
        self.dtables, self.dlens = self.tables.to(DEV), ints(lens)
        total = sum(max(n, 0) for n in lens)
        kv = torch.randn((total, 2, nkv, hd), generator=g) * torch.exp(0.5 * torch.randn(hd, generator=g))
        seq = [b for b, n in enumerate(lens) for _ in range(n)]
        pos = [i for n in lens for i in range(n)]
        if total:
            p.write(layer, kv[:, 0].to(DEV), kv[:, 1].to(DEV), self.dtables, ints(pos), ints(seq))
            k, v = (t.double().cpu() for t in p.read(layer, self.dtables, ints(pos), ints(seq)))
        else:
            k = v = torch.zeros((0, nkv, hd), dtype=torch.float64)
        cuts = [0]
        for n in lens:
            cuts.append(cuts[-1] + max(n, 0))
        cut = lambda t: [t[a:b] for a, b in zip(cuts, cuts[1:])]  # noqa: E731
        self.k, self.v = cut(k), cut(v)

        def terms(x):  # n step <= the group's range, low >= -its largest: their sum in size
            if pool != "i4":
                return x.abs()
            y = torch.zeros_like(x)
            for i in range(0, hd, 32):
                part = x[..., i:i + 32]
                y[..., i:i + 32] = (part.amax(-1, keepdim=True) - part.amin(-1, keepdim=True)) + part.abs().amax(-1, keepdim=True)
            return y

        self.ka, self.va = cut(terms(k)), cut(terms(v))


def attention64(c, b, q, pos, first, last, cap=0.0, slopes=None, scale=None, io=torch.float32, runs=False):
    """(out, room, p, room of p) of rows q [rows][nh][hd] of sequence b in 64 bits.

    fp32 scores: a sum of hd products of a query held in 24 bits is off by (hd + 2) 2^-24 S, S = scale sum |q| |k| at
    most, the factors, the cap (a tanh to 8 steps) and the bias B = slope x distance by 24 more of S and 8 of S + B.
    Weights: twice that relative, 2 n + 16 steps of the sums; 4-bit pages with bf16 queries take a weight times
    a step as one fp16 number, 2^-11 of it.  A weight far below the largest ends at 2^-39 of the largest weight times
    value.

    Runs of 16-bit rows: a tanh is off by 4 steps of 1, so 8 more of the cap for two scores; a weight is one number of
    the product's type (fp16 over fp16 and 4-bit values, 2^-11; bf16 over the others, 2^-8, or 2^-16 in two parts where
    the outputs are fp16), a 4-bit value one fp16 number, another 2^-11; and fp16 weights end at half a step of their
    smallest, 2^-25 of the largest."""
    rows, nh, hd = q.shape
    runs = runs and io is not torch.float32
    k, v, ka, va = c.k[b], c.v[b], c.ka[b], c.va[b]
    n, per = k.shape[0], nh // c.nkv
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out, room = torch.zeros((rows, nh, hd), dtype=torch.float64), torch.zeros((rows, nh, hd), dtype=torch.float64)
    P, PR = torch.zeros((rows, nh, n), dtype=torch.float64), torch.zeros((rows, nh, n), dtype=torch.float64)
    j = torch.arange(n)
    for h in range(nh):
        x = q[:, h].double()
        s = x @ k[:, h // per].T * scale
        S = (x.abs() @ ka[:, h // per].T * abs(scale))
        if cap:
            s = cap * torch.tanh(s / cap)
        B = torch.zeros_like(s)
        if slopes is not None:
            B = float(slopes[h]) * (torch.tensor(pos)[:, None] - j).abs().double()
            s = s - B
        live = (j >= torch.tensor(first)[:, None]) & (j < torch.tensor(last)[:, None])
        for r in range(rows):
            at = live[r]
            m = int(at.sum())
            if not m:
                continue
            p = torch.softmax(s[r, at], 0)
            ds = 2.0**-24 * ((hd + 24) * S[r, at].max() + 8 * (S[r, at] + B[r, at].abs()).max() + (8 * cap if runs else 0.0))
            rel = float(2 * ds) + (2 * m + 16) * 2.0**-24
            vv, va_ = v[at][:, h // per], va[at][:, h // per]
            out[r, h] = p @ vv
            one = 2.0**-11 if c.kind == "i4" and io is torch.bfloat16 else 0.0
            far = 2.0**-39
            if runs:
                half = c.kind in ("f16", "i4")
                one = {"i4": 2.0**-10, "f16": 2.0**-11}[c.kind] if half else 2.0**-8 if io is torch.bfloat16 else 2.0**-16
                far = 2.0**-25 if half else 2.0**-39
            room[r, h] = (rel + one) * (p @ va_) + m * far * va_.amax()
            P[r, h, at], PR[r, h, at] = p, rel * p + 2.0**-126
    return out, room, P, PR


def check(got, want, room):
    tiny = 2.0**-25 if got.dtype is torch.float16 else 0.0
    off = (got.double().cpu() - want).abs()
    limit = room + HALF[got.dtype] * (want.abs() + room) + tiny
    assert torch.isfinite(got).all() and (off <= limit).all(), f"error {(off / limit.clamp(min=1e-300)).max():.3g} of the bound"


def single(c, q, first=None, max_len=None, **kw):
    """(want, room, p, room of p) of one row per sequence"""
    parts = []
    for b, n in enumerate(c.lens):
        lo = 0 if first is None else max(first[b], 0)
        hi = max(n, 0) if max_len is None or first is None else min(max(n, 0), lo + max_len)
        if max_len is not None and first is None:
            hi = min(hi, max_len)
        parts.append(attention64(c, b, q[b:b + 1], [n - 1], [lo], [hi], io=q.dtype, **kw))
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), [p[2][0] for p in parts], [p[3][0] for p in parts]


SHAPES = [(14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 64), (10, 2, 112), (6, 3, 96), (8, 1, 256), (9, 3, 80), (4, 2, 16),
          (3, 1, 32), (40, 2, 64), (33, 1, 128), (4, 4, 48), (2, 2, 144), (2, 1, 192), (64, 1, 160)]


@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
def test_4bit_shapes(jy, nh, nkv, hd, io):
    c = Cache(jy, [1, 37, 0, 130], nkv, hd, 16, "i4", seed=nh + hd)
    q = torch.randn((4, nh, hd), generator=gen(5)).to(IO[io])
    got = c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 130)
    want, room, _, _ = single(c, q)
    check(got, want, room)
    assert not got[2].any()


@pytest.mark.parametrize("lens", [[1], [15], [16], [17], [31], [32], [33], [127], [129], [1023], [1025], [4097], [0], [0, 0, 5], [1, 1, 1, 2000]])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_4bit_lengths(jy, lens, hd):
    c = Cache(jy, lens, 2, hd, 32, "i4", seed=len(lens) + lens[0])
    q = torch.randn((len(lens), 4, hd), generator=gen(3))
    check(c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, max(lens)), *single(c, q)[:2])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO))
def test_rules_types_and_pages(jy, page, pool, io):
    c = Cache(jy, [page, page + 1, 3 * page + 7], 2, 64, page, pool, seed=page)
    q = (3 * torch.randn((3, 6, 64), generator=gen(2))).to(IO[io])
    slopes = torch.tensor([0.0, 0.5, -0.01, 0.03, 1.0, 0.002])
    got = c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, max(c.lens), cap=4.0, slopes=slopes.to(DEV))
    check(got, *single(c, q, cap=4.0, slopes=slopes)[:2])


@pytest.mark.parametrize("rule", ["cap", "slopes", "first", "weights", "scale"])
@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (7, 1, 64), (24, 1, 80), (2, 2, 256)])
def test_each_rule(jy, rule, pool, nh, nkv, hd):
    lens = [1, 70, 0, 1500]
    c = Cache(jy, lens, nkv, hd, 16, pool, seed=hd)
    q = 2 * torch.randn((4, nh, hd), generator=gen(2))
    kw, mine = {}, {}
    if rule == "cap":
        kw = mine = dict(cap=0.7)
    if rule == "slopes":
        mine = dict(slopes=torch.rand(nh, generator=gen(1)) * 0.1)
        kw = dict(slopes=mine["slopes"].to(DEV))
    if rule == "scale":
        kw = mine = dict(scale=-0.05)
    if rule == "first":
        first = [0, 33, 5, 1471]
        kw, mine = dict(first=ints(first)), dict(first=first)
    if rule == "weights":
        w = torch.rand((4, nkv, 1600), generator=gen(9))
        kw = dict(weights=w.to(DEV))
    got = c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 1500, **kw)
    want, room, p, pr = single(c, q, **mine)
    check(got, want, room)
    if rule == "weights":
        for b, n in enumerate(lens):
            add, far = (t.view(nkv, nh // nkv, n).sum(1) for t in (p[b], pr[b]))
            want_w = w[b].double().clone()
            want_w[:, :n] += add
            off = (kw["weights"][b].double().cpu() - want_w).abs()
            limit = 2.0**-24 * want_w.abs()
            limit[:, :n] += far + 2.0**-24 * (nh // nkv) * add
            assert (off <= limit).all() and torch.equal(kw["weights"][b, :, n:].cpu(), w[b, :, n:])


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("window", [1, 2, 15, 16, 31, 32, 33, 64, 100, 1000, 1025, 3000])
def test_windows(jy, pool, window):
    """positions in front of a window are left out, whatever they hold; their pages may be gone; weights beside"""
    lens = [2900, 1, 64, 33, window]
    c = Cache(jy, lens, 2, 64, 16, pool, seed=window)
    first = [max(0, n - window) for n in lens]
    t = c.tables.clone()
    for b, f in enumerate(first):
        t[b, :f // 16] = [-1, 1 << 30][b % 2]  # whole pages before the window: given back
        for j in range(f // 16 * 16, f):  # the rest of its first page: anything
            pg = int(t[b, j // 16])
            for s in (c.pool.k_scale, c.pool.v_scale):
                if s is not None:
                    s[c.layer, pg, :, j % 16] = math.nan if j % 2 else 60000.0
            if pool in ("f16", "bf16"):
                c.pool.k[c.layer, pg, :, j % 16] = math.inf
                c.pool.v[c.layer, pg, :, j % 16] = math.nan if j % 2 else -math.inf
    q = torch.randn((5, 4, 64), generator=gen(2))
    w = torch.zeros((5, 2, max(lens)), device=DEV)
    for kw in ({}, dict(weights=w)):
        got = c.pool.attend(c.layer, q.to(DEV), t.to(DEV), c.dlens, window, first=ints(first), **kw)
        want, room, p, pr = single(c, q, first=first)
        check(got, want, room)
    for b, n in enumerate(lens):
        add, far = (x.view(2, 2, n).sum(1) for x in (p[b], pr[b]))
        assert ((w[b, :, :n].double().cpu() - add).abs() <= far + 2.0**-22 * add).all() and not w[b, :, n:].any()


def test_window_cut_by_max_len(jy):
    """of more positions than max_len the first max_len count; none with 0; short weights"""
    c = Cache(jy, [100, 50], 1, 64, 16, "i4", seed=3)
    q = torch.randn((2, 2, 64), generator=gen(2))
    for m in (0, 1, 40, 99):
        first = [7, 45]
        w = torch.zeros((2, 1, 20), device=DEV)
        got = c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, m, first=ints(first), weights=w)
        want, room, p, pr = single(c, q, first=first, max_len=m)
        check(got, want, room)
        assert ((w[0, 0].double().cpu() - p[0].sum(0)[:20]).abs() <= pr[0].sum(0)[:20] + 1e-6).all() and not w[1].any()


def test_holes_negative_lengths_and_odd_firsts(jy):
    for pool in POOL:
        c = Cache(jy, [70, 100, 33, 48], 2, 64, 16, pool, seed=8)
        t = c.tables.clone()
        gone = {0: [0], 1: [3, 6], 2: [0, 1, 2]}
        for b, pages in gone.items():
            for i, pg in enumerate(pages):
                t[b, pg] = [-1, 1 << 30, -(1 << 31)][i % 3]
        live = [torch.tensor([p // 16 not in gone.get(b, []) for p in range(n)]) for b, n in enumerate(c.lens)]
        q = torch.randn((4, 4, 64), generator=gen(3))
        w = torch.zeros((4, 2, 112), device=DEV)
        n = ints([70, 100, 33, -5])
        got = c.pool.attend(c.layer, q.to(DEV), t.to(DEV), n, 100, cap=5.0, weights=w)
        for x in ("k", "v", "ka", "va"):
            setattr(c, x, [y[m] for y, m in zip(getattr(c, x), live)])
        c.lens = [int(m.sum()) for m in live[:3]] + [0]
        c.k[3], c.v[3], c.ka[3], c.va[3] = (y[:0] for y in (c.k[3], c.v[3], c.ka[3], c.va[3]))
        check(got, *single(c, q, cap=5.0)[:2])
        assert not got[2:].any() and not w[2:].any()
        assert not w[0, :, :16].any() and not w[1, :, 48:64].any() and (w[0, :, 16:70] > 0).all()
        # a first behind the end, before 0, and at the ends of int
        q1 = q[:1].repeat(4, 1, 1)
        got = c.pool.attend(c.layer, q1.to(DEV), t[[0, 0, 0, 0]].to(DEV), ints([70, 70, 70, -(1 << 31)]), 100,
                            first=ints([(1 << 31) - 1, -(1 << 31), 70, 0]))
        assert not got[[0, 2, 3]].any() and got[1].any()


MASKS = ["causal", "prefix", "documents", "window", "mixed"]


def bounds(mask, pos, n, rng):
    first, last = [0] * len(pos), [p + 1 for p in pos]
    if mask == "prefix":
        last = [max(p + 1, n // 2) for p in pos]
    if mask == "documents":
        first = [p // 37 * 37 for p in pos]
    if mask == "window":
        first = [max(0, p - 20) for p in pos]
    if mask == "mixed":  # rows that see nothing, one position, everything, a piece in the middle
        for i, p in enumerate(pos):
            a, b = sorted((int(rng[i]) % (n + 1), int(rng[i] * 7) % (n + 1)))
            first[i], last[i] = [(a, b), (5, 5), (p, p + 1), (0, n), (9, 3), (-4, n)][i % 6]
    return first, last


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (7, 1, 128), (20, 1, 80), (3, 3, 256)])
def test_runs(jy, mask, pool, io, nh, nkv, hd):
    """runs of 0 to 70 rows over earlier positions, every mask; rows in no run stay"""
    new, past = [3, 0, 70, 1, 17], [0, 9, 40, 130, 15]
    lens = [a + b for a, b in zip(new, past)]
    c = Cache(jy, lens, nkv, hd, 16, pool, seed=hd + nh)
    total = sum(new)
    lead, rest = 2, 3
    q = torch.randn((lead + total + rest, nh, hd), generator=gen(4)).to(IO[io])
    starts = [lead]
    for a in new:
        starts.append(starts[-1] + a)
    pos, first, last, parts = [0] * lead, [0] * lead, [1] * lead, []
    slopes = torch.rand(nh, generator=gen(1)) * 0.05
    rng = torch.randint(0, 1 << 20, (100,), generator=gen(6))
    for b, (a, p) in enumerate(zip(new, past)):
        at = list(range(p, p + a))
        f, l = bounds(mask, at, lens[b], rng)
        pos, first, last = pos + at, first + f, last + l
        parts.append(attention64(c, b, q[starts[b]:starts[b + 1]], at, f, [min(x, lens[b]) for x in l], cap=6.0, slopes=slopes, io=q.dtype, runs=True))
    pos, first, last = pos + [0] * rest, first + [0] * rest, last + [1] * rest
    out = torch.full_like(q, 5.0).to(DEV)
    kw = {} if mask == "causal" else dict(first=ints(first), last=ints(last))
    c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints(starts), ints(pos), max(lens), out=out, cap=6.0, slopes=slopes.to(DEV), **kw)
    assert (out[:lead] == 5.0).all() and (out[lead + total:] == 5.0).all()
    check(out[lead:lead + total], torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]))


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_runs_over_long_caches(jy, pool, io):
    """a few rows each over thousands of positions: chunks joined, and a run past 4096 positions"""
    lens, new = [5000, 1200, 9], [2, 5, 9]
    c = Cache(jy, lens, 1, 64, 64, pool, seed=2)
    q = torch.randn((16, 4, 64), generator=gen(4)).to(IO[io])
    starts, pos = [0, 2, 7, 16], [i for n, a in zip(lens, new) for i in range(n - a, n)]
    parts = [attention64(c, b, q[starts[b]:starts[b + 1]], pos[starts[b]:starts[b + 1]], [0] * new[b],
                         [p + 1 for p in pos[starts[b]:starts[b + 1]]], io=q.dtype, runs=True) for b in range(3)]
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints(starts), ints(pos), 5000)
    check(got, torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]))


def test_a_long_prompt_in_fp32(jy):
    """groups that fill the chip are not cut: one goes through more than 4096 positions"""
    c = Cache(jy, [4500], 1, 16, 256, "bf16", seed=2)
    q = torch.randn((4500, 16, 16), generator=gen(4))
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, 4500]), ints(list(range(4500))), 4500)
    at = [0, 1, 31, 32, 2047, 4095, 4096, 4097, 4499]
    want, room, _, _ = attention64(c, 0, q[at], at, [0] * 9, [a + 1 for a in at])
    check(got[at], want, room)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,lens,new", [(32, 8, 128, [700], [700]), (4, 4, 64, [300, 129, 64], [300, 129, 1]), (24, 1, 80, [90, 65], [90, 3]),
                                                (6, 3, 96, [3000], [200]), (8, 1, 256, [260], [260]), (14, 2, 64, [1000], [1]),
                                                (150, 1, 16, [40, 70], [40, 7]), (2, 1, 240, [70], [66]), (28, 4, 128, [513, 5], [100, 5])])
@pytest.mark.parametrize("rules", [False, True])
def test_prompts(jy, pool, io, nh, nkv, hd, lens, new, rules):
    """runs that fill the matrix products' columns, and some that do not"""
    c = Cache(jy, lens, nkv, hd, 32, pool, seed=hd + nh)
    total = sum(new)
    q = torch.randn((total, nh, hd), generator=gen(4)).to(IO[io])
    starts, pos = [0], [i for n, a in zip(lens, new) for i in range(n - a, n)]
    for a in new:
        starts.append(starts[-1] + a)
    slopes = torch.rand(nh, generator=gen(1)) * 0.05
    kw, mine = {}, {}
    first = [max(0, p - 77) if rules else 0 for p in pos]
    if rules:
        kw, mine = dict(cap=5.0, slopes=slopes.to(DEV), first=ints(first)), dict(cap=5.0, slopes=slopes)
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints(starts), ints(pos), max(lens), **kw)
    for b in range(len(lens)):
        a, e = starts[b], starts[b + 1]
        some = sorted({a, e - 1, *range(a, e, max(1, (e - a) // 40))})  # (rows all over the run)
        want, room, _, _ = attention64(c, b, q[some], [pos[r] for r in some], [first[r] for r in some], [pos[r] + 1 for r in some],
                                       io=q.dtype, runs=True, **mine)
        check(got[some], want, room)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
def test_runs_over_holes(jy, pool, io):
    """pages that do not exist are left out of a run's attention, and a run over nothing but holes gives zeros"""
    lens = [150, 40]
    c = Cache(jy, lens, 2, 64, 16, pool, seed=3)
    t = c.tables.clone()
    gone = {0: [0, 3, 4, 8], 1: [0, 1, 2]}
    for b, pages in gone.items():
        for i, pg in enumerate(pages):
            t[b, pg] = [-1, 1 << 30, -(1 << 31)][i % 3]
    q = torch.randn((190, 8, 64), generator=gen(4)).to(IO[io])
    pos = list(range(150)) + list(range(40))
    got = c.pool.attend_rows(c.layer, q.to(DEV), t.to(DEV), ints([0, 150, 190]), ints(pos), 150)
    live = torch.tensor([p // 16 not in gone[0] for p in range(150)])
    for x in ("k", "v", "ka", "va"):
        getattr(c, x)[0] = getattr(c, x)[0][live]
    last = [int(live[:p + 1].sum()) for p in range(150)]
    want, room, _, _ = attention64(c, 0, q[:150], pos[:150], [0] * 150, last, io=q.dtype, runs=True)
    check(got[:150], want, room)
    assert not got[:16].any() and not got[150:].any()


@pytest.mark.parametrize("pool", ["f16", "bf16", "i8", "i4"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(jy, pool, io):
    n = 70
    c = Cache(jy, [n], 2, 64, 16, pool, seed=5)
    q = torch.randn((n, 4, 64), generator=gen(4)).to(IO[io])
    clean = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), ints(list(range(n))), n)
    bad = {20: math.inf, 33: -math.inf, 47: math.nan}
    for j, x in bad.items():
        k = torch.randn((1, 2, 64), generator=gen(j)).to(DEV)
        v = torch.randn((1, 2, 64), generator=gen(j + 1)).to(DEV)
        v[0, 1, 11 if pool in ("f16", "bf16") else slice(None)] = x
        c.pool.write(c.layer, k, v, c.dtables, ints([j]))
        kk, vv = c.pool.read(c.layer, c.dtables, ints([j]))
        c.k[0][j], c.v[0][j] = kk[0].double().cpu(), vv[0].double().cpu()
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), ints(list(range(n))), n)
    assert torch.equal(got[:20], clean[:20])
    # kv head 0 never reads one, nor do dims but 11 of 16-bit values
    assert torch.isfinite(got[:, :2]).all()
    hit = torch.zeros((n, 2, 64), dtype=torch.bool)
    hit[20:, :, 11 if pool in ("f16", "bf16") else slice(None)] = True
    assert torch.equal(~torch.isfinite(got[:, 2:]).cpu(), hit)
    if pool in ("f16", "bf16"):
        assert (got[20:33, 2:, 11] == math.inf).all() and torch.isnan(got[47:, 2:, 11]).all()


def test_scores_that_are_not_finite(jy):
    """an infinite key: its rows' scores by the formula, capped ones stay finite"""
    c = Cache(jy, [40], 1, 64, 16, "bf16", seed=5)
    c.pool.k[c.layer, int(c.tables[0, 1]), 0, 3, 0] = math.inf  # position 19
    q = torch.rand((40, 1, 64), generator=gen(4)) + 0.5
    run = lambda **kw: c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, 40]), ints(list(range(40))), 40, **kw)  # noqa: E731
    a = run()
    assert torch.isfinite(a[:19]).all() and torch.isnan(a[19:]).all()
    b = run(cap=2.0)
    assert torch.isfinite(b).all()
    c.k[0][19, 0, 0] = 1e9  # a tanh of 1 all the same
    want, _, _, _ = attention64(c, 0, q, list(range(40)), [0] * 40, [i + 1 for i in range(40)], cap=2.0)
    assert (b.double().cpu() - want).abs().max() < 1e-4


def test_queries_that_are_not_finite(jy):
    c = Cache(jy, [40, 20], 2, 64, 16, "i4", seed=5)
    q = torch.randn((2, 4, 64), generator=gen(4))
    q[0, 1, 3], q[1, 2, 0] = math.inf, math.nan
    got = c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 40).cpu()
    bad = torch.isnan(got).all(-1)
    assert bad.tolist() == [[False, True, False, False], [False, False, True, False]] and torch.isfinite(got[~bad]).all()


@pytest.mark.parametrize("size", [1e-7, 1e-3, 5e3])
@pytest.mark.parametrize("io", list(IO))
def test_4bit_values_of_any_size(jy, size, io):
    """steps far from one, groups of very different ranges, constant groups"""
    c = Cache(jy, [90], 1, 128, 16, "i4", seed=11)
    g = gen(3)
    k, v = torch.randn((90, 1, 128), generator=g), torch.randn((90, 1, 128), generator=g) * size
    v[:, :, 32:64] *= 1e-3
    v[:, :, 64:96] = size * 1.5
    k[:, :, 96:] = 0.25
    c.pool.write(c.layer, k.to(DEV), v.to(DEV), c.dtables, ints(list(range(90))), ints([0] * 90))
    k, v = (t.double().cpu() for t in c.pool.read(c.layer, c.dtables, ints(list(range(90))), ints([0] * 90)))
    c.k, c.v, c.ka, c.va = [k], [v], [3 * k.abs().amax(-1, keepdim=True).expand_as(k)], [3 * v.abs().amax(-1, keepdim=True).expand_as(v)]
    q = torch.randn((1, 4, 128), generator=gen(2)).to(IO[io])
    check(c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 90), *single(c, q)[:2])


@pytest.mark.parametrize("io", ["f16", "bf16"])
@pytest.mark.parametrize("pool", list(POOL))
def test_strides_of_prompts(jy, io, pool):
    """heads that do not start at multiples of 16 bytes"""
    c = Cache(jy, [70], 2, 48, 16, pool, seed=10)
    fused = torch.randn((70, 6, 51), generator=gen(3)).to(IO[io]).to(DEV)
    q = fused[:, 1:5, 1:49]
    buf = torch.full((72, 4, 60), 7.0, dtype=IO[io], device=DEV)
    out = buf[1:71, :, 3:51]
    c.pool.attend_rows(c.layer, q, c.dtables, ints([0, 70]), ints(list(range(70))), 70, out=out)
    want, room, _, _ = attention64(c, 0, q.cpu(), list(range(70)), [0] * 70, [i + 1 for i in range(70)], io=q.dtype, runs=True)
    check(out, want, room)
    left = buf.clone()
    left[1:71, :, 3:51] = 7.0
    assert (left == 7.0).all()


@pytest.mark.parametrize("io", list(IO))
def test_strides(jy, io):
    """q a part of a fused projection's rows, out a transposed buffer; what lies between stays"""
    c = Cache(jy, [50, 3], 2, 48, 16, "i4", seed=10)
    fused = torch.randn((2, 6, 51), generator=gen(3)).to(IO[io]).to(DEV)
    q = fused[:, 1:5, 1:49]
    buf = torch.full((7, 2, 60), 7.0, dtype=IO[io], device=DEV)
    out = buf[2:6, :, 3:51].permute(1, 0, 2)
    assert c.pool.attend(c.layer, q, c.dtables, c.dlens, 50, out=out, cap=9.0) is out
    check(out, *single(c, q.cpu(), cap=9.0)[:2])
    left = buf.clone()
    left[2:6, :, 3:51] = 7.0
    assert (left == 7.0).all()


@pytest.mark.parametrize("pool", ["i4", "bf16"])
def test_another_stream_and_replayed_graphs(jy, pool):
    """two captured calls of different shapes, each with its workspace, replayed beside eager ones"""
    c = Cache(jy, [1500, 700], 2, 64, 32, pool, seed=12)
    q1, q2 = torch.randn((2, 4, 64), generator=gen(1)).to(DEV), torch.randn((9, 4, 64), generator=gen(2)).to(DEV).bfloat16()
    starts, pos = ints([0, 4, 9]), ints([1496, 1497, 1498, 1499, 695, 696, 697, 698, 699])
    w = torch.zeros((2, 2, 1500), device=DEV)
    one = lambda **kw: c.pool.attend(c.layer, q1, c.dtables, c.dlens, 1500, cap=3.0, **kw)  # noqa: E731
    two = lambda **kw: c.pool.attend_rows(c.layer, q2, c.dtables, starts, pos, 1500, **kw)  # noqa: E731
    s = torch.cuda.Stream()
    a = one()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = one()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b)
    o1, o2 = torch.empty_like(q1), torch.empty_like(q2)
    two()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one(out=o1, weights=w)
        two(out=o2)
    w.zero_()
    total = torch.zeros_like(w)
    for i in range(4):
        q1.mul_(1.1)
        q2.neg_()
        g.replay()
        torch.cuda.synchronize()
        step = torch.zeros_like(w)
        assert torch.equal(o1, one(weights=step)) and torch.equal(o2, two())
        total += step
        assert torch.equal(w, total)


def test_no_rows(jy):
    c = Cache(jy, [5], 2, 64, 16, "i4", seed=12)
    e = torch.empty((0, 4, 64), device=DEV)
    assert c.pool.attend_rows(c.layer, e, c.dtables, ints([0, 0]), ints([]), 5).shape == (0, 4, 64)


@pytest.mark.parametrize("pool", ["i4", "bf16"])
@pytest.mark.parametrize("first", [0, (1 << 30) - 4096, (1 << 30) - 100])
def test_windows_at_the_far_end(jy, pool, first):
    """a window near position 2^30 with bounds as large: positions and pieces whose sum passes 31 bits"""
    n = 1 << 30
    p = jy.PagePool.empty(1, 2, 256, 1, 64, dtype=POOL[pool], device=DEV)
    t = torch.full((1, n // 256), -1, dtype=torch.int32, device=DEV)
    t[0, -1], t[0, 3] = 1, 0
    g = gen(3)
    k, v = (torch.randn((2, 1, 64), generator=g).to(DEV) for _ in range(2))
    for pg in range(2):
        p.k[0, pg], p.v[0, pg] = 0, 0
        if p.k_scale is not None:
            p.k_scale[0, pg], p.v_scale[0, pg] = 0, 0
    where, zero = ints([n - 1, 800]), ints([0, 0])
    p.write(0, k, v, t, where, seq=zero)
    kk, vv = p.read(0, t, where, seq=zero)
    q = torch.randn((1, 1, 64), generator=g).to(DEV)
    seen = 512 if first == 0 else min(n - first, 256)  # (all the rest are holes)
    s = torch.zeros(seen, dtype=torch.float64)
    s[0] = (q[0, 0].double() @ kk[0, 0].double()).cpu() / 8
    if first == 0:
        s[1] = (q[0, 0].double() @ kk[1, 0].double()).cpu() / 8
    w = torch.softmax(s, 0)
    want = w[0] * vv[0, 0].double().cpu() + (w[1] * vv[1, 0].double().cpu() if first == 0 else 0)
    rows = q.expand(1, 1, 64).contiguous()
    # (a sum of two products, whose weights are off by 2^-20 of 1 at scores of a few: far under 1e-5 of values of a few)
    for got in (p.attend(0, rows, t, ints([n]), n, first=ints([first])),
                p.attend_rows(0, rows, t, ints([0, 1]), ints([n - 1]), n, first=ints([first]))):
        assert (got[0, 0].double().cpu() - want).abs().max() < 1e-5
