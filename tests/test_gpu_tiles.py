"""Runs of 16-bit rows at the ends of their numbers' ranges, rule by rule, and beside single tokens, against the
definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_ruled import DEV, POOL, Cache, attention64, check, gen, ints, jy  # noqa: E402, F401

pytestmark = pytest.mark.gpu

IO16 = {"f16": torch.float16, "bf16": torch.bfloat16}


def room16(c, b, p, room, last, first, far=2.0**-25):
    """The room of 32-bit scores and sums, and what a weight's rounding to the product's type adds: fp16 over fp16 and
    4-bit values (half a step 2^-11; a 4-bit value is one fp16 number, another 2^-11; `far` of the largest weight is where
    fp16 ends), else bf16, 2^-8, or two of them, 2^-16."""
    va, per = c.va[b], p.shape[1] // c.nkv
    out = room.clone()
    for r in range(p.shape[0]):
        lo, hi = max(first[r], 0), last[r]
        for h in range(p.shape[1]):
            v = va[lo:hi, h // per]
            out[r, h] += c.one * (p[r, h, lo:hi] @ v) + (hi - lo) * (far if c.kind in ("f16", "i4") else 2.0**-39) * v.amax()
    return out


def tiles64(c, b, q, pos, first, last, far=2.0**-25, **kw):
    """(want, room): a cap's tanh is off by 8 steps of itself, not of the cap"""
    want, room, p, _ = attention64(c, b, q, pos, first, last, **kw)
    c.one = {"i4": 2.0**-10, "f16": 2.0**-11}.get(c.kind, 2.0**-8 if q.dtype is torch.bfloat16 else 2.0**-16)
    return want, room16(c, b, p, room, last, first, far)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("scale", [2.0**-30, 2.0**-45, -2.0**-30])
def test_queries_so_small_that_scores_are_zeros(jy, pool, scale):
    """tiles that are cut by the diagonal: the factor of such scores is under fp32's smallest number"""
    n = 150
    c = Cache(jy, [n], 2, 64, 16, pool, seed=3)
    q = (torch.randn((n, 8, 64), generator=gen(4)) * 2.0**-120).bfloat16()
    at = list(range(n))
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), ints(at), n, scale=scale)
    check(got, *tiles64(c, 0, q, at, [0] * n, [p + 1 for p in at], scale=scale))


def prompt(jy, pool, io, nh, nkv, hd, n, new, q_size=1.0, first=None, far=2.0**-25, every=7, **kw):
    """a run of `new` rows behind n - new positions under rules, some of its rows against the definition"""
    c = Cache(jy, [n], nkv, hd, 32, pool, seed=hd + n)
    q = (torch.randn((new, nh, hd), generator=gen(4)) * q_size).to(IO16[io])
    pos = list(range(n - new, n))
    lo = [0 if first is None else max(0, p - first) for p in pos]
    mine = dict(kw)
    if kw.get("slopes") is not None:
        kw["slopes"] = kw["slopes"].to(DEV)
    if first is not None:
        kw["first"] = ints(lo)
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, new]), ints(pos), n, **kw)
    some = sorted({0, new - 1, *range(0, new, every)})
    want, room = tiles64(c, 0, q[some], [pos[r] for r in some], [lo[r] for r in some], [pos[r] + 1 for r in some], far=far, **mine)
    check(got[some], want, room)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO16))
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e5, 1e6])
@pytest.mark.parametrize("slopes", [False, True])
def test_large_caps(jy, pool, io, cap, slopes):
    """scores that are a small part of the cap keep their digits, on the diagonal and off it"""
    prompt(jy, pool, io, 8, 2, 64, 300, 200, 2.0, cap=cap, slopes=torch.rand(8, generator=gen(1)) * 0.02 if slopes else None)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO16))
@pytest.mark.parametrize("cap,size", [(30.0, 1.0), (50.0, 1.0), (50.0, 8.0), (6.0, 1.0), (6.0, 2.5), (0.5, 1.0)])
@pytest.mark.parametrize("scale", [None, -0.1])
def test_caps_alone(jy, pool, io, cap, size, scale):
    """scores all within half the cap, some past it, most at it; tiles seen whole among them"""
    prompt(jy, pool, io, 8, 2, 64, 400, 130, size, cap=cap, scale=scale)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
def test_a_value_of_no_weight_that_is_not_finite(jy, pool, io):
    """the rows that see it are NaN all the same, on the diagonal and off it, and no others"""
    n = 200
    c = Cache(jy, [n], 2, 64, 16, pool, seed=5)
    k, v = torch.full((1, 2, 64), -60.0), torch.randn((1, 2, 64), generator=gen(1))
    v[0, 1] = math.nan
    c.pool.write(c.layer, k.to(DEV), v.to(DEV), c.dtables, ints([20]))
    q = torch.ones((n, 8, 64)).to({"f32": torch.float32, **IO16}[io])
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), ints(list(range(n))), n)
    assert torch.isfinite(got[:, :4]).all() and torch.isfinite(got[:20]).all()
    assert torch.isnan(got[20:, 4:]).all()


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("single", [False, True])
def test_caps_at_the_ends_of_their_type(jy, pool, io, single):
    """tiny caps make every weight the same, of queries of any size and of zeros; huge ones change nothing"""
    n = 200
    c = Cache(jy, [n], 2, 64, 16, pool, seed=5)
    dtype = {"f32": torch.float32, **IO16}[io]
    kz = torch.zeros((3, 2, 64))
    c.pool.write(c.layer, kz.to(DEV), torch.ones((3, 2, 64)).to(DEV), c.dtables, ints([4, 90, 150]), ints([0, 0, 0]))
    at = ints(list(range(n)))
    k, v = (t.double().cpu() for t in c.pool.read(c.layer, c.dtables, at, ints([0] * n)))
    c.k[0], c.v[0] = k, v
    c.va[0] = torch.maximum(c.va[0], v.abs())
    size = 1.0 if io == "f16" else 1e30
    rows = [n - 1] if single else list(range(n))

    def run(q, **kw):
        if single:
            return c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, n, **kw)
        return c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), at, n, **kw)

    def mean(scores=None):
        """(want, room) of weights that are all the same, in 32 bits or as one number of 16"""
        want = torch.stack([v[:r + 1].mean(0) for r in rows]).repeat_interleave(4, 1)
        room = torch.stack([c.va[0][:r + 1].mean(0) for r in rows]).repeat_interleave(4, 1)
        # (a 4-bit value is one fp16 number; a weight times an int8 value's scale one bf16 number, or two; weights of 1 are exact)
        one = 2.0**-8 if pool == "i8" else 2.0**-10
        return want, room * ((2 * n + 16) * 2.0**-24 + one)

    for cap, x in ((1e-8, 0.0), (1e-20, 0.0), (1e-8, 1.0), (1e-20, size)):
        q = torch.randn((len(rows), 8, 64), generator=gen(2)).mul(x).to(dtype)
        check(run(q, cap=cap), *mean())
    q = torch.randn((len(rows), 8, 64), generator=gen(3)).to(dtype)
    some = list(range(0, len(rows), 9))
    pos = [rows[r] for r in some]
    for cap in (1e9, 1e19, 1e25, 1e36, 3e38):
        want, room = tiles64(c, 0, q[some], pos, [0] * len(some), [p + 1 for p in pos])
        check(run(q, cap=cap)[some], want, room)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO16))
@pytest.mark.parametrize("below", [15, 20, 26, 30])
def test_many_small_weights_beside_a_large_one(jy, pool, io, below):
    """thousands of positions of 2^-below of the largest weight each, which alone make some dims of the output"""
    n, new, hd = 6000, 40, 64
    c = Cache(jy, [n], 1, hd, 256, pool, seed=2)
    k, v = torch.zeros((n, 1, hd)), torch.zeros((n, 1, hd))
    k[7, 0, 0] = 1.0
    v[:, 0, :32] = torch.rand((n, 32), generator=gen(1)) + 1.0
    v[7, 0, :32], v[7, 0, 32:] = 0.0, 1.0
    at = ints(list(range(n)))
    c.pool.write(c.layer, k.to(DEV), v.to(DEV), c.dtables, at, ints([0] * n))
    c.k[0], c.v[0] = (t.double().cpu() for t in c.pool.read(c.layer, c.dtables, at, ints([0] * n)))
    c.ka[0] = c.k[0].abs()
    c.va[0] = c.v[0].abs()  # (a 4-bit group here: its low 0 or 1, a number times a step of at most 1)
    q = torch.zeros((new, 1, hd))
    q[:, :, 0] = below * math.log(2.0)
    q = q.repeat(1, 4, 1).to(IO16[io])
    pos = list(range(n - new, n))
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, new]), ints(pos), n, scale=1.0)
    some = [0, 1, 17, new - 1]
    want, room = tiles64(c, 0, q[some], [pos[r] for r in some], [0] * 4, [pos[r] + 1 for r in some], far=2.0**-34, scale=1.0)
    # (dims of the small ones alone: the large one's value there is 0, so that `far` counts the small values alone)
    check(got[some], want, room)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO16))
@pytest.mark.parametrize("rule", ["none", "slopes", "first", "scale", "rising"])
def test_each_rule_alone(jy, pool, io, rule):
    """tiles seen whole and tiles that are cut, under one rule at a time"""
    kw = {}
    if rule == "slopes":
        kw = dict(slopes=torch.tensor([0.0, 0.5, -0.01, 0.03, 1.0, 0.002, 0.1, 0.004]))
    if rule == "first":
        kw = dict(first=150)
    if rule == "scale":
        kw = dict(scale=-0.2)
    if rule == "rising":  # the maximum grows from tile to tile
        kw = dict(slopes=torch.full((8,), 0.2))
    prompt(jy, pool, io, 8, 2, 64, 500, 140, 1.5, **kw)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [512, 1000])
def test_a_prompt_beside_single_tokens(jy, pool, io, rows):
    """one prompt and 63 sequences of one new token in a call: whichever kernel the call's average columns choose"""
    g = gen(rows)
    past = [0] + torch.randint(0, 700, (63,), generator=g).tolist()
    new = [rows] + [1] * 63
    lens = [a + b for a, b in zip(past, new)]
    c = Cache(jy, lens, 2, 64, 32, pool, seed=rows)
    q = torch.randn((sum(new), 8, 64), generator=g).to({"f32": torch.float32, **IO16}[io])
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    pos = [i for n, a in zip(lens, new) for i in range(n - a, n)]
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints(starts), ints(pos), max(lens))
    for b in range(64):
        some = list(range(0, rows, 37)) + [rows - 1] if b == 0 else [starts[b]]
        at = [pos[r] for r in some]
        want, room = tiles64(c, b, q[some], at, [0] * len(at), [p + 1 for p in at])
        check(got[some], want, room)
    again = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints(starts), ints(pos), max(lens))
    assert torch.equal(got, again)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("power,cap", [(0, None), (8, None), (14, None), (20, None), (26, None), (50, None), (100, None),
                                       (0, 1e9), (8, 1e9), (14, 1e9)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(jy, pool, io, power, sign, cap):
    """scores far apart and up to 2^114, above or under 0, within a cap: the row is the value of its largest"""
    n = 300
    c = Cache(jy, [n], 1, 64, 32, pool, seed=6)
    a = torch.randperm(n, generator=gen(power)).float() % 150 + 1.0
    k = (sign * a)[:, None, None].expand(n, 1, 64).contiguous()
    v = torch.randn((n, 1, 64), generator=gen(2))
    at = ints(list(range(n)))
    c.pool.write(c.layer, k.to(DEV), v.to(DEV), c.dtables, at, ints([0] * n))
    v = c.pool.read(c.layer, c.dtables, at, ints([0] * n))[1].double().cpu()
    q = torch.ones((n, 4, 64)).to({"f32": torch.float32, **IO16}[io])
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), at, n, scale=2.0**power, cap=cap)
    assert torch.isfinite(got).all()
    # Scores are 64 2^power a: of two that differ the smaller is 1/150 and more below, 64 and more.  Equal ones share; a cap's
    # tanh is off by 8 steps of 2^-24 of a score of 10^8, that is 50, in tiles that are cut and others by different steps, so
    # there equal ones may weigh anything, and the row lies between their values.
    for r in range(n):
        top = (sign * a[:r + 1])
        equal = v[:r + 1][top == top.max()]
        # (at most two share: their weights are the same number; 4-bit values are one fp16 number in tiles)
        limit = (2.0**-9 + {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}.get(q.dtype, 0)) * v[:r + 1].abs().amax()
        if cap:
            limit = limit + (equal.amax(0) - equal.amin(0)) / 2
        assert ((got[r].double().cpu() - equal.mean(0)).abs() <= limit).all(), r


@pytest.mark.parametrize("pool", ["bf16", "i8"])
@pytest.mark.parametrize("below", [0.5, 3.0, 5.5, 7.0])
def test_large_values_of_the_largest_weight(jy, pool, below):
    """a value near the type's largest number that weighs a little more than what came before it"""
    n = 200
    c = Cache(jy, [n], 1, 64, 32, pool, seed=6)
    k, v = torch.zeros((n, 1, 64)), torch.zeros((n, 1, 64))
    k[100, 0, 0] = 1.0
    v[100] = 1e38
    at = ints(list(range(n)))
    c.pool.write(c.layer, k.to(DEV), v.to(DEV), c.dtables, at, ints([0] * n))
    c.k[0], c.v[0] = (t.double().cpu() for t in c.pool.read(c.layer, c.dtables, at, ints([0] * n)))
    c.ka[0], c.va[0] = c.k[0].abs(), c.v[0].abs()
    q = torch.zeros((n, 4, 64))
    q[:, :, 0] = below * math.log(2.0)
    q = q.bfloat16()
    pos = list(range(n))
    got = c.pool.attend_rows(c.layer, q.to(DEV), c.dtables, ints([0, n]), at, n, scale=1.0)
    want, room = tiles64(c, 0, q, pos, [0] * n, [p + 1 for p in pos], scale=1.0)
    check(got, want, room)
