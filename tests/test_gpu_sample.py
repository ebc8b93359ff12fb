"""Sampling with temperature, top-k, top-p and min-p against its definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def jy():
    import jieyu_amd
    if jieyu_amd.device_count() < 1:
        pytest.fail("no HIP device visible")
    return jieyu_amd


def pick64(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """(ids that the definition allows) for one row.  The kernel holds masses in steps of at least
    2^-40 of the largest, each off by half a step, and its exponential in fp64: a sum of V of them
    is off by V 2^-40 at most, so where a border lies within that of a running sum, either side of
    it is right; elsewhere there is one id."""
    x = x.double()
    ok = x > -math.inf  # (false for NaN)
    if not ok.any():
        return {-1}
    top = x[ok].max()
    first = int(torch.nonzero(x == top)[0])
    if not T > 0:
        return {first}
    e = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / T))
    e = torch.where(ok, e, torch.zeros_like(e))
    if top == math.inf:
        e = (x == top).double()
    order = torch.sort(torch.where(ok, x, torch.full_like(x, -math.inf)), descending=True, stable=True).indices
    es = e[order]
    n = len(x) if k <= 0 else min(k, len(x))
    slack = len(x) * 2.0**-40
    cum = torch.cumsum(es[:n], 0)
    sizes = {n}
    if p < 1:
        want = max(p, 0.0) * float(cum[-1])
        before = cum - es[:n]
        sizes = {max(1, int((before < want + d).sum())) for d in (-slack, slack)}
        if p <= 0:
            sizes = {1}
    got = set()
    u = min(max(u, 0.0), 1 - 2.0**-24) if u == u else 0.0
    for size in sizes:
        keep = torch.zeros_like(ok)
        keep[order[:size]] = True
        keep &= e >= min(m, 1.0)
        c = torch.cumsum(e * keep, 0)
        w = (e * keep) > 2.0**-41
        for d in (-slack, 0.0, slack):
            t = min(max(u * float(c[-1]) + d, 0.0), float(c[-1]))
            hit = torch.nonzero((c > t) & w)
            if len(hit):
                got.add(int(hit[0]))
    return got


def logits(rows, V, seed, io, spread=3.0, step=None):
    g = torch.Generator()
    g.manual_seed(seed)
    x = spread * torch.randn((rows, V), generator=g)
    if step:
        x = torch.round(x / step) * step
    u = torch.rand(rows, generator=g)
    return x.to(IO[io]), u


SETTINGS = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.9, 0.0),
            (1.0, 0, 0.0, 0.0), (1.5, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.05), (1.0, 0, 1.0, 1.0), (2.0, 0, 1.0, 3.0),
            (0.8, 50, 0.95, 0.01), (3.0, 7, 0.6, 0.2), (0.3, 1000, 0.99, 0.0), (1.0, 2000, 0.999, 1e-4), (-1.0, 5, 0.5, 0.5),
            (5.0, 0, 0.97, 0.0), (1e-3, 0, 1.0, 0.0), (1e-6, 3, 0.5, 0.0), (math.inf, 0, 1.0, 0.0), (math.inf, 9, 0.5, 0.0),
            (1.0, 1 << 30, 1.5, -1.0), (1.0, -7, 1.0, 0.0), (math.nan, 3, 0.5, 0.1), (1.0, 0, math.nan, math.nan),
            (20.0, 0, 0.999, 0.0), (1.0, 900, 1.0, 0.0), (1.0, 1024, 1.0, 0.0), (1.0, 1025, 0.9, 0.0)]


def run(jy, x, u, settings):
    f = lambda v, t=torch.float32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    T, k, p, m = (list(c) for c in zip(*settings))
    return jy.sample(x.to(DEV), u.to(DEV), f(T), f(k, torch.int32), f(p), f(m)).cpu().tolist()


def check(jy, x, u, settings):
    got = run(jy, x, u, settings)
    for r, (i, s) in enumerate(zip(got, settings)):
        T, k, p, m = s
        want = pick64(x[r], float(u[r]), T, k, 1.0 if p != p else p, 0.0 if m != m else m)
        assert i in want, f"row {r}, settings {s}, u {float(u[r])}: {i}, not {want}"


@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 100, 255, 257, 1000, 1023, 1025, 4097, 32000, 151936])
def test_sizes_and_settings(jy, io, V):
    x, u = logits(len(SETTINGS), V, V, io)
    check(jy, x, u, SETTINGS)


@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("step", [0.5, 4.0, 100.0])
def test_ties(jy, io, step):
    """many equal logits: the order among them is by index, and a border may fall among them"""
    for V in (70, 5000, 40000):
        x, u = logits(len(SETTINGS), V, V + int(step), io, step=step)
        check(jy, x, u, SETTINGS)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("step", [0.003, 0.03, 0.1, 0.3, 1.0])
def test_large_top_k_with_ties_at_the_border(jy, io, step):
    """the borders of top-k and of top-p within it among one, few and hundreds of equal logits"""
    settings = [(T, k, p, 0.0) for T in (1.0, 4.0) for k in (127, 257, 300, 500, 1000, 1024) for p in (1.0, 0.9375, 0.5)]
    for V in (1500, 30000):
        x, u = logits(len(settings), V, 11, io, step=step)
        check(jy, x, u, settings)


@pytest.mark.parametrize("io,rows", [("f32", 2), ("bf16", 2), ("bf16", 600), ("f16", 70)])
def test_the_longest_rows(jy, io, rows):
    """2^22 logits, by 64 workgroups a row and by as few as there may be"""
    V = 1 << 22
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    x = torch.empty((rows, V), dtype=IO[io], device=DEV).normal_(0.0, 3.0, generator=g)
    u = torch.rand(rows, generator=g, device=DEV)
    settings = [(1.0, 0, 0.9375, 0.0), (0.75, 50, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (1.5, 0, 1.0, 0.03125), (0.5, 1000, 0.5, 0.0), (1.0, 5000, 0.875, 0.0)]
    at = sorted({0, rows - 1})
    for i in range(0, len(settings), len(at)):
        mine = [settings[(r + i) % len(settings)] for r in range(rows)]
        T, k, p, m = (list(c) for c in zip(*mine))
        f = lambda v, t=torch.float32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
        got = jy.sample(x, u, f(T), f(k, torch.int32), f(p), f(m)).cpu()
        for r in at:
            want = pick64(x[r].cpu(), float(u[r]), *mine[r])
            assert int(got[r]) in want, f"row {r}, settings {mine[r]}: {int(got[r])}, not {want}"


def test_all_equal(jy):
    for V in (1, 64, 9001, 152064):
        check(jy, torch.zeros(len(SETTINGS), V), torch.rand(len(SETTINGS)), SETTINGS)


def test_zero_of_either_sign_is_one_value(jy):
    x = torch.full((3, 50), -5.0)
    x[:, 7], x[:, 3] = 0.0, -0.0
    assert run(jy, x, torch.tensor([0.0, 0.9, 0.2]), [(0.0, 0, 1.0, 0.0), (0.1, 1, 1.0, 0.0), (0.1, 2, 0.4, 0.0)]) == [3, 3, 3]


@pytest.mark.parametrize("V", [40, 3000, 50000])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_masked_logits(jy, V, io):
    """masked tokens (-infinity, the type's lowest value, NaN) are never picked; a row of
    infinities and NaN has none"""
    n = len(SETTINGS)
    x, u = logits(n, V, 3, io)
    g = torch.Generator()
    g.manual_seed(1)
    x[torch.rand((n, V), generator=g) < 0.8] = -math.inf
    x[torch.rand((n, V), generator=g) < 0.05] = math.nan
    x[torch.rand((n, V), generator=g) < 0.05] = torch.finfo(IO[io]).min
    check(jy, x, u, SETTINGS)
    x[:] = -math.inf
    x[::2, ::3] = math.nan
    assert run(jy, x, u, SETTINGS) == [-1] * n
    x[:, V // 2] = -3.0
    assert run(jy, x, u, SETTINGS) == [V // 2] * n


@pytest.mark.parametrize("centre", [0.0, 20.0, -20.0, 1e4, -1e8, 1e30, -1e30])
def test_temperatures_far_under_the_logits_spacing(jy, centre):
    """next to a large logit the float before it is many temperatures away: it has no mass"""
    Ts = [1.0, 1e-3, 1e-5, 3e-7, 1e-7, 3e-8, 1e-8, 1e-10, 1e-20, 1e-37, 1e-42]
    for V in (500, 20000):
        settings = [(torch.tensor(T).item(), k, p, m) for T in Ts
                    for k, p, m in ((0, 1.0, 0.0), (0, 1.0, 0.1), (40, 1.0, 0.0), (300, 0.9, 0.0), (0, 0.9, 0.0), (2000, 0.99, 0.0))]
        x, u = logits(len(settings), V, 5, "f32")
        x = (centre + x * max(1.0, abs(centre) * 1e-6)).float()
        check(jy, x, u, settings)


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("centre,spread", [(0.0, 3.0), (0.0, 1e-3), (20.0, 3.0), (-20.0, 3.0), (-3.0, 3.0), (8.0, 0.01), (0.0, 30.0), (-1e4, 900.0)])
def test_long_rows_of_16_bit_logits(jy, io, centre, spread):
    """few values, met many times, of one sign or both; half of one row masked, another mostly zeros"""
    V = 152064
    settings = [(torch.tensor(T).item(), 0, torch.tensor(p).item(), m) for T in (0.3, 1.0, 5.0, 50.0)
                for p, m in ((0.5, 0.0), (0.9, 0.0), (0.99, 0.0), (0.9, 0.02), (1e-4, 0.0))]
    x, u = logits(len(settings), V, 9, io, spread=spread)
    x = (centre + x.float()).to(IO[io])
    x[1::5, ::2] = -math.inf
    x[2::5, 3:] = torch.where(x[2::5, 3:].float().abs() < 2.5 * spread, torch.zeros_like(x[2::5, 3:]), x[2::5, 3:])
    x[3::5, 1::3] = math.nan
    check(jy, x, u, settings)


def test_positive_infinity(jy):
    x, u = logits(len(SETTINGS), 3000, 4, "f32")
    x[:, 100] = x[:, 2000] = math.inf
    check(jy, x, u, SETTINGS)


def test_random_numbers_at_the_ends(jy):
    x, _ = logits(1, 5000, 5, "f32")
    us = [0.0, -1.0, math.nan, 1 - 2.0**-24, 1.0, 2.0, math.inf, 2.0**-149, 0.5]
    for s in SETTINGS:
        check(jy, x.expand(len(us), -1).contiguous(), torch.tensor(us), [s] * len(us))


def test_settings_may_be_left_out(jy):
    x, u = logits(4, 3000, 6, "f32")
    d = x.to(DEV)
    got = jy.sample(d, u.to(DEV)).cpu().tolist()
    assert all(i in pick64(x[r], float(u[r])) for r, i in enumerate(got))
    got = jy.sample(d, u.to(DEV), top_p=torch.full((4,), 0.5, device=DEV)).cpu().tolist()
    assert all(i in pick64(x[r], float(u[r]), p=0.5) for r, i in enumerate(got))


def test_strided_rows_and_given_output(jy):
    x, u = logits(6, 1003, 7, "bf16")
    wide = torch.zeros((6, 1100), dtype=torch.bfloat16, device=DEV)
    wide[:, 3:1006] = x.to(DEV)
    out = torch.full((6,), -9, dtype=torch.int32, device=DEV)
    assert jy.sample(wide[:, 3:1006], u.to(DEV), out=out) is out
    assert all(i in pick64(x[r], float(u[r])) for r, i in enumerate(out.tolist()))
    one = x[:1].to(DEV).expand(3, -1)  # one row of logits, three numbers
    got = jy.sample(one, u[:3].to(DEV)).tolist()
    assert all(i in pick64(x[0], float(u[r])) for r, i in enumerate(got))
    assert jy.sample(wide[:0], u[:0].to(DEV)).shape == (0,)


def test_every_index_is_reached(jy):
    """u on a grid over a small distribution gives each token its share"""
    V = 300
    x, _ = logits(1, V, 8, "f32", spread=1.0)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    got = torch.tensor(run(jy, x.expand(n, -1).contiguous(), u, [(1.0, 0, 1.0, 0.0)] * n))
    assert (got[1:] >= got[:-1]).all()
    share = torch.bincount(got, minlength=V).double() / n
    p = torch.softmax(x[0].double(), 0)
    assert (share - p).abs().max() <= 1.0 / n + 1e-12


def test_same_every_time_and_in_a_graph(jy):
    n = len(SETTINGS)
    x, u = logits(n, 50000, 9, "f32")
    f = lambda v, t=torch.float32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    T, k, p, m = (list(c) for c in zip(*SETTINGS))
    args = [f(T), f(k, torch.int32), f(p), f(m)]
    dx, du = x.to(DEV), u.to(DEV)
    first = jy.sample(dx, du, *args)
    for _ in range(3):
        assert torch.equal(jy.sample(dx, du, *args), first)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(jy.sample(dx, du, *args))
        graphs.append(g)
    for r in range(6):
        x, u = logits(n, 50000, 20 + r, "f32")
        dx.copy_(x)
        du.copy_(u)
        graphs[r % 2].replay()
        torch.cuda.synchronize()
        want = jy.sample(dx.clone(), du.clone(), *args)
        assert torch.equal(outs[r % 2], want), r
    check(jy, x, u, SETTINGS)


def test_two_streams_at_once(jy):
    n = len(SETTINGS)
    data = [logits(n, 30000, 40 + i, "f32") for i in range(2)]
    f = lambda v, t=torch.float32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    T, k, p, m = (list(c) for c in zip(*SETTINGS))
    args = [f(T), f(k, torch.int32), f(p), f(m)]
    dev = [(x.to(DEV), u.to(DEV)) for x, u in data]
    want = [jy.sample(x, u, *args) for x, u in dev]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in dev], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(jy.sample(*dev[i], *args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals(jy):
    x, u = torch.zeros((2, 10), device=DEV), torch.zeros(2, device=DEV)
    with pytest.raises(jy.JyError, match="u must be"):
        jy.sample(x, u[:1])
    with pytest.raises(jy.JyError, match="top_k must be"):
        jy.sample(x, u, top_k=torch.zeros(2, device=DEV))
    with pytest.raises(jy.JyError, match="logits are"):
        jy.sample(x.double(), u)
    with pytest.raises(jy.JyError, match="side by side"):
        jy.sample(x.t().contiguous().t(), u)
    with pytest.raises(jy.JyError, match="vocab"):
        jy.sample(x[:, :0], u)
