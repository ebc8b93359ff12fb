"""The paged key/value cache and the attention over it against plain implementations in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
POOL = {"i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}
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


def held(x, pool):
    """(values as held, float64; q; scale) of x [..., hd] in the pool's format"""
    if pool != "i8":
        q = x.float().to(POOL[pool])
        return q.double(), q, None
    x = x.float()
    a = x.abs().amax(-1)
    top = torch.full_like(a, 127.0)
    on = a > 1e-8
    inv, s = torch.where(on, top / a, torch.zeros_like(a)), torch.where(on, a / top, torch.zeros_like(a))
    q = torch.round((x * inv[..., None]).clamp(-127, 127)).to(torch.int8)
    bad = ~torch.isfinite(x).all(-1)
    q[bad] = 0
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    return q.double() * s.double()[..., None], q, s


class Cache:
    """A pool on the device and what it holds on the host; pages of the sequences in random order,
    everything outside them set to what must never be read (NaN scales, NaN or huge values)."""

    def __init__(self, jy, lens, nkv, hd, page, pool, seed=1, layers=2, layer=1, spare=2, outliers=True):
        g = gen(seed)
        self.lens, self.nkv, self.hd, self.page, self.kind, self.layer = lens, nkv, hd, page, pool, layer
        need = [-(-max(n, 0) // page) for n in lens]
        self.npages = sum(need) + spare
        width = max(max(need), 1)
        order = torch.randperm(self.npages, generator=g)
        self.tables = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n].int()
            at += n
        shape = (layers, self.npages, nkv, page, hd)
        if pool == "i8":
            self.kq, self.vq = (torch.full(shape, -128, dtype=torch.int8) for _ in range(2))
            self.ks, self.vs = (torch.full(shape[:4], math.nan) for _ in range(2))
        else:
            self.kq, self.vq = (torch.full(shape, math.nan, dtype=POOL[pool]) for _ in range(2))
            self.ks = self.vs = None
        self.k, self.v = [], []  # per sequence [n][nkv][hd] float64
        for b, n in enumerate(lens):
            for name, out in (("k", self.k), ("v", self.v)):
                x = torch.randn((max(n, 0), nkv, hd), generator=g)
                if outliers:
                    x = x * torch.exp(0.5 * torch.randn(hd, generator=g))
                val, q, s = held(x, pool)
                out.append(val)
                for p in range(n):
                    pg, sl = int(self.tables[b, p // page]), p % page
                    getattr(self, name + "q")[layer, pg, :, sl] = q[p]
                    if s is not None:
                        getattr(self, name + "s")[layer, pg, :, sl] = s[p]
        on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        self.pool = jy.PagePool(on(self.kq), on(self.vq), on(self.ks), on(self.vs))
        self.dtables = self.tables.to(DEV)
        self.dlens = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def attend(self, q, max_len=None, **kw):
        return self.pool.attend(self.layer, q, self.dtables, self.dlens, max(self.lens) if max_len is None else max_len, **kw)


def attention64(q, ks, vs, scale):
    """(out, bound): the definition in 64 bits for q [nseq][nh][hd] and each sequence's k, v
    [n][nkv][hd], and the kernels' error bound before the output's own rounding.

    fp32 scores: a query rounded to 2^-24 of its largest element and a sum of hd products in
    fp32 give |ds| <= (hd + 2) 2^-24 S, S = scale * max|q| * sum|k|; the factors (key scale,
    softmax scale, log2 e, the difference to the maximum) at most 6 more roundings of values up to
    2 S.  The weights are then off by 2 |ds| relative (their own and the maximum's or sum's), the
    exponential's 2 steps, a weight carried in 21 bits (2^-21 = 8 * 2^-24), and the sums over n
    positions n 2^-24 each (weights and products).

    A weight far below the largest (1) has no relative accuracy: fp32 ends at 2^-126, and a weight
    carried as two halves scaled by 2^15 at their smallest step, 2^-24 2^-15, rounded by at most
    2^-39 of the largest product weight x value.  A key that takes the row leaves exactly such
    weights, so where its own value is zero the output's error is n 2^-39 max|v| and not relative
    to sum p|v|."""
    out, bound = [], []
    for b, (k, v) in enumerate(zip(ks, vs)):
        nh, hd = q.shape[1:]
        if k.shape[0] == 0:
            out.append(torch.zeros(nh, hd, dtype=torch.float64))
            bound.append(torch.zeros(nh, hd, dtype=torch.float64))
            continue
        per = nh // k.shape[1]
        qq = q[b].double()
        kk, vv = k.repeat_interleave(per, 1).permute(1, 0, 2), v.repeat_interleave(per, 1).permute(1, 0, 2)
        s = (kk @ qq[:, :, None])[..., 0] * scale
        p = torch.softmax(s, -1)
        S = scale * qq.abs().amax(-1) * kk.abs().sum(-1).amax(-1)
        rel = (2 * (hd + 14) * S + 2 * k.shape[0] + 16) * 2.0**-24
        out.append((p[:, None] @ vv)[:, 0])
        far = k.shape[0] * 2.0**-39 * vv.abs().amax(dim=(1, 2))
        bound.append(rel[:, None] * (p[:, None] @ vv.abs())[:, 0] + far[:, None])
    return torch.stack(out), torch.stack(bound)


def check(got, want, bound):
    assert got.dtype in HALF
    # (fp16: values below its normal range have a step of their own)
    tiny = 2.0**-25 if got.dtype is torch.float16 else 0.0
    off = (got.double().cpu() - want).abs()
    room = bound + HALF[got.dtype] * (want.abs() + bound) + tiny
    worst = (off / room.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"error {worst:.3g} of the bound"


SHAPES = [(14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 64), (16, 16, 128), (10, 2, 112), (6, 3, 96), (8, 1, 256),
          (9, 3, 80), (4, 2, 16), (3, 1, 32), (40, 2, 64), (33, 1, 128), (4, 4, 48), (2, 2, 144), (2, 1, 192), (2, 1, 240),
          (64, 1, 160)]


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("pool", list(POOL))
def test_attend_shapes(jy, nh, nkv, hd, pool):
    c = Cache(jy, [1, 37, 0, 130], nkv, hd, 16, pool, seed=nh + hd)
    io = {"i8": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[pool]
    q = torch.randn((4, nh, hd), generator=gen(5)).to(io)
    got = c.attend(q.to(DEV))
    check(got, *attention64(q, c.k, c.v, 1 / math.sqrt(hd)))
    assert not got[2].any()


@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attend_types_and_pages(jy, io, pool, page):
    c = Cache(jy, [page, page + 1, page - 1, 3 * page + 7], 2, 64, page, pool, seed=page)
    q = torch.randn((4, 6, 64), generator=gen(2)).to(IO[io])
    check(c.attend(q.to(DEV)), *attention64(q, c.k, c.v, 0.125))


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [31], [32], [33], [63], [64], [65], [127], [128], [129],
                                  [255], [256], [257], [511], [513], [1023], [1025], [4097], [0], [0, 0, 5], [1, 1, 1, 2000]])
@pytest.mark.parametrize("pool", ["i8", "bf16"])
def test_attend_lengths(jy, lens, pool):
    c = Cache(jy, lens, 2, 128, 32, pool, seed=len(lens) + lens[0])
    q = torch.randn((len(lens), 8, 128), generator=gen(3))
    check(c.attend(q.to(DEV)), *attention64(q, c.k, c.v, 1 / math.sqrt(128)))


def test_attend_long(jy):
    lens = [32769, 7]
    c = Cache(jy, lens, 1, 64, 256, "i8", seed=4, layers=1, layer=0)
    q = torch.randn((2, 7, 64), generator=gen(3))
    check(c.attend(q.to(DEV)), *attention64(q, c.k, c.v, 0.125))


@pytest.mark.parametrize("max_len", [0, 1, 50, 64, 300, 10000])
def test_attend_cut_to_max_len_and_to_the_table(jy, max_len):
    """a longer length is cut to max_len; positions past the table do not exist"""
    lens = [100, 20, 200]
    c = Cache(jy, lens, 2, 64, 16, "i8", seed=6)
    dl = torch.tensor([100, 20, 1 << 30], dtype=torch.int32, device=DEV)
    q = torch.randn((3, 4, 64), generator=gen(3))
    # the third table ends after 200 positions (13 pages hold 208; the last 8 slots are NaN), so cut it at 12 pages
    t = c.dtables[:, :12].contiguous()
    got = c.pool.attend(c.layer, q.to(DEV), t, dl, max_len)
    n = [min(100, max_len), min(20, max_len), min(192, max_len)]
    check(got, *attention64(q, [k[:m] for k, m in zip(c.k, n)], [v[:m] for v, m in zip(c.v, n)], 0.125))


@pytest.mark.parametrize("pool", list(POOL))
def test_attend_holes(jy, pool):
    """pages that do not exist are left out, wherever they lie; all of them: zeros"""
    lens = [70, 100, 33, 48, 200]
    c = Cache(jy, lens, 2, 64, 16, pool, seed=8)
    t = c.tables.clone()
    gone = {0: [0], 1: [3, 6], 2: [0, 1, 2], 3: [1], 4: list(range(1, 12))}
    for b, pages in gone.items():
        for i, pg in enumerate(pages):
            t[b, pg] = [-1, c.npages, 1 << 30, -(1 << 31)][i % 4]
    live = [torch.tensor([p // 16 not in gone[b] for p in range(n)]) for b, n in enumerate(lens)]
    q = torch.randn((5, 4, 64), generator=gen(3))
    got = c.pool.attend(c.layer, q.to(DEV), t.to(DEV), c.dlens, 200)
    check(got, *attention64(q, [k[m] for k, m in zip(c.k, live)], [v[m] for v, m in zip(c.v, live)], 0.125))
    assert not got[2].any()


def test_attend_negative_lengths_and_shared_pages(jy):
    c = Cache(jy, [40, 90], 2, 64, 32, "i8", seed=9)
    t = torch.stack([c.tables[1], c.tables[0], c.tables[1]]).to(DEV)  # two sequences over the same pages
    q = torch.randn((3, 4, 64), generator=gen(3))
    n = torch.tensor([90, -5, 64], dtype=torch.int32, device=DEV)
    got = c.pool.attend(c.layer, q.to(DEV), t, n, 90)
    z = c.k[0][:0]
    check(got, *attention64(q, [c.k[1], z, c.k[1][:64]], [c.v[1], z, c.v[1][:64]], 0.125))


@pytest.mark.parametrize("io", list(IO))
def test_attend_strides(jy, io):
    """q a part of a fused projection's rows, out a transposed buffer; what lies between stays"""
    c = Cache(jy, [50, 3], 2, 48, 16, "i8", seed=10)
    fused = torch.randn((2, 5 + 1, 51), generator=gen(3)).to(IO[io]).to(DEV)
    q = fused[:, 1:5, 1:49]
    buf = torch.full((7, 2, 60), 7.0, dtype=IO[io], device=DEV)
    out = buf[2:6, :, 3:51].permute(1, 0, 2)
    assert c.attend(q, out=out) is out
    check(out, *attention64(q.cpu(), c.k, c.v, 1 / math.sqrt(48)))
    left = buf.clone()
    left[2:6, :, 3:51] = 7.0
    assert (left == 7.0).all()


@pytest.mark.parametrize("pool,size", [("i8", 1e-30), ("i8", 1e30), ("f16", 1e-6), ("f16", 3e4), ("bf16", 1e-30), ("bf16", 1e25)])
def test_attend_scales_far_from_one(jy, pool, size):
    """values and queries of any size: the scores stay moderate, the outputs are of the values' size"""
    c = Cache(jy, [100], 1, 64, 16, pool, seed=11)
    if pool == "i8":
        vs, ks = c.vs * size, c.ks / size
        c.pool = jy.PagePool(c.pool.k, c.pool.v, ks.to(DEV), vs.to(DEV))
        v, k = [x * size for x in c.v], [x / size for x in c.k]
        # (fp32 rounds the scales once more)
        k = [(c.kq.double() * ks.double()[..., None])[c.layer, c.tables[0].long()].permute(1, 0, 2, 3).reshape(1, -1, 64)[:, :100].permute(1, 0, 2)]
        v = [(c.vq.double() * vs.double()[..., None])[c.layer, c.tables[0].long()].permute(1, 0, 2, 3).reshape(1, -1, 64)[:, :100].permute(1, 0, 2)]
        q = torch.randn((1, 4, 64), generator=gen(3)) * size
    else:
        vq = (c.vq.float() * (size / (8 if pool == "f16" and size > 1 else 1))).to(POOL[pool]) if size > 1 else (c.vq.float() * size).to(POOL[pool])
        c.pool = jy.PagePool(c.pool.k, vq.to(DEV))
        k = c.k
        v = [vq.double()[c.layer, c.tables[0].long()].permute(1, 0, 2, 3).reshape(1, -1, 64)[:, :100].permute(1, 0, 2)]
        q = torch.randn((1, 4, 64), generator=gen(3))
    got = c.pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 100)
    check(got, *attention64(q, k, v, 0.125))


@pytest.mark.parametrize("pool", ["i8", "bf16"])
def test_attend_peaked(jy, pool):
    """scores far apart: one key takes the row, wherever it lies; equal keys share it"""
    n = 700
    for at in (0, 31, 32, 350, n - 1):
        c = Cache(jy, [n], 1, 64, 16, pool, seed=12, outliers=False)
        q = (c.k[0][at, 0] * 4).float()[None, None]
        got = c.attend(q.to(DEV).contiguous(), scale=1.0)
        check(got, *attention64(q, c.k, c.v, 1.0))
    zero = torch.zeros((1, 1, 64))
    check(c.attend(zero.to(DEV)), *attention64(zero, c.k, c.v, 1.0))  # a mean of the values


@pytest.mark.parametrize("n", [2, 40, 3000])
def test_attend_scores_near_the_types_lowest(jy, n):
    """finite scores down to fp32's lowest value have weight: equal ones the same"""
    k = torch.zeros((1, (n + 255) // 256, 1, 256, 64), dtype=torch.bfloat16)
    v = torch.randn(k.shape, generator=gen(3)).to(torch.bfloat16)
    k[..., 0] = 2.0**63
    q = torch.zeros((1, 3, 64))
    q[..., 0] = torch.tensor([-1.3 * 2.0**64, -1.0, 0.0])
    pool = jy.PagePool(k.to(DEV), v.to(DEV))
    tables = torch.arange(k.shape[1], dtype=torch.int32, device=DEV)[None]
    got = pool.attend(0, q.to(DEV), tables, torch.tensor([n], dtype=torch.int32, device=DEV), n, scale=1.0)
    x = v[0, :, 0].reshape(-1, 64)[:n].double()
    # equal weights of exactly 1: the sums' n steps of fp32, one division
    room = (n + 1) * 2.0**-24 * x.abs().mean(0)
    assert ((got[0].double().cpu() - x.mean(0)).abs() <= room).all()


def test_attend_max_len_is_checked(jy):
    c = Cache(jy, [5], 1, 64, 16, "i8")
    q = torch.zeros((1, 1, 64), device=DEV)
    for n in (-1, (1 << 30) + 1, 1 << 32):
        with pytest.raises(jy.JyError, match="max_len"):
            c.attend(q, max_len=n)


def test_attend_nan_and_infinity_reach_their_own_rows_only(jy):
    c = Cache(jy, [40, 40, 40], 2, 64, 16, "i8", seed=13)
    q = torch.randn((3, 4, 64), generator=gen(3))
    q[0, 1, 7] = math.nan
    q[1, 2, 9] = math.inf
    got = c.attend(q.to(DEV)).cpu()
    bad = torch.zeros(3, 4, dtype=torch.bool)
    bad[0, 1] = bad[1, 2] = True
    assert torch.isnan(got[bad]).all()
    assert torch.isfinite(got[~bad]).all()
    # a held NaN reaches the heads that read it, of that sequence alone
    q = torch.randn((3, 4, 64), generator=gen(3))
    ks = c.pool.k_scale.clone()
    ks[c.layer, int(c.tables[1, 1]), 0, 3] = math.nan
    got = jy.PagePool(c.pool.k, c.pool.v, ks, c.pool.v_scale).attend(c.layer, q.to(DEV), c.dtables, c.dlens, 40).cpu()
    assert torch.isnan(got[1, :2]).all() and torch.isfinite(got[1, 2:]).all() and torch.isfinite(got[[0, 2]]).all()


def test_attend_is_the_same_every_time(jy):
    c = Cache(jy, [3000, 1, 77], 2, 128, 32, "i8", seed=14)
    q = torch.randn((3, 8, 128), generator=gen(3)).to(DEV)
    first = c.attend(q)
    for _ in range(5):
        assert torch.equal(c.attend(q), first)
    # a sequence's rows do not depend on what else is in the batch, given the launch's max_len
    one = c.pool.attend(c.layer, q[2:], c.dtables[2:].contiguous(), c.dlens[2:].contiguous(), 3000)
    check(one, *attention64(q[2:].cpu(), c.k[2:], c.v[2:], 1 / math.sqrt(128)))


# ---------------------------------------------------------------- writing and reading

def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("nkv,hd,page", [(2, 64, 16), (8, 128, 32), (1, 256, 16), (3, 80, 64), (2, 112, 16), (1, 16, 256), (5, 144, 32)])
def test_write_and_read(jy, pool, io, nkv, hd, page):
    g = gen(hd)
    c = Cache(jy, [100, 40], nkv, hd, page, pool, seed=20)
    before = {n: getattr(c.pool, n).clone() for n in ("k", "v", "k_scale", "v_scale") if getattr(c.pool, n) is not None}
    rows = 37
    seq = torch.randint(0, 2, (rows,), generator=g)
    pos = torch.stack([torch.randperm(100, generator=g)[:rows], torch.randperm(40, generator=g)[:rows]])[seq, torch.arange(rows)]
    skip = torch.tensor([3, 9, 11, 20])
    seqs, poss = seq.clone(), pos.clone()
    poss[3], poss[9], seqs[11], seqs[20] = -1, 1 << 30, -1, 2
    k, v = (torch.randn((rows, nkv, hd), generator=g) * 3 for _ in range(2))
    k[0], v[1], k[2, 0, 0] = 0.0, 1e-9, 60.0
    k[4] = torch.randint(-127, 128, (nkv, hd), generator=g).float()  # (whole steps and ties of them)
    k[5] = torch.randint(-254, 255, (nkv, hd), generator=g).float() / 2
    k, v = k.to(IO[io]), v.to(IO[io])
    di = lambda t: t.to(torch.int32).to(DEV)  # noqa: E731
    c.pool.write(c.layer, k.to(DEV), v.to(DEV), c.dtables, di(poss), di(seqs))
    keep = torch.ones(rows, dtype=torch.bool)
    keep[skip] = False
    want = {n: t.clone() for n, t in before.items()}
    for name, x in (("k", k), ("v", v)):
        _, q, s = held(x, pool)
        for r in torch.nonzero(keep).flatten().tolist():
            pg, sl = int(c.tables[seq[r], pos[r] // page]), int(pos[r]) % page
            want[name][c.layer, pg, :, sl] = q[r].to(DEV)
            if s is not None:
                want[name + "_scale"][c.layer, pg, :, sl] = s[r].to(DEV)
    for n, t in want.items():  # every byte, those that no row names included
        assert torch.equal(bits(getattr(c.pool, n)), bits(t)), n
    for out in IO.values():
        rk, rv = c.pool.read(c.layer, c.dtables, di(poss), di(seqs), dtype=out)
        for x, got in ((k, rk), (v, rv)):
            val, q, s = held(x, pool)
            f = q.float() * s[..., None] if s is not None else q.float()
            f[skip] = 0.0
            assert torch.equal(bits(got.cpu()), bits(f.to(out)))


def test_write_decode_rows_and_unaligned_strides(jy):
    """without seq row r is sequence r; k and v parts of one buffer at odd offsets"""
    c = Cache(jy, [33, 5, 64], 2, 64, 16, "i8", seed=21)
    buf = torch.randn((3, 300), generator=gen(2)).to(torch.bfloat16).to(DEV)
    k, v = buf[:, 1:129].unflatten(1, (2, 64)), buf[:, 151:279].unflatten(1, (2, 64))
    pos = torch.tensor([32, 4, 63], dtype=torch.int32, device=DEV)
    c.pool.write(c.layer, k, v, c.dtables, pos)
    rk, rv = c.pool.read(c.layer, c.dtables, pos)
    for x, got in ((k, rk), (v, rv)):
        _, q, s = held(x.cpu(), "i8")
        assert torch.equal(got.cpu(), q.float() * s[..., None])
    # read into rows of a wider buffer at an odd offset
    wide = torch.full((3, 2, 70), 5.0, device=DEV)
    out = c.pool.read(c.layer, c.dtables, pos, out=(wide[:, :, 1:65], torch.empty((3, 2, 64), device=DEV)))
    assert torch.equal(out[0], rk) and (wide[:, :, 0] == 5).all() and (wide[:, :, 65:] == 5).all()


def test_write_nan_and_infinity(jy):
    c = Cache(jy, [16], 2, 64, 16, "i8", seed=22)
    k = torch.randn((3, 2, 64), generator=gen(1))
    k[0, 0, 3], k[1, 1, 63], k[2, 0, 0] = math.nan, math.inf, -math.inf
    pos = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    seq = torch.zeros(3, dtype=torch.int32, device=DEV)
    c.pool.write(c.layer, k.to(DEV), k.to(DEV), c.dtables, pos, seq)
    got = c.pool.read(c.layer, c.dtables, pos, seq)[0].cpu()
    bad = torch.tensor([[1, 0], [0, 1], [1, 0]], dtype=torch.bool)
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()


def test_write_needs_int32_rows(jy):
    c = Cache(jy, [16], 1, 64, 16, "i8")
    k = torch.zeros((1, 1, 64), device=DEV)
    with pytest.raises(jy.JyError, match="int32"):
        c.pool.write(0, k, k, c.dtables, torch.zeros(1, dtype=torch.int64, device=DEV))
    with pytest.raises(jy.JyError, match="layer"):
        c.pool.write(2, k, k, c.dtables, torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(jy.JyError, match="k: "):
        c.pool.write(0, k[:, :, :32], k, c.dtables, torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(jy.JyError, match="one query row"):
        c.pool.attend(0, torch.zeros((2, 1, 64), device=DEV), c.dtables, torch.zeros(2, dtype=torch.int32, device=DEV), 4)


def test_no_rows(jy):
    c = Cache(jy, [16], 2, 64, 16, "i8", seed=23)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    before = c.pool.k.clone()
    c.pool.write(c.layer, torch.zeros((0, 2, 64), device=DEV), torch.zeros((0, 2, 64), device=DEV), c.dtables, none, none)
    assert torch.equal(c.pool.k, before)
    assert c.pool.read(c.layer, c.dtables, none, none)[0].shape == (0, 2, 64)


def test_offsets_past_32_bits(jy):
    """a pool of more than 2^32 bytes: its last pages are the ones used"""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    npages = (1 << 32) // (16 * 8 * 128) + 300
    pool = jy.PagePool.empty(1, npages, 16, 8, 128, device=DEV)
    n = 40
    t = torch.tensor([[npages - 1, 3, npages - 2]], dtype=torch.int32, device=DEV)
    k, v = (torch.randn((n, 8, 128), generator=gen(i)) for i in (1, 2))
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    pool.write(0, k.to(DEV), v.to(DEV), t, pos, torch.zeros_like(pos))
    kv, kq, ks = held(k, "i8")
    vv, _, _ = held(v, "i8")
    assert torch.equal(pool.k[0, npages - 1].cpu(), kq[:16].permute(1, 0, 2))
    got = pool.read(0, t, pos, torch.zeros_like(pos))[0]
    assert torch.equal(got.cpu(), kq.float() * ks[..., None])
    q = torch.randn((1, 32, 128), generator=gen(3))
    out = pool.attend(0, q.to(DEV), t, torch.tensor([n], dtype=torch.int32, device=DEV), n)
    check(out, *attention64(q, [kv], [vv], 1 / math.sqrt(128)))


# ---------------------------------------------------------------- together

def step(c, k, v, q, pos, max_len):
    c.pool.write(c.layer, k, v, c.dtables, pos)
    return c.pool.attend(c.layer, q, c.dtables, pos + 1, max_len)


def test_decode_steps_together(jy):
    """a batch grows position by position: each step's rows are written, then attended over"""
    lens = [60, 1, 17]
    c = Cache(jy, [n + 12 for n in lens], 2, 64, 16, "i8", seed=30)
    for i in range(12):
        k, v, q = (torch.randn(s, generator=gen(100 * j + i)) for j, s in enumerate([(3, 2, 64), (3, 2, 64), (3, 4, 64)]))
        for b, n in enumerate(lens):
            c.k[b][n + i], c.v[b][n + i] = held(k[b], "i8")[0], held(v[b], "i8")[0]
        pos = torch.tensor([n + i for n in lens], dtype=torch.int32, device=DEV)
        got = step(c, k.to(DEV), v.to(DEV), q.to(DEV), pos, 128)
        now = [n + i + 1 for n in lens]
        check(got, *attention64(q, [x[:m] for x, m in zip(c.k, now)], [x[:m] for x, m in zip(c.v, now)], 0.125))


@pytest.mark.parametrize("max_len", [100, 3000])
def test_captured_step_replays(jy, max_len):
    """write and attend recorded into a graph (two graphs, replayed in turn, eager work between):
    every replay gives the eager result, with the positions that stand in its buffers then"""
    lens = [60, 1, 17, 90]
    c = Cache(jy, lens, 2, 64, 16, "i8", seed=31)
    c2 = Cache(jy, lens, 2, 64, 16, "i8", seed=31)
    new = lambda i: [torch.randn(s, generator=gen(10 * i + j)).to(DEV) for j, s in enumerate([(4, 2, 64), (4, 2, 64), (4, 4, 64)])]  # noqa: E731
    pos = torch.tensor([59, 0, 16, -1], dtype=torch.int32, device=DEV)
    bufs, graphs, outs = [new(i) for i in range(2)], [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(c, *bufs[0], pos, max_len)
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c, *bufs[i], pos, max_len))
        graphs.append(g)
    for r in range(6):
        i = r % 2
        for t, x in zip(bufs[i], new(50 + r)):
            t.copy_(x)
        pos.copy_(torch.tensor([59 - r, r, 16 - r, -1 if r % 3 else 89], dtype=torch.int32))
        graphs[i].replay()
        torch.cuda.synchronize()
        want = step(c2, *bufs[i], pos, max_len)
        assert torch.equal(outs[i], want), r
        assert torch.equal(c.pool.k, c2.pool.k)
        assert pos[3] >= 0 or not outs[i][3].any()


def test_on_other_streams(jy):
    """two streams at once, each with its own workspace"""
    c = Cache(jy, [2000, 500], 2, 64, 16, "i8", seed=32)
    qs = [torch.randn((2, 8, 64), generator=gen(i)).to(DEV) for i in range(2)]
    want = [c.attend(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("max_len", [40, 3000])
def test_attend_refuses_heads_at_any_length(jy, max_len):
    """query heads that are no multiple of the key/value heads, fewer of them among those"""
    c = Cache(jy, [40], 4, 64, 16, "i8", seed=33)
    for heads in (1, 2, 3, 6):
        with pytest.raises(jy.JyError, match="multiple"):
            c.attend(torch.zeros((1, heads, 64), device=DEV), max_len=max_len)


@pytest.mark.parametrize("size", [1e-33, 1e-34, 1e-36])
def test_attend_value_scales_down_to_the_smallest(jy, size):
    """value scales of any size, those far under 2^-112 among them.  There a weight times its scale counts
    in steps of 2^-24 2^-127 (the smallest half, times the largest power of two that fp32 holds) instead of
    2^-39 of the largest: each of the n products is off by at most that times a byte of 127, over a sum of
    weights of at least 1; and fp32's own steps down there are 2^-149, once per product and for the output."""
    c = Cache(jy, [100], 1, 64, 16, "i8", seed=11)
    vs = c.vs * size
    pool = jy.PagePool(c.pool.k, c.pool.v, c.pool.k_scale, vs.to(DEV))
    at = c.tables[0].long()
    v = (c.vq.double() * vs.double()[..., None])[c.layer, at].permute(1, 0, 2, 3).reshape(1, -1, 64)[:, :100].permute(1, 0, 2)
    q = torch.randn((1, 4, 64), generator=gen(3))
    got = pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 100)
    want, bound = attention64(q, c.k, [v], 0.125)
    check(got, want, bound + 100 * 127 * 2.0**-151 + 101 * 2.0**-149)


@pytest.mark.parametrize("size", [1e-30, 1e-31, 1e-33, 1e-38, 1e-42])
def test_attend_queries_down_to_the_smallest(jy, size):
    """a query under 2^-104 against int8 keys counts as zeros, however large the keys (the row is a mean);
    above that it does not"""
    c = Cache(jy, [100], 1, 64, 16, "i8", seed=11)
    pool = jy.PagePool(c.pool.k, c.pool.v, (c.ks * 2.0**100).to(DEV), c.pool.v_scale)
    q = torch.randn((1, 4, 64), generator=gen(3)) * size
    got = pool.attend(c.layer, q.to(DEV), c.dtables, c.dlens, 100)
    if q.abs().max() < 2.0**-104:
        q.zero_()
    check(got, *attention64(q, [x * 2.0**100 for x in c.k], c.v, 0.125))


# ---------------------------------------------------------------- infinities in 16-bit pools

@pytest.mark.parametrize("hd", [16, 32, 48, 80, 96, 112, 144, 192, 240])
@pytest.mark.parametrize("pool", ["f16", "bf16"])
def test_attend_infinite_keys_of_any_head_size(jy, pool, hd):
    """a key's infinity in any of its dims, against the query's sign: that position has no weight, and the
    row is the others'"""
    n = 60
    c = Cache(jy, [n], 1, hd, 16, pool, seed=43, layers=1, layer=0)
    q = torch.ones((1, 2, hd), dtype=POOL[pool])
    live = torch.ones(n, dtype=torch.bool)
    for p in range(0, n, 3):
        c.pool.k[0, int(c.tables[0, p // 16]), 0, p % 16, (p // 3 * 5) % hd] = -math.inf
        live[p] = False
    got = c.attend(q.to(DEV))
    # (a weight of 0 and what stands beside it add nothing: the bound is the others')
    check(got, *attention64(q, [c.k[0][live]], [c.v[0][live]], 1 / math.sqrt(hd)))


def attention_of_infinities(q, k, v, scale):
    """(out, bound) of one sequence's definition in 64 bits with infinities among keys and values:
    a score of -infinity has no weight (all of them: zeros), one of +infinity or NaN makes its row NaN,
    a value that is not finite its dim of the rows whose head reads it.  (No position here has both.)"""
    nh, hd = q.shape
    per = nh // k.shape[1]
    out, bound = torch.empty(nh, hd, dtype=torch.float64), torch.zeros(nh, hd, dtype=torch.float64)
    for h in range(nh):
        kk, vv = k[:, h // per], v[:, h // per]
        s = (kk * q[h].double()).sum(-1) * scale
        live = s != -math.inf
        if not torch.isfinite(s[live]).all():
            out[h] = math.nan
            continue
        if not live.any():
            out[h] = 0.0
            continue
        kk, vv = kk[live][:, None], vv[live][:, None]
        a, b = attention64(q[None, h:h + 1], [kk], [torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)], scale)
        inf = torch.where(torch.isfinite(vv), torch.zeros_like(vv), vv).sum((0, 1))  # (opposite ones: NaN)
        out[h], bound[h] = a[0, 0] + inf, b[0, 0]
    return out, bound


def check_infinities(got, want, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])
    return ~(torch.isnan(want) | inf)


@pytest.mark.parametrize("n", [40, 700, 3000])
@pytest.mark.parametrize("hd", [64, 80, 112, 128, 256])
@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("pool", ["f16", "bf16"])
def test_attend_infinities_in_16_bit_pages(jy, pool, io, hd, n):
    """infinite keys and values, as fp32 rows past a 16-bit type's range are held, whatever the query's type
    and the head size: whole numbers as queries, which need no second part"""
    c = Cache(jy, [n, 33, 20], 2, hd, 16, pool, seed=40, layers=1, layer=0, outliers=False)
    g = gen(41)
    q = torch.randint(1, 4, (3, 4, hd), generator=g).float() * (torch.randint(0, 2, (3, 4, hd), generator=g) * 2 - 1)
    q[:, 2:] += torch.rand((3, 2, hd), generator=g) * 0.9  # (and others)
    q = q.to(IO[io])

    def put(which, b, p, head, d, x):
        getattr(c.pool, which)[0, int(c.tables[b, p // 16]), head, p % 16, d] = x
        getattr(c, which)[b][p, head, d] = x

    # a key against the sign of head 0's query, so the position has no weight there
    for p, d in ((0, 0), (1, hd - 1), (17, 5), (n - 1, hd // 2)):
        put("k", 0, p, 0, d, -math.inf * float(torch.sign(q[0, 0, d].float())))
        q[0, 1, d] = q[0, 0, d]
    # values: one dim of each sign, one with both
    for p, d, x in ((3, 0, math.inf), (n - 2, 9, -math.inf), (5, hd - 1, math.inf), (30, hd - 1, -math.inf)):
        put("v", 0, p, 0, d, x)
    # a key along the query of head 2 (kv head 1): its row is NaN; head 3 by its own sign
    put("k", 0, 6, 1, 2, math.inf * float(torch.sign(q[0, 2, 2].float())))
    # an infinity that meets a zero, and a held NaN
    q[1, 0, 7] = 0.0
    put("k", 1, 4, 0, 7, math.inf)
    put("v", 1, 32, 1, 3, math.nan)
    # every score -infinity: zeros
    for p in range(20):
        put("k", 2, p, 0, 1, -math.inf)
    q[2, :2, 1] = 1.0
    scale = 0.25 / math.sqrt(hd)
    got = c.attend(q.to(DEV), scale=scale)
    want, bound = (torch.stack(x) for x in zip(*[attention_of_infinities(q[b], c.k[b], c.v[b], scale) for b in range(3)]))
    ok = check_infinities(got, want, bound)
    zero = torch.zeros((), dtype=torch.float64)
    check(torch.where(ok.to(DEV), got, zero.to(got.dtype).to(DEV)), torch.where(ok, want, zero), bound)
    assert not got[2, :2].any() and torch.isfinite(got[2, 2:]).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_rows_past_fp16s_range_from_write_to_attention(jy, io):
    """written to an fp16 pool they are held as infinities, and attention takes them as such"""
    c = Cache(jy, [40], 1, 80, 16, "f16", seed=42, layers=1, layer=0)
    k, v = torch.randn((1, 1, 80), generator=gen(1)), torch.randn((1, 1, 80), generator=gen(2))
    k[0, 0, 3], v[0, 0, 70] = -1e5, 7e4
    pos = torch.tensor([21], dtype=torch.int32, device=DEV)
    c.pool.write(0, k.to(IO[io]).to(DEV), v.to(IO[io]).to(DEV), c.dtables, pos)
    c.k[0][21], c.v[0][21] = held(k.to(IO[io]), "f16")[0], held(v.to(IO[io]), "f16")[0]
    assert c.k[0][21, 0, 3] == -math.inf and c.v[0][21, 0, 70] == math.inf
    q = torch.ones((1, 2, 80)).to(IO[io])
    q[0, 1, 3] = -1.0
    got = c.attend(q.to(DEV), scale=0.05)
    # head 0's score there is -infinity: its weight, 0, times the infinite value is NaN, the rest is finite
    want, bound = attention_of_infinities(q[0], c.k[0], c.v[0], 0.05)
    want[0, 70] = math.nan
    check_infinities(got[0], want, bound)
    assert torch.isnan(got[0, 1]).all() and torch.isfinite(got[0, 0, :70]).all()
