"""Eviction of the positions with the least weight against sorting, and one layer's step over several sequences
with all the operators around the cache in a row."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"
POOL = {"i4": torch.uint8, "i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}


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


def paged(lens, page, g, lead=0):
    """tables of these lengths over pages from `lead` on in random order, and how many"""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=g) + lead
    t = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n].int()
        at += n
    return t, sum(need)


def stays(w, n, keep, recent, there):
    """the positions that stay, in order"""
    old = max(n - recent, 0)
    late = [j for j in range(old, n) if there[j]]
    early = [j for j in range(old) if there[j]]
    rank = lambda j: (-math.inf, 1) if math.isnan(w[j]) else (w[j], 0)  # noqa: E731
    early.sort(key=lambda j: (math.isnan(w[j]), -rank(j)[0], j))
    return sorted(early[:max(0, min(keep, len(late) + len(early)) - len(late))]) + late


def run(jy, pool, lens, nkv, hd, page, keep, recent, weights, gone=(), max_len=None, cols=None, strided=False):
    g = gen(7)
    tables, used = paged(lens, page, g)
    to, fresh = paged([min(keep, max(lens))] * len(lens), page, g, lead=used)
    p = jy.PagePool.empty(2, used + fresh + 1, page, nkv, hd, dtype=POOL[pool], device=DEV)
    for t in (p.k, p.v, p.k_scale, p.v_scale):
        if t is not None:
            t.zero_()
    rows = [(b, j) for b, n in enumerate(lens) for j in range(n)]
    seq, pos = ints([r[0] for r in rows]), ints([r[1] for r in rows])
    if rows:
        x = torch.randn((len(rows), 2, nkv, hd), generator=g).to(DEV)
        p.write(1, x[:, 0], x[:, 1], tables.to(DEV), pos, seq)
    for b, i in gone:
        tables[b, i] = [-1, 1 << 30][i % 2]
    before = [t.clone() for t in (p.k, p.v, p.k_scale, p.v_scale) if t is not None]
    dt, dto = tables.to(DEV), to.to(DEV)
    old_k, old_v = p.read(1, dt, pos, seq)
    w = weights.to(DEV)
    if strided:
        wide = torch.full((w.shape[0] + 1, w.shape[1] + 2, w.shape[2] + 5), 3.0, device=DEV)
        wide[1:, 1:-1, 2:-3] = w
        w = wide[1:, 1:-1, 2:-3]
    most = max(lens) if max_len is None else max_len
    new_w = None if cols is None else torch.full((len(lens), nkv, cols), -7.0, device=DEV)
    kept, new_lens, got_w = p.evict(1, w, dt, ints(lens), keep, recent, most, dto, new_weights=new_w)
    width = min(keep, most)
    for b, n in enumerate(lens):
        n = min(n, most)
        there = [0 <= int(tables[b, j // page]) < p.pages for j in range(n)]
        for h in range(nkv):
            row = weights[b, h].tolist()
            row = row + [0.0] * (n - len(row))
            want = stays(row, n, keep, recent, there)
            assert kept[b, h].tolist() == want + [-1] * (keep - len(want)), (b, h)
            assert int(new_lens[b]) == len(want)
            have = [row[j] for j in want][:got_w.shape[2]]
            have = torch.tensor(have + [0.0] * (got_w.shape[2] - len(have)), dtype=torch.float32)
            assert torch.equal(got_w[b, h].cpu().nan_to_num(-9.0), have.nan_to_num(-9.0))
            if want:
                at = [rows.index((b, 0)) + j for j in want]
                k, v = p.read(1, dto, ints(list(range(len(want)))), ints([b] * len(want)))
                assert torch.equal(k[:, h], old_k[at, h]) and torch.equal(v[:, h], old_v[at, h])
    # nothing but the new pages' first `width` positions has changed
    for t, was in zip((t for t in (p.k, p.v, p.k_scale, p.v_scale) if t is not None), before):
        left = t.clone()
        for b in range(len(lens)):
            for i in range(min(width, int(new_lens[b]))):
                left[1, int(to[b, i // page]), :, i % page] = was[1, int(to[b, i // page]), :, i % page]
        assert torch.equal(left.view(torch.uint8), was.view(torch.uint8))
    return kept, new_lens, got_w


@pytest.mark.parametrize("pool", list(POOL))
@pytest.mark.parametrize("nkv,hd,page", [(2, 64, 16), (1, 128, 64), (3, 80, 32), (2, 256, 16), (1, 16, 256), (5, 144, 16)])
def test_shapes(jy, pool, nkv, hd, page):
    lens = [1, 50, 0, 201, 33]
    w = torch.rand((5, nkv, 201), generator=gen(1))
    run(jy, pool, lens, nkv, hd, page, 40, 7, w)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (64, 0), (64, 64), (64, 63), (299, 10), (300, 0), (301, 301), (1000, 5)])
def test_keep_and_recent(jy, keep, recent):
    run(jy, "i8", [300, 299, 64, 1], 2, 32, 16, keep, recent, torch.rand((4, 2, 300), generator=gen(2)))


@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "negative", "tiny", "special", "rising", "falling"])
def test_weights_of_every_kind(jy, kind):
    """ties by position, both zeros the same, signs, subnormals, infinities and NaN"""
    n, g = 700, gen(3)
    w = torch.randn((2, 2, n), generator=g)
    if kind == "equal":
        w = torch.full_like(w, 0.25)
    if kind == "zeros":
        w = torch.where(w > 0, 0.0, -0.0)
    if kind == "few":
        w = (w * 2).round()
    if kind == "tiny":
        w = w * 1e-40
    if kind == "special":
        w[:, :, ::3] = math.inf
        w[:, :, 1::7] = -math.inf
        w[:, :, 2::5] = math.nan
    if kind == "rising":
        w = 1 + torch.arange(n).float().expand(2, 2, n) * 2.0**-23
    if kind == "falling":
        w = 1 - torch.arange(n).float().expand(2, 2, n) * 2.0**-24
    for keep in (1, 100, 350, 699):
        run(jy, "f16", [n, n - 3], 2, 16, 16, keep, min(keep, 20), w.contiguous())


def test_long(jy):
    """several chunks of positions, a border far inside one"""
    w = torch.exp(2 * torch.randn((1, 1, 20011), generator=gen(4)))
    w[0, 0, torch.rand(20011, generator=gen(5)) < 0.2] = 0.0
    for keep in (37, 9000, 17500):
        run(jy, "i4", [20011], 1, 32, 64, keep, 30, w)


def test_holes_cuts_and_strides(jy):
    w = torch.rand((3, 2, 150), generator=gen(6))
    gone = [(0, 0), (0, 5), (1, 2), (1, 3), (1, 6), (2, 0), (2, 1), (2, 2)]
    for keep, recent in ((30, 20), (100, 0), (200, 200)):
        run(jy, "bf16", [150, 111, 40], 2, 48, 16, keep, recent, w, gone=gone, strided=True)
    run(jy, "i8", [150, 111, 40], 2, 48, 16, 30, 10, w, max_len=100)
    run(jy, "i8", [150, 111, 40], 2, 48, 16, 30, 10, w, max_len=0)
    run(jy, "i8", [150, 111, 40], 2, 48, 16, 60, 10, w[:, :, :70].contiguous(), cols=25)  # short weights, short new ones
    run(jy, "i8", [150, 111, 40], 2, 48, 16, 60, 10, w[:, :, :0].contiguous(), cols=500)


def test_weights_in_place(jy):
    w = torch.rand((2, 2, 9000), generator=gen(7))
    _, _, want = run(jy, "i8", [9000, 4444], 2, 16, 256, 3000, 100, w)
    g = gen(7)
    tables, used = paged([9000, 4444], 256, g)
    to, fresh = paged([3000, 3000], 256, g, lead=used)
    p = jy.PagePool.empty(1, used + fresh, 256, 2, 16, device=DEV)
    mine = w.to(DEV)
    got = p.evict(0, mine, tables.to(DEV), ints([9000, 4444]), 3000, 100, 9000, to.to(DEV), new_weights=mine)[2]
    assert got is mine and torch.equal(mine, want)


def test_refusals_in_python(jy):
    p = jy.PagePool.empty(1, 8, 16, 2, 16, device=DEV)
    t, w, n = ints([[0, 1]]), torch.zeros((1, 2, 32), device=DEV), ints([20])
    with pytest.raises(jy.JyError, match="keep"):
        p.evict(0, w, t, n, 0, 0, 32, ints([[2]]))
    with pytest.raises(jy.JyError, match="keep"):
        p.evict(0, w, t, n, 3, 4, 32, ints([[2]]))
    with pytest.raises(jy.JyError, match="too few pages"):
        p.evict(0, w, t, n, 17, 4, 32, ints([[2]]))
    with pytest.raises(jy.JyError, match="other sequences"):
        p.evict(0, w, t, n, 3, 2, 32, ints([[2], [3]]))
    with pytest.raises(jy.JyError, match="weights"):
        p.evict(0, w[:, :1], t, n, 3, 2, 32, ints([[2]]))
    with pytest.raises(jy.JyError, match="lens"):
        p.evict(0, w, t, n.long(), 3, 2, 32, ints([[2]]))


@pytest.mark.parametrize("pool", ["i4", "i8", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_a_layers_steps(jy, pool, layout):
    """prompts of three sequences, steps whose weights add up, an eviction, steps over what stayed: rotary
    positions, writes, attention and eviction against one dense computation in 64 bits of the same cache"""
    nh, nkv, hd, page, keep, recent = 6, 2, 64, 16, 24, 6
    g = gen(9)
    new = [40, 17, 29]
    steps, after = 5, 4
    tables, used = paged([n + steps for n in new], page, g)
    to, fresh = paged([keep + after] * 3, page, g, lead=used)
    p = jy.PagePool.empty(1, used + fresh, page, nkv, hd, dtype=POOL[pool], device=DEV)
    dt, dto = tables.to(DEV), to.to(DEV)
    freq = jy.rope_frequencies(hd, 10000.0, "ramp", 4.0, trained=64, device=DEV)
    store = [[[] for _ in range(nkv)] for _ in range(3)]  # what each head's cache holds, (k, v) float64 in order
    acc = [[[] for _ in range(nkv)] for _ in range(3)]
    weights = torch.zeros((3, nkv, 64), device=DEV)

    def turn(x, pos):
        a = pos.double()[:, None, None] * freq.cpu()
        x = x.double()
        i, j = (slice(0, hd // 2), slice(hd // 2, hd)) if layout == "half" else (slice(0, hd, 2), slice(1, hd, 2))
        y = x.clone()
        y[..., i], y[..., j] = x[..., i] * torch.cos(a) - x[..., j] * torch.sin(a), x[..., i] * torch.sin(a) + x[..., j] * torch.cos(a)
        return y

    def append(qkv, pos, at, seq, table):
        """(q turned) after the rows' keys and values are held"""
        q, k, v = qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:]
        q, k = jy.rope(q, k, ints(pos), freq, layout=layout)
        want = turn(qkv[:, :nh].cpu(), torch.tensor(pos))
        assert (q.double().cpu() - want).abs().max() < 1e-5
        p.write(0, k, v, table, ints(at), ints(seq))
        kk, vv = (t.double().cpu() for t in p.read(0, table, ints(at), ints(seq)))
        close = turn(qkv[:, nh:nh + nkv].cpu(), torch.tensor(pos))
        limit = {"i4": 1 / 15, "i8": 1 / 200, "bf16": 1 / 200}[pool] * 2 * close.abs().amax(-1, keepdim=True)
        assert ((kk - close).abs() <= limit).all()
        for r, s in enumerate(seq):
            for h in range(nkv):
                store[s][h].append((kk[r, h], vv[r, h]))
                acc[s][h].append(0.0)
        return q

    def dense(q, s, h, n, dist_cap=20.0):
        k, v = (torch.stack([x[i] for x in store[s][h // (nh // nkv)][:n]]) for i in range(2))
        x = dist_cap * torch.tanh((k @ q.double()) / math.sqrt(hd) / dist_cap)
        w = torch.softmax(x, 0)
        return w @ v, w

    total = sum(new)
    qkv = torch.randn((total, nh + 2 * nkv, hd), generator=g).to(DEV)
    seq = [s for s in range(3) for _ in range(new[s])]
    pos = [i for n in new for i in range(n)]
    q = append(qkv, pos, pos, seq, dt)
    starts = [0, new[0], new[0] + new[1], total]
    out = p.attend_rows(0, q, dt, ints(starts), ints(pos), 64, cap=20.0).double().cpu()
    for r in range(0, total, 3):
        for h in range(nh):
            assert (out[r, h] - dense(q[r, h].cpu(), seq[r], h, pos[r] + 1)[0]).abs().max() < 2e-5
    for t in range(steps):
        at = [n + t for n in new]
        q = append(torch.randn((3, nh + 2 * nkv, hd), generator=g).to(DEV), at, at, [0, 1, 2], dt)
        out = p.attend(0, q, dt, ints([a + 1 for a in at]), 64, cap=20.0, weights=weights).double().cpu()
        for s in range(3):
            for h in range(nh):
                o, w = dense(q[s, h].cpu(), s, h, at[s] + 1)
                assert (out[s, h] - o).abs().max() < 2e-5
                acc[s][h // (nh // nkv)] = [a + float(b) for a, b in zip(acc[s][h // (nh // nkv)], w)]
    for s in range(3):
        assert (weights[s, :, :new[s] + steps].double().cpu() - torch.tensor(acc[s])).abs().max() < 1e-4
        assert not weights[s, :, new[s] + steps:].any()
    kept, lens, weights = p.evict(0, weights, dt, ints([n + steps for n in new]), keep, recent, 64, dto)
    assert lens.tolist() == [min(keep, n + steps) for n in new]
    for s in range(3):
        for h in range(nkv):
            ids = [i for i in kept[s, h].tolist() if i >= 0]
            assert len(ids) == int(lens[s]) and ids == sorted(set(ids)) and ids[-recent:] == list(range(new[s] + steps - recent, new[s] + steps))
            lost = set(range(new[s] + steps)) - set(ids)
            old = [i for i in ids if i < new[s] + steps - recent]
            assert not lost or not old or min(acc[s][h][i] for i in old) >= max(acc[s][h][i] for i in lost) - 1e-4
            store[s][h] = [store[s][h][i] for i in ids]
            acc[s][h] = [acc[s][h][i] for i in ids]
    # the next tokens stand where they stand in the text, and lie behind what stayed
    n = lens.tolist()
    for t in range(after):
        where, at = [a + steps + t for a in new], [a + t for a in n]
        q = append(torch.randn((3, nh + 2 * nkv, hd), generator=g).to(DEV), where, at, [0, 1, 2], dto)
        out = p.attend(0, q, dto, ints([a + 1 for a in at]), 64, cap=20.0, weights=weights).double().cpu()
        for s in range(3):
            for h in range(nh):
                o, w = dense(q[s, h].cpu(), s, h, at[s] + 1)
                assert (out[s, h] - o).abs().max() < 2e-5
                acc[s][h // (nh // nkv)] = [a + float(b) for a, b in zip(acc[s][h // (nh // nkv)], w)]
    for s in range(3):
        assert (weights[s, :, :n[s] + after].double().cpu() - torch.tensor(acc[s])).abs().max() < 1e-4


def test_a_replayed_graph(jy):
    g = gen(1)
    tables, used = paged([500, 300], 16, g)
    to, fresh = paged([100, 100], 16, g, lead=used)
    p = jy.PagePool.empty(1, used + fresh, 16, 2, 64, dtype=torch.uint8, device=DEV)
    for t in (p.k, p.v):
        t.random_(0, 256)
    p.k_scale.normal_()
    p.v_scale.normal_()
    dt, dto, lens = tables.to(DEV), to.to(DEV), ints([500, 300])
    w = torch.rand((2, 2, 500), device=DEV)
    graph = torch.cuda.CUDAGraph()
    p.evict(0, w, dt, lens, 100, 10, 500, dto)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kept, new_lens, new_w = p.evict(0, w, dt, lens, 100, 10, 500, dto)
    for i in range(3):
        w.copy_(torch.rand((2, 2, 500), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        a, b, c, pages = kept.clone(), new_lens.clone(), new_w.clone(), p.k.clone()
        again = p.evict(0, w, dt, lens, 100, 10, 500, dto)
        assert torch.equal(a, again[0]) and torch.equal(b, again[1]) and torch.equal(c, again[2]) and torch.equal(pages, p.k)


def test_a_table_of_2_to_the_30_positions(jy):
    """an upper bound far past the sequence: the ranks of 100 positions, not of all that the table could hold"""
    g = gen(4)
    p = jy.PagePool.empty(1, 2, 256, 1, 16, dtype=torch.float16, device=DEV)
    k, v = (torch.randn((100, 1, 16), generator=g).to(DEV) for _ in range(2))
    t = torch.full((1, 1 << 22), -1, dtype=torch.int32, device=DEV)
    t[0, 0] = 0
    at, zero = ints(list(range(100))), ints([0] * 100)
    p.write(0, k, v, t, at, seq=zero)
    w = torch.rand((1, 1, 100), generator=g).to(DEV)
    for bound in (1 << 29, 1 << 30):
        kept, n, left = p.evict(0, w, t, ints([100]), 40, 10, bound, ints([[1]]))
        want = stays(w[0, 0].tolist(), 100, 40, 10, [True] * 100)
        assert kept[0, 0].tolist() == want and n.tolist() == [40]
        assert torch.equal(left[0, 0, :40], w[0, 0, want]) and not left[0, 0, 40:].any()
        got, _ = p.read(0, ints([[1]]), ints(list(range(40))), seq=ints([0] * 40))
        assert torch.equal(got, k[want].half().float())
