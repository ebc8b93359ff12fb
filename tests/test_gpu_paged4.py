"""The key/value cache in 4 bits against plain implementations in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step, relative
SIZES = [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 240, 256]


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


def held4(x):
    """What the format holds of fp32 vectors x [..., hd], element by element from its rule: (values float64, numbers
    int [..., hd], words fp16 [..., groups, 2])."""
    hd = x.shape[-1]
    G = 2 if hd <= 64 else 4 if hd <= 128 else 8
    values, numbers = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.int32)
    words = torch.zeros((*x.shape[:-1], G, 2), dtype=torch.float16)
    for g in range(-(-hd // 32)):
        part = x[..., 32 * g:32 * g + 32].float()
        low = part.amin(-1).half()
        u = ((part.amax(-1) - low.float()) / torch.tensor(15.0)).view(torch.int32)
        step = ((u + 0xffff + ((u >> 17) & 1)) & ~0x1ffff).view(torch.float32).half()
        s, lo = step.float()[..., None], low.float()[..., None]
        inv = torch.where(s > 0, torch.ones_like(s) / s, torch.zeros_like(s))
        n = torch.round((part - lo) * inv).clamp(0, 15)
        words[..., g, 0], words[..., g, 1] = step, low
        numbers[..., 32 * g:32 * g + 32] = n.int()
        values[..., 32 * g:32 * g + 32] = n.double() * s.double() + lo.double()
    bad = ~(x.abs() <= 30000).all(-1)
    values[bad], numbers[bad] = math.nan, 0
    words[..., :-(-hd // 32), :][bad] = math.nan
    return values, numbers, words


def packed4(numbers):
    """the bytes of a vector's numbers"""
    hd = numbers.shape[-1]
    G = 2 if hd <= 64 else 4 if hd <= 128 else 8
    b = torch.zeros((*numbers.shape[:-1], 16 * G), dtype=torch.uint8)
    for e in range(hd):
        g, r = e // 32, e % 32 // 2
        b[..., r * G + g] |= (numbers[..., e] << (4 * (e % 2))).to(torch.uint8)
    return b


@pytest.mark.parametrize("hd", SIZES)
@pytest.mark.parametrize("io", list(IO))
def test_write_bytes_and_read(jy, hd, io):
    """the bytes and words of every vector by the rule, the slots beside them untouched, the values back"""
    g = gen(hd)
    rows, nkv, page = 21, 3, 16
    kv = torch.randn((rows, 2, nkv, hd), generator=g) * torch.exp(0.5 * torch.randn(hd, generator=g))
    kv[3], kv[4, 0], kv[5, 1] = 0.0, 7.25, kv[5, 1] * 1e-6
    kv = kv.to(IO[io])
    p = jy.PagePool.empty(2, 5, page, nkv, hd, dtype=torch.uint8, device=DEV)
    for t in (p.k, p.v, p.k_scale.view(torch.int16), p.v_scale.view(torch.int16)):
        t.fill_(0x5a)
    tables = torch.tensor([[3, -1], [0, 4]], dtype=torch.int32)
    seq = torch.tensor([r % 2 for r in range(rows)], dtype=torch.int32)
    pos = torch.tensor([r // 2 * 2 + (r % 2) * 5 for r in range(rows)], dtype=torch.int32)
    pos[20] = -1
    p.write(1, kv.to(DEV)[:, 0], kv.to(DEV)[:, 1], tables.to(DEV), pos.to(DEV), seq.to(DEV))
    got = p.read(1, tables.to(DEV), pos.to(DEV), seq.to(DEV), dtype=IO[io])
    for side, (bytes_, words, back) in enumerate(((p.k, p.k_scale, got[0]), (p.v, p.v_scale, got[1]))):
        values, numbers, w = held4(kv[:, side].float())
        b = packed4(numbers)
        wantb, wantw = torch.full_like(bytes_.cpu(), 0x5a), torch.full_like(words.cpu().view(torch.int16), 0x5a)
        for r in range(rows):
            at = int(pos[r])
            pg = int(tables[int(seq[r]), at // page]) if 0 <= at < 2 * page else -1
            if pg < 0:
                values[r] = 0.0
                continue
            wantb[1, pg, :, at % page] = b[r]
            wantw[1, pg, :, at % page] = w[r].view(torch.int16)
        assert torch.equal(bytes_.cpu(), wantb)
        assert torch.equal(words.cpu().view(torch.int16), wantw)
        assert torch.equal(back.cpu(), values.float().to(IO[io]))  # (number x step is exact: fp32's rounding, then the type's)


def test_write_what_is_not_finite(jy):
    x = torch.randn((6, 1, 80), generator=gen(1))
    x[0, 0, 3], x[1, 0, 79], x[2, 0, 64], x[3, 0, 0] = math.nan, math.inf, -math.inf, 30001.0
    x[4, 0, 1], x[4, 0, 2] = 30000.0, -30000.0
    p = jy.PagePool.empty(1, 1, 16, 1, 80, dtype=torch.uint8, device=DEV)
    t, pos, seq = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([[0]], list(range(6)), [0] * 6))
    p.write(0, x.to(DEV), x.to(DEV), t, pos, seq)
    k, v = p.read(0, t, pos, seq)
    assert torch.isnan(k[:4]).all() and torch.isfinite(k[4:]).all() and torch.equal(k[4:], v[4:])
    assert torch.equal(k[4:].cpu(), held4(x[4:])[0].float())


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("io", list(IO))
def test_strides(jy, io, off):
    """rows and heads of any stride, pairs that lie across their alignment; what lies between stays"""
    p = jy.PagePool.empty(1, 3, 16, 2, 48, dtype=torch.uint8, device=DEV)
    buf = torch.randn((7, 5, 51), generator=gen(2)).to(IO[io]).to(DEV)
    k, v = buf[:, 0:4:2, off:off + 48], buf[:, 1:5:2, off:off + 48]
    t, pos = torch.arange(3, dtype=torch.int32, device=DEV)[:, None].contiguous(), torch.tensor([0, 3, 15, 1, 2, 5, 9], dtype=torch.int32, device=DEV)
    seq = torch.tensor([0, 1, 2, 0, 1, 2, 0], dtype=torch.int32, device=DEV)
    p.write(0, k, v, t, pos, seq)
    out = torch.full_like(buf, 9.0)
    p.read(0, t, pos, seq, out=(out[:, 0:4:2, off:off + 48], out[:, 1:5:2, off:off + 48]))
    for a, b in ((k, out[:, 0:4:2, off:off + 48]), (v, out[:, 1:5:2, off:off + 48])):
        assert torch.equal(b.cpu(), held4(a.cpu().float())[0].float().to(IO[io]))
    out[:, 0:4, off:off + 48] = 9.0
    assert (out == 9.0).all()
