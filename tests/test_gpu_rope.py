"""Rotary positions against the formula in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
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


def turned(x, pos, freq, layout, factor=1.0):
    """(values, room) in 64 bits.  fp32: a cosine or sine rounded from its polynomial of six steps and from the
    factor is off by at most 4 steps of 2^-24 of the factor, and a product, the other's rounding and the sum's by
    3 more: 8 times 2^-24 (|x| + |y|) factor, then the output's own rounding."""
    x, n = x.double().cpu(), freq.numel()
    a = pos.double().cpu()[:, None, None] * freq.double().cpu()
    i = torch.arange(n) if layout == "half" else 2 * torch.arange(n)
    j = i + (n if layout == "half" else 1)
    u, w = x[..., i], x[..., j]
    y, room = x.clone(), torch.zeros_like(x)
    y[..., i] = factor * (u * torch.cos(a) - w * torch.sin(a))
    y[..., j] = factor * (u * torch.sin(a) + w * torch.cos(a))
    room[..., i] = room[..., j] = 8 * 2.0**-24 * abs(factor) * (u.abs() + w.abs())
    return y, room


def check(got, want, room):
    tiny = 2.0**-25 if got.dtype is torch.float16 else 0.0
    off = (got.double().cpu() - want).abs()
    limit = room + HALF[got.dtype] * (want.abs() + room) + tiny
    assert torch.isfinite(got).all() and (off <= limit).all(), (off / limit.clamp(min=1e-300)).max()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("rows,nh,nkv,hd,pairs", [(1, 14, 2, 64, 32), (1, 1, 1, 2, 1), (5, 3, 3, 80, 40), (37, 32, 8, 128, 64),
                                                  (3, 4, 1, 128, 16), (2, 2, 1, 96, 13), (9, 5, 2, 7, 3), (2, 1, 1, 1024, 512),
                                                  (4, 3, 1, 256, 96), (1100, 2, 1, 64, 32), (4097, 3, 2, 40, 12), (2050, 1, 1, 16, 1)])
def test_shapes(jy, rows, nh, nkv, hd, pairs, io, layout):
    g = gen(rows + hd)
    q, k = torch.randn((rows, nh, hd), generator=g).to(IO[io]), torch.randn((rows, nkv, hd), generator=g).to(IO[io])
    pos = torch.randint(0, 5000, (rows,), generator=g, dtype=torch.int32)
    freq = jy.rope_frequencies(2 * pairs, device="cpu")
    a, b = jy.rope(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), layout=layout)
    check(a, *turned(q, pos, freq, layout))
    check(b, *turned(k, pos, freq, layout))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_and_factor(jy, layout):
    """far, negative and equal positions, a frequency of 0 and of more than one, a factor"""
    pos = torch.tensor([0, 1, -1, 7, 1 << 20, (1 << 31) - 1, -(1 << 31), 12345678, 7], dtype=torch.int32)
    freq = torch.tensor([0.0, 1.0, 3.7, -0.25, 1e-6, 5e-4, math.pi / 2, math.pi / 4], dtype=torch.float64)
    x = torch.randn((9, 3, 20), generator=gen(1))
    a, none = jy.rope(x.to(DEV), None, pos.to(DEV), freq.to(DEV), layout=layout, factor=1.375)
    assert none is None
    check(a, *turned(x, pos, freq, layout, 1.375))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("io", list(IO))
@pytest.mark.parametrize("off", [0, 1])
def test_strides_and_in_place(jy, io, layout, off):
    """heads of one fused projection turned where they lie, aligned and not; what is beside them stays"""
    buf = torch.randn((6, 9, 72), generator=gen(2)).to(IO[io])
    dev = buf.to(DEV)
    q, k = dev[:, :4, off:off + 64], dev[:, 4:6, off:off + 64]
    pos, freq = torch.arange(6, dtype=torch.int32) * 911, jy.rope_frequencies(48, 500000.0, device="cpu")
    assert jy.rope(q, k, pos.to(DEV), freq.to(DEV), layout=layout, out=(q, k))[0] is q
    check(q, *turned(buf[:, :4, off:off + 64], pos, freq, layout))
    check(k, *turned(buf[:, 4:6, off:off + 64], pos, freq, layout))
    left = dev.cpu()
    left[:, :6, off:off + 64] = buf[:, :6, off:off + 64]
    assert torch.equal(left, buf)


def test_what_is_not_finite_stays_in_its_pair(jy):
    x = torch.randn((2, 2, 64), generator=gen(3))
    x[0, 1, 5], x[1, 0, 40], x[1, 1, 63] = math.inf, math.nan, -math.inf
    freq = jy.rope_frequencies(32, device="cpu")
    pos = torch.tensor([3, 4], dtype=torch.int32)
    y = jy.rope(x.to(DEV), None, pos.to(DEV), freq.to(DEV))[0].cpu()
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 1, [5, 21]] = want[1, 0, 40] = want[1, 1, 63] = True
    assert torch.equal(bad, want) and y[1, 1, 63] == -math.inf


def test_another_stream_and_a_replayed_graph(jy):
    x = torch.randn((33, 4, 64), generator=gen(4), dtype=torch.float32).to(DEV)
    pos, freq = torch.arange(33, dtype=torch.int32, device=DEV), jy.rope_frequencies(64, device=DEV)
    want = jy.rope(x, None, pos, freq)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = jy.rope(x, None, pos, freq)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        jy.rope(x, None, pos, freq, out=(out, None))
    for i in range(4):
        x.add_(1.0)
        pos.add_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, jy.rope(x, None, pos, freq)[0])


def test_no_rows(jy):
    e = torch.empty((0, 2, 64), device=DEV)
    q, k = jy.rope(e, e, torch.empty(0, dtype=torch.int32, device=DEV), jy.rope_frequencies(64, device=DEV))
    assert q.shape == k.shape == (0, 2, 64)
