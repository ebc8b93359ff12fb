"""Eviction from sequences whose weights do not fit a workgroup's memory (over 35840 positions), against sorting."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_evict import DEV, gen, ints, jy, paged, run  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [35839, 35840, 35841, 50001])
@pytest.mark.parametrize("keep", [1, 40, 16384, 16385, 33000])
def test_lengths(jy, n, keep):
    """both sides of the limit; lists of one chunk of 16384 and of several"""
    w = torch.exp(2 * torch.randn((1, 1, n), generator=gen(n)))
    run(jy, "i4", [n], 1, 32, 256, keep, min(keep, 30), w)


@pytest.mark.parametrize("keep", [100, 17000, 30000])
def test_ties_across_chunks(jy, keep):
    """a few weights that are equal over the whole length: of the border's the first stay, chunks on"""
    w = (torch.randn((1, 2, 50001), generator=gen(2))).round()
    run(jy, "i8", [50001], 2, 16, 256, keep, 64, w)
    run(jy, "i8", [50001], 2, 16, 256, keep, 0, torch.full_like(w, 0.5))


def test_holes_short_weights_and_several_sequences(jy):
    g = gen(3)
    w = torch.rand((3, 1, 41000), generator=g)
    gone = [(0, 0), (0, 64), (0, 65), (0, 150), (2, 3)]
    run(jy, "f16", [41000, 36000, 1000], 1, 16, 256, 20000, 300, w, gone=gone, strided=True)
    run(jy, "f16", [41000, 36000, 1000], 1, 16, 256, 20000, 300, w[:, :, :17001].contiguous(), gone=gone, cols=18001)
    run(jy, "f16", [41000, 36000, 1000], 1, 16, 256, 37000, 37000, w, max_len=36001)


@pytest.mark.parametrize("keep", [3000, 16385, 40000])
def test_weights_in_place(jy, keep):
    """new weights in the old ones' place, written while later ones are still to be read"""
    lens = [50001, 36000]
    w = torch.rand((2, 2, 50001), generator=gen(7))
    w[:, 1] = (w[:, 1] * 50).round()
    want = run(jy, "i8", lens, 2, 16, 256, keep, 100, w)
    g = gen(7)
    tables, used = paged(lens, 256, g)
    to, fresh = paged([keep, keep], 256, g, lead=used)
    p = jy.PagePool.empty(1, used + fresh, 256, 2, 16, device=DEV)
    mine = w.to(DEV)
    got = p.evict(0, mine, tables.to(DEV), ints(lens), keep, 100, 50001, to.to(DEV), new_weights=mine)
    assert got[2] is mine and all(torch.equal(a, b) for a, b in zip(got, want))
