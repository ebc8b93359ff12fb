"""Writing 4-bit pages in calls of tens of thousands of vectors, byte by byte against the format's rule."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged4 import DEV, IO, gen, held4, jy, packed4  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,nkv", [(4095, 8), (4096, 8), (4097, 8), (10923, 3), (32769, 1)])
@pytest.mark.parametrize("hd,off,io", [(64, 0, "f32"), (128, 0, "bf16"), (128, 1, "f16"), (48, 3, "bf16"), (256, 0, "f16")])
def test_rows(jy, rows, nkv, hd, off, io):
    """odd numbers of vectors, idle rows and holes beside live ones, heads that start anywhere; slots beside them stay"""
    page, g = 64, gen(rows + hd)
    fused = torch.randn((rows, 2, nkv, hd + off), generator=g).to(IO[io])
    kv = fused[..., off:]
    need = -(-rows // page)
    table = torch.randperm(need + 1, generator=g)[:need].int()
    table[need // 2] = -1
    table[need - 1 if need % 2 else 0] = 1 << 30
    pos = torch.randperm(rows, generator=g).int()
    pos[::7] = -1
    p = jy.PagePool.empty(1, need + 1, page, nkv, hd, dtype=torch.uint8, device=DEV)
    for t in (p.k, p.v, p.k_scale.view(torch.int16), p.v_scale.view(torch.int16)):
        t.fill_(0x5a)
    dev = fused.to(DEV)
    k, v = dev[:, 0, :, off:], dev[:, 1, :, off:]
    seq = torch.zeros(rows, dtype=torch.int32, device=DEV)
    p.write(0, k, v, table[None].to(DEV), pos.to(DEV), seq)
    back = p.read(0, table[None].to(DEV), pos.to(DEV), seq, dtype=IO[io])
    where = torch.where(pos >= 0, table[pos.clamp(min=0).long() // page].long(), -1)
    live = (where >= 0) & (where <= need)
    pg, slot = where[live], (pos[live] % page).long()
    for side, (have, words, got) in enumerate(((p.k, p.k_scale, back[0]), (p.v, p.v_scale, back[1]))):
        values, numbers, w = held4(kv[:, side].float())
        b = packed4(numbers)
        wantb, wantw = torch.full_like(have.cpu(), 0x5a), torch.full_like(words.cpu().view(torch.int16), 0x5a)
        wantb[0, pg, :, slot] = b[live]
        wantw[0, pg, :, slot] = w[live].view(torch.int16)
        values[~live] = 0.0
        assert torch.equal(have.cpu(), wantb)
        assert torch.equal(words.cpu().view(torch.int16), wantw)
        assert torch.equal(got.cpu(), values.float().to(IO[io]))
