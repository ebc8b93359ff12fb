"""jyhip_rope refuses what it cannot run before anything reaches a device; rope_frequencies' rules."""
import math

import pytest

import jieyu_amd
from jieyu_amd import batch as B


@pytest.fixture(scope="module")
def b():
    return B._bind()


def vectors(address=0x10000, row=128, head=64):
    return B._Vectors(address, row, head)


def call(b, **over):
    d = dict(q=vectors(), qo=vectors(), nh=2, k=vectors(), ko=vectors(), nkv=1, rows=3, hd=64, pos=0x20000, freq=0x30000, pairs=32,
             interleaved=0, factor=1.0, type=B.T_F32, device=0, stream=None)
    d.update(over)
    return b.rope(*d.values())


@pytest.mark.parametrize("over,text", [
    (dict(type=B.T_I8), "type"), (dict(type=B.T_I4), "type"), (dict(rows=-1), "negative"), (dict(nh=-1), "negative"),
    (dict(nkv=-2), "negative"), (dict(hd=1), "head_dim"), (dict(hd=1025), "head_dim"), (dict(pairs=0), "pairs"),
    (dict(pairs=33), "pairs"), (dict(pairs=1 << 30), "pairs"), (dict(pos=None), "NULL"), (dict(freq=None), "NULL"),
    (dict(freq=0x30004), "aligned"), (dict(q=vectors(None)), "q is NULL"), (dict(qo=vectors(None)), "q_out is NULL"),
    (dict(k=vectors(None)), "k is NULL"), (dict(ko=vectors(0x10002)), "k_out is not aligned"), (dict(q=vectors(row=-1)), "negative stride"),
    (dict(nh=1 << 20), "2^20"), (dict(rows=(1 << 31) - 1, hd=1024, pairs=512), "too many rows")])
def test_refused(b, over, text):
    assert call(b, **over) == -1
    assert text in b.error().decode()


def test_nothing_to_do(b):
    assert call(b, rows=0) == 0 and call(b, nh=0, nkv=0) == 0


def test_python_refusals():
    import torch
    x = torch.zeros((2, 2, 64))
    with pytest.raises(jieyu_amd.JyError, match="device tensor"):
        jieyu_amd.rope(x, None, torch.zeros(2, dtype=torch.int32), torch.zeros(32, dtype=torch.float64))


def test_frequencies():
    f = jieyu_amd.rope_frequencies
    base = f(64, 10000.0, device="cpu")
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert base.tolist() == pytest.approx(want, rel=1e-14)
    assert f(64, 10000.0, "linear", 4.0, device="cpu").tolist() == pytest.approx([w / 4 for w in want], rel=1e-14)
    b = f(64, 10000.0, "base", 4.0, device="cpu").tolist()
    assert b[0] == 1.0 and b[-1] == pytest.approx(want[-1] / 4, rel=1e-12)
    r = f(64, 10000.0, "ramp", 8.0, trained=1000, low=1.0, high=4.0, device="cpu").tolist()
    for a, w in zip(r, want):
        turns = 1000 * w / (2 * math.pi)
        mix = min(1.0, max(0.0, (turns - 1) / 3))
        assert a == pytest.approx(w * mix + w / 8 * (1 - mix), rel=1e-12)
    assert f(2, device="cpu").tolist() == [1.0]
    for bad in (dict(dim=3), dict(dim=0), dict(dim=4, theta=-1.0), dict(dim=4, factor=0.0), dict(dim=4, scaling="ramp"),
                dict(dim=4, scaling="ramp", trained=9, low=2.0, high=2.0), dict(dim=4, scaling="other")):
        with pytest.raises(jieyu_amd.JyError):
            f(device="cpu", **bad)
