"""jyhip_sample refuses what it cannot run before anything reaches a device."""
import pytest

from jieyu_amd import batch as B


@pytest.fixture(scope="module")
def b():
    return B._bind()


def call(b, **over):
    d = dict(logits=0x10000, type=B.T_F32, rows=2, vocab=100, stride=100, u=0x20000, T=None, k=None, p=None, m=None,
             ids=0x30000, ws=0x40000, bytes=1 << 30, device=0, stream=None)
    d.update(over)
    return b.sample(*d.values())


@pytest.mark.parametrize("over,text", [
    (dict(type=B.T_I8), "type"), (dict(type=7), "type"), (dict(rows=-1), "negative"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 22) + 1), "vocab"), (dict(rows=1 << 21), "too many"), (dict(logits=None), "NULL"),
    (dict(u=None), "NULL"), (dict(ids=None), "NULL"), (dict(logits=0x10002), "aligned"), (dict(stride=-1), "negative")])
def test_refused(b, over, text):
    assert call(b, **over) == -1
    assert text in b.error().decode()


def test_no_rows_is_no_work(b):
    assert call(b, rows=0) == 0


def test_workspace_of_what_is_refused(b):
    assert b.sample_workspace(0, 10) == b.sample_workspace(1, 0) == b.sample_workspace(1, (1 << 22) + 1) == 0
