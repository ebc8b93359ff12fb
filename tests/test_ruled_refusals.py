"""What the entry points of masked attention, 4-bit pages and eviction refuse, before anything reaches a device."""
import ctypes as C

import pytest

import jieyu_amd
from jieyu_amd import batch as B


@pytest.fixture(scope="module")
def b():
    return B._bind()


def pages(**over):
    d = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, num_pages=4, page_size=16, num_kv_heads=2,
             head_dim=64, type=B.T_I4, device=0)
    d.update(over)
    return B._Pages(*(d[n] for n, _ in B._Pages._fields_))


def tables(address=0x50000, n=3, stride=2):
    return B._Tables(address, n, stride)


def vectors(address=0x60000, row=128, head=64):
    return B._Vectors(address, row, head)


def rules(cap=0.0, slopes=None, first=None, last=None):
    return B._Rules(cap, slopes, first, last)


def one(b, **over):
    d = dict(p=pages(), t=tables(), lens=0x80000, max_len=20, heads=4, scale=0.125, rules=None, q=vectors(row=256),
             out=vectors(row=256), type=B.T_F32, w=None, ws=0, hs=0, wn=0, work=0x90000, bytes=1 << 30, stream=None)
    d.update(over)
    return b.attend_ruled(*d.values())


def rows(b, **over):
    d = dict(p=pages(), t=tables(), starts=0x80000, pos=0x81000, rows=5, max_len=20, heads=4, scale=0.125, rules=None,
             q=vectors(row=256), out=vectors(row=256), type=B.T_F32, work=0x90000, bytes=1 << 30, stream=None)
    d.update(over)
    return b.attend_rows(*d.values())


def evict(b, **over):
    d = dict(p=pages(), t=tables(), to=tables(0x51000), lens=0x80000, new=0x80100, max_len=32, keep=8, recent=2, w=0x81000, ws=64,
             hs=32, wn=32, nw=None, ns=0, nh=0, nn=0, kept=0x82000, stream=None)
    d.update(over)
    return b.evict(*d.values())


BOTH = [(dict(max_len=-1), "max_len"), (dict(max_len=(1 << 30) + 1), "2^30"), (dict(heads=0), "multiple"), (dict(heads=3), "multiple"),
        (dict(scale=float("nan")), "finite"), (dict(q=vectors(None)), "q is NULL"), (dict(out=vectors(0x60002)), "not aligned"),
        (dict(type=B.T_I4), "type"), (dict(type=B.T_I8), "type"), (dict(rules=rules(cap=-1.0)), "cap"),
        (dict(rules=rules(cap=float("nan"))), "cap"), (dict(rules=rules(cap=float("inf"))), "cap"),
        (dict(rules=rules(cap=1e-45), scale=1e30), "over the cap"), (dict(rules=rules(slopes=0x7)), "aligned"),
        (dict(rules=rules(first=0x2)), "aligned"), (dict(t=tables(None)), "NULL page tables"), (dict(p=pages(k_scale=None)), "need scales"),
        (dict(p=pages(head_dim=72)), "head_dim"), (dict(p=pages(v_scale=0x30008)), "aligned")]


@pytest.mark.parametrize("over,text", BOTH + [
    (dict(lens=None), "lens is NULL"), (dict(rules=rules(last=0x1000)), "last"), (dict(w=0x1002), "aligned"),
    (dict(w=0x1000, ws=-1), "negative stride"), (dict(w=0x1000, wn=-1), "length"), (dict(w=0x1000, work=None), "workspace"),
    (dict(max_len=5000, work=0x90004), "workspace"), (dict(max_len=5000, bytes=1000), "workspace"),
    (dict(t=tables(n=1 << 24)), "too many")])
def test_single_rows(b, over, text):
    assert one(b, **over) == -1
    assert text in b.error().decode()


@pytest.mark.parametrize("over,text", BOTH + [
    (dict(starts=None), "NULL starts"), (dict(pos=None), "NULL starts or pos"), (dict(rows=-1), "negative"),
    (dict(rows=1 << 24, bytes=1 << 50), "too many")])
def test_runs(b, over, text):
    assert rows(b, **over) == -1
    assert text in b.error().decode()


def test_no_rows_is_no_work(b):
    assert rows(b, rows=0) == 0
    assert rows(b, rows=0, t=tables(None)) == -1


def test_workspaces(b):
    w, r = b.attend_ruled_workspace, b.attend_rows_workspace
    p = pages()
    for bad in (dict(heads=3), dict(heads=0), dict(n=0), dict(max_len=-1), dict(max_len=(1 << 30) + 1)):
        d = dict(n=3, heads=4, max_len=100)
        d.update(bad)
        assert w(p, d["n"], d["heads"], d["max_len"], 1, 1) == 0
        assert r(p, d["n"], 10, d["heads"], d["max_len"], B.T_F32) == 0
    assert r(p, 3, 0, 4, 100, B.T_F32) == 0 and w(C.POINTER(B._Pages)(), 1, 1, 1, 0, 0) == 0
    assert w(p, 3, 4, 0, 0, 1) > 0 and w(p, 3, 4, 100, 0, 0) == 0 and w(p, 3, 4, 100, 1, 1) >= 3 * 4 * 132 * 4
    assert w(p, 1, 4, 1 << 30, 1, 1) > 1 << 32
    assert b.attend_workspace(p, 3, 4, 5000) > 0


@pytest.mark.parametrize("over,text", [
    (dict(lens=None), "NULL lens"), (dict(new=None), "NULL lens"), (dict(w=None), "NULL"), (dict(kept=None), "NULL"),
    (dict(new=0x80000), "apart"), (dict(kept=0x82002), "aligned"), (dict(max_len=-1), "max_len"), (dict(keep=0), "keep"),
    (dict(keep=(1 << 30) + 1), "keep"), (dict(recent=-1), "recent"), (dict(recent=9), "recent"), (dict(ws=-1), "negative"),
    (dict(wn=-1), "negative"), (dict(nn=-3), "negative"), (dict(to=tables(n=2)), "other sequences"), (dict(to=tables(None)), "NULL"),
    (dict(keep=32, to=tables(stride=1)), "too few pages"), (dict(p=pages(type=B.T_F32)), "type"),
    (dict(t=tables(n=1 << 21), to=tables(n=1 << 21)), "too large"), (dict(t=tables(n=1 << 20, stride=99), to=tables(n=1 << 20, stride=99),
                                                                          keep=1000, max_len=1000), "too large")])
def test_evictions(b, over, text):
    assert evict(b, **over) == -1
    assert text in b.error().decode()


def test_4bit_pools_want_their_layout():
    torch = pytest.importorskip("torch")
    x = torch.zeros((1, 2, 2, 16, 32), dtype=torch.uint8)
    with pytest.raises(jieyu_amd.JyError, match="device tensors"):
        jieyu_amd.PagePool(x, x, None, None)


@pytest.mark.parametrize("ws,hs,wn,ok", [(0, 32, 32, False), (64, 0, 32, False), (64, 32, 33, False), (63, 32, 32, False), (32, 96, 32, True),
                                         (32, 95, 32, False), (31, 96, 32, False), (1 << 62, 1 << 62, 5, False), (0, 0, 0, True)])
def test_weights_that_are_written_share_no_elements(b, ws, hs, wn, ok):
    """3 sequences of 2 heads, in either order"""
    bad = dict(bytes=0, max_len=5000) if ok else {}  # (good strides reach the check of the workspace)
    assert one(b, w=0x1000, ws=ws, hs=hs, wn=wn, **bad) == -1
    assert ("workspace" if ok else "share") in b.error().decode()
    if not ok:
        assert evict(b, nw=0x1000, ns=ws, nh=hs, nn=wn) == -1
        assert "share" in b.error().decode()
