"""The paged cache's entry points refuse what they cannot run, before anything reaches a device."""
import ctypes as C

import pytest

import jieyu_amd
from jieyu_amd import batch as B


@pytest.fixture(scope="module")
def b():
    return B._bind()


def pages(**over):
    d = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, num_pages=4, page_size=16, num_kv_heads=2,
             head_dim=64, type=B.T_I8, device=0)
    d.update(over)
    return B._Pages(*(d[n] for n, _ in B._Pages._fields_))


def tables(address=0x50000, n=3, stride=2):
    return B._Tables(address, n, stride)


def vectors(address=0x60000, row=128, head=64):
    return B._Vectors(address, row, head)


def error(b):
    return b.error().decode()


def move(b, fn="write", p=None, t=None, rows=3, seq=None, pos=0x70000, k=None, v=None, type=B.T_F32):
    return getattr(b, fn)(p or pages(), t or tables(), rows, seq, pos, k or vectors(), v or vectors(), type, None)


BAD_PAGES = [(dict(k=None), "NULL k or v"), (dict(v=None), "NULL k or v"), (dict(k=0x10008), "aligned"),
             (dict(k_scale=None), "need scales"), (dict(v_scale=0x40004), "aligned"), (dict(type=B.T_F16), "no scales"),
             (dict(type=B.T_F32), "type"), (dict(type=9), "type"), (dict(num_pages=0), "positive"),
             (dict(num_kv_heads=-1), "positive"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
             (dict(page_size=512), "page_size"), (dict(head_dim=0), "head_dim"), (dict(head_dim=72), "head_dim"),
             (dict(head_dim=272), "head_dim")]


@pytest.mark.parametrize("over,text", BAD_PAGES)
@pytest.mark.parametrize("fn", ["write", "read", "attend"])
def test_bad_pages(b, fn, over, text):
    p = pages(**over)
    if fn == "attend":
        rc = b.attend(p, tables(), 0x80000, 20, 4, 0.125, vectors(), vectors(), B.T_F32, 0x90000, 1 << 30, None)
    else:
        rc = move(b, fn, p)
    assert rc == -1 and text in error(b)


@pytest.mark.parametrize("fn", ["write", "read"])
@pytest.mark.parametrize("args,text", [
    (dict(t=tables(None)), "NULL page tables"), (dict(t=tables(n=0)), "positive"), (dict(t=tables(stride=0)), "positive"),
    (dict(rows=-1), "negative"), (dict(pos=None), "pos is NULL"), (dict(rows=4), "more rows than sequences"),
    (dict(k=vectors(None)), "k is NULL"), (dict(v=vectors(None)), "v is NULL"), (dict(type=B.T_I8), "type"),
    (dict(type=-1), "type"), (dict(k=vectors(0x60002)), "k is not aligned"), (dict(v=vectors(row=-1)), "negative stride"),
    (dict(v=vectors(head=-1)), "negative stride"), (dict(rows=1 << 30, seq=0x70000), "too large")])
def test_bad_rows(b, fn, args, text):
    assert move(b, fn, **args) == -1
    assert text in error(b)


@pytest.mark.parametrize("fn", ["write", "read"])
def test_no_rows_is_no_work(b, fn):
    assert move(b, fn, rows=0) == 0


def attend(b, **over):
    d = dict(p=pages(), t=tables(), lens=0x80000, max_len=20, heads=4, scale=0.125, q=vectors(row=256),
             out=vectors(row=256), type=B.T_F32, ws=0x90000, bytes=1 << 30)
    d.update(over)
    return b.attend(d["p"], d["t"], d["lens"], d["max_len"], d["heads"], d["scale"], d["q"], d["out"], d["type"], d["ws"],
                    d["bytes"], None)


@pytest.mark.parametrize("over,text", [
    (dict(lens=None), "lens is NULL"), (dict(max_len=-1), "max_len"), (dict(heads=0), "multiple"), (dict(heads=3), "multiple"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(q=vectors(None)), "q is NULL"),
    (dict(out=vectors(None)), "out is NULL"), (dict(type=B.T_I8), "type"), (dict(out=vectors(0x60001)), "not aligned"),
    (dict(t=tables(n=-2)), "positive")])
def test_bad_attention(b, over, text):
    assert attend(b, **over) == -1
    assert text in error(b)


def test_lengths_whose_chunks_pass_an_int(b):
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        assert attend(b, max_len=n) == -1 and "2^30" in error(b)
        assert b.attend_workspace(pages(), 1, 4, n) == 0
    assert 0 < b.attend_workspace(pages(), 1, 4, 1 << 30) < 1 << 32


def test_null_structs(b):
    none = C.POINTER(B._Pages)()
    assert b.write(none, tables(), 1, None, 0x1000, vectors(), vectors(), B.T_F32, None) == -1
    assert "pages is NULL" in error(b)
    assert b.read(pages(), C.POINTER(B._Tables)(), 1, None, 0x1000, vectors(), vectors(), B.T_F32, None) == -1
    assert "NULL page tables" in error(b)
    assert b.attend_workspace(none, 1, 1, 1) == 0


def test_pool_wants_device_tensors():
    import torch
    x = torch.zeros((1, 2, 2, 16, 64), dtype=torch.int8)
    with pytest.raises(jieyu_amd.JyError, match="device tensors"):
        jieyu_amd.PagePool(x, x, torch.zeros(1, 2, 2, 16), torch.zeros(1, 2, 2, 16))


@pytest.mark.parametrize("nkv,heads", [(4, 2), (4, 1), (8, 7), (4, 6), (3, 2)])
@pytest.mark.parametrize("max_len", [1, 1000, 1025, 2000, 1 << 30])
def test_workspace_of_heads_that_are_refused(b, nkv, heads, max_len):
    """fewer query heads than key/value heads, or no multiple of them: no workspace at any length, and
    attend says why"""
    p = pages(num_kv_heads=nkv)
    assert b.attend_workspace(p, 1, heads, max_len) == 0
    assert attend(b, p=p, heads=heads, max_len=max_len, ws=None, bytes=0) == -1 and "multiple" in error(b)
    for hd in (0, -16, 272):
        assert b.attend_workspace(pages(head_dim=hd), 1, 4, max_len) == 0


@pytest.mark.parametrize("fn", ["write", "read"])
@pytest.mark.parametrize("nkv,rows", [(1, (1 << 28) - 15), (1, 1 << 28), (2, (1 << 27) - 7), (8, (1 << 25) - 1), (3, 89478481)])
def test_rows_past_one_launch(b, fn, nkv, rows):
    """more than 2^28 - 16 rows x heads, 16 threads each, would be 2^32 threads"""
    assert move(b, fn, p=pages(num_kv_heads=nkv), rows=rows, seq=0x70000) == -1
    assert "too large" in error(b)


def paged_pass(**over):
    """GpuModel.forward_paged of a model and a pool that only have their shapes: what it refuses before it
    comes to a device."""
    np = pytest.importorskip("numpy")
    g = jieyu_amd.GpuModel.__new__(jieyu_amd.GpuModel)
    g.h, g.num_layers, g.hidden = None, 1, 8
    pool = type("Pool", (), dict(layers=1, device=None, _layers=[]))()
    d = dict(tables=[[0, 1], [2, 3]], pos=[3, 4], seq=[0, 1])
    d.update(over)
    return g.forward_paged(pool, np.zeros((2, 8), np.float32), d["tables"], d["pos"], d["seq"])


@pytest.mark.parametrize("name,value", [("pos", [3, 1 << 32]), ("pos", [3.5, 4.0]), ("pos", [3, float("nan")]), ("seq", [0, (1 << 32) + 1]),
                                        ("tables", [[0, 1], [2, -(1 << 31) - 1]]), ("tables", [[0, 1e20]] * 2)])
@pytest.mark.parametrize("as_array", [False, True])
def test_indices_that_would_wrap_around(name, value, as_array):
    """an index of 64 bits is not cut to its lower 32, a fraction not to a whole number"""
    np = pytest.importorskip("numpy")
    with pytest.raises(jieyu_amd.JyError, match=name + ": whole numbers"):
        paged_pass(**{name: np.array(value) if as_array else value})


def test_indices_of_other_whole_types():
    np = pytest.importorskip("numpy")
    for t in (np.int64, np.uint32, np.int16, np.uint8, np.int32, np.float64):
        got = jieyu_amd._int32s(np.array([[0, 7], [3, 100]], t)[:, ::-1], "tables")
        assert got.dtype == np.int32 and got.flags.c_contiguous and got.tolist() == [[7, 0], [100, 3]]
    assert jieyu_amd._int32s([], "pos").shape == (0,) and jieyu_amd._int32s([-1, (1 << 31) - 1], "pos").tolist() == [-1, (1 << 31) - 1]
