"""Operators of a decode step over several sequences at once (include/jieyu_amd.h), on torch
tensors in device memory: a paged key/value cache, attention over it, and sampling.

Everything runs on torch's current stream of the tensors' device and nothing waits for it, so
calls can be recorded into a graph.  Workspaces come from torch's allocator, call by call.  There are
no gradients: what comes out is not connected to what went in.
"""
import ctypes as C
import math

from . import JyError, lib

P = C.c_void_p
I = C.c_int
LL = C.c_longlong

T_F32, T_F16, T_BF16, T_I8 = 0, 1, 2, 3


class _Pages(C.Structure):
    _fields_ = [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("num_pages", I), ("page_size", I),
                ("num_kv_heads", I), ("head_dim", I), ("type", I), ("device", I)]


class _Tables(C.Structure):
    _fields_ = [("tables", P), ("num_seqs", I), ("table_stride", I)]


class _Vectors(C.Structure):
    _fields_ = [("data", P), ("row_stride", LL), ("head_stride", LL)]


_bound = None


class _Bound:
    """torch, its types by number, and the library's entry points with their prototypes."""

    def __init__(self):
        import torch
        L = lib()
        self.torch, self.int32 = torch, torch.int32
        self.io = {torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16}
        self.pool = {torch.int8: T_I8, torch.float16: T_F16, torch.bfloat16: T_BF16}
        # the address of the current stream of device i (without torch.cuda.Stream's object around it,
        # where this torch has that)
        self.stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: torch.cuda.current_stream(i).cuda_stream)

        def proto(name, res, *args):
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, list(args)
            return fn

        ref = C.POINTER
        moved = (ref(_Pages), ref(_Tables), I, P, P, ref(_Vectors), ref(_Vectors), I, P)
        self.write = proto("jyhip_pages_write", I, *moved)
        self.read = proto("jyhip_pages_read", I, *moved)
        self.attend = proto("jyhip_pages_attend", I, ref(_Pages), ref(_Tables), P, I, I, C.c_float, ref(_Vectors),
                            ref(_Vectors), I, P, C.c_size_t, P)
        self.attend_workspace = proto("jyhip_pages_attend_workspace", C.c_size_t, ref(_Pages), I, I, I)
        self.sample = proto("jyhip_sample", I, P, I, I, I, LL, P, P, P, P, P, P, P, C.c_size_t, I, P)
        self.sample_workspace = proto("jyhip_sample_workspace", C.c_size_t, I, I)
        self.error = L.jyhip_last_error


def _bind():
    global _bound
    if _bound is None:
        _bound = _Bound()
    return _bound


def _failed(b):
    raise JyError(b.error().decode("utf-8", "replace"))


def _indices(b, t, n, device, name):
    """The address of n int32 values."""
    if t.dtype is not b.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise JyError(f"{name}: {n} contiguous int32 values on {device} are needed")
    return t.data_ptr()


class PagePool:
    """The pages of a key/value cache: k, v [layers][pages][kv heads][page size][head size] in int8
    (then with fp32 scales [layers][pages][kv heads][page size]), float16 or bfloat16.  The tensors
    stay the caller's, and the pool keeps a reference to them.

    `tables` (int32 [sequences][pages of each]) says which page holds a sequence's positions; an id
    outside the pool is a hole: its positions are not written, read as zeros, and left out of the
    attention."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        b = self._b = _bind()
        if k.dim() != 5 or not k.is_cuda or k.dtype not in b.pool:
            raise JyError("pool: k and v are device tensors [layers][pages][kv heads][page size][head size] in int8, "
                          "float16 or bfloat16")
        for t, shape, dtype, name in ((k, k.shape, k.dtype, "k"), (v, k.shape, k.dtype, "v"),
                                      (k_scale, k.shape[:4], b.torch.float32, "k_scale"),
                                      (v_scale, k.shape[:4], b.torch.float32, "v_scale")):
            if t is None and name.endswith("scale") and k.dtype is not b.torch.int8:
                continue
            if t is None or t.shape != shape or t.dtype is not dtype or t.device != k.device or not t.is_contiguous():
                raise JyError(f"pool: {name} must be a contiguous {dtype} tensor of {tuple(shape)} on {k.device}")
            if t is not None and name.endswith("scale") and k.dtype is not b.torch.int8:
                raise JyError("pool: 16-bit pages have no scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self.layers, self.pages, self.nkv, self.page_size, self.hd = k.shape
        if not self.layers or not self.pages or not self.nkv:
            raise JyError("pool: no pages")

        def at(t, i):
            return None if t is None else t.data_ptr() + t.stride(0) * t.element_size() * i

        self._layers = [_Pages(at(k, i), at(v, i), at(k_scale, i), at(v_scale, i), self.pages, self.page_size, self.nkv,
                               self.hd, b.pool[k.dtype], k.device.index) for i in range(self.layers)]

    @classmethod
    def empty(cls, layers, pages, page_size, num_kv_heads, head_dim, dtype=None, device="cuda"):
        """A new pool, int8 unless `dtype` says otherwise, without any contents of its own."""
        torch = _bind().torch
        dtype = dtype or torch.int8
        shape = (layers, pages, num_kv_heads, page_size, head_dim)
        new = lambda s, t: torch.empty(s, dtype=t, device=device)  # noqa: E731
        scales = [new(shape[:4], torch.float32) for _ in range(2)] if dtype is torch.int8 else [None, None]
        return cls(new(shape, dtype), new(shape, dtype), *scales)

    def _layer(self, layer):
        if not 0 <= layer < self.layers:
            raise JyError("pool: layer out of range")
        return self._layers[layer]

    def _tables(self, t):
        shape = t.shape
        if t.dtype is not self._b.int32 or len(shape) != 2 or t.device != self.device or not t.is_contiguous():
            raise JyError(f"tables: a contiguous int32 tensor [sequences][pages] on {self.device} is needed")
        return _Tables(t.data_ptr(), *shape)

    def _vectors(self, t, shape, dtype, name):
        if t.shape != shape or t.dtype is not dtype or t.device != self.device:
            raise JyError(f"{name}: a {dtype} tensor of {shape} on {self.device} is needed")
        row, head, one = t.stride()
        if one != 1:
            raise JyError(f"{name}: a vector's elements must lie side by side")
        return _Vectors(t.data_ptr(), row, head)

    def _move(self, fn, layer, k, v, tables, pos, seq):
        b, device, dtype, shape = self._b, self.device, k.dtype, k.shape
        code = b.io.get(dtype)
        if code is None or len(shape) != 3:
            raise JyError("k and v: float32, float16 or bfloat16 [rows][kv heads][head size]")
        rows = shape[0]
        shape = (rows, self.nkv, self.hd)
        pages = self._layer(layer)
        K, V = self._vectors(k, shape, dtype, "k"), self._vectors(v, shape, dtype, "v")
        at = None if seq is None else _indices(b, seq, rows, device, "seq")
        p = _indices(b, pos, rows, device, "pos")
        if rows and fn(pages, self._tables(tables), rows, at, p, K, V, code, b.stream(device.index)) != 0:
            _failed(b)

    def write(self, layer, k, v, tables, pos, seq=None):
        """Hold keys and values k, v [rows][kv heads][head size] (float32, float16 or bfloat16) as
        position pos[r] of sequence seq[r] (without seq: of sequence r).  A row whose position does
        not exist (-1 in a padded batch) is skipped; the rows of a call are different positions."""
        self._move(self._b.write, layer, k, v, tables, pos, seq)

    def read(self, layer, tables, pos, seq=None, dtype=None, out=None):
        """(k, v) of the same positions as values, float32 unless `dtype` or `out` (a pair of
        tensors) says otherwise; zeros where there is no such position."""
        if out is None:
            shape = (pos.shape[0], self.nkv, self.hd)
            dtype = dtype or self._b.torch.float32
            out = [self.k.new_empty(shape, dtype=dtype) for _ in range(2)]
        self._move(self._b.read, layer, out[0], out[1], tables, pos, seq)
        return out[0], out[1]

    def attend(self, layer, q, tables, lens, max_len, scale=None, out=None):
        """Attention of q [sequences][heads][head size], one row per sequence, over the first lens[s]
        (int32) positions of each; zeros for a sequence without any.  `max_len`, an upper bound of
        lens, sizes the launch: a longer one is cut to it.  scale: 1 / sqrt(head size) unless given."""
        b = self._b
        pages, T = self._layer(layer), self._tables(tables)
        code = b.io.get(q.dtype)
        if code is None or q.dim() != 3:
            raise JyError("q: float32, float16 or bfloat16 [sequences][heads][head size]")
        batch, heads, _ = q.shape
        if out is None:
            out = q.new_empty((batch, heads, self.hd))
        shape = (batch, heads, self.hd)
        Q, O = self._vectors(q, shape, q.dtype, "q"), self._vectors(out, shape, q.dtype, "out")
        n = _indices(b, lens, batch, self.device, "lens")
        if T.num_seqs != batch:
            raise JyError("attend: one query row for each sequence of the tables")
        if not 0 <= max_len <= 1 << 30:
            raise JyError("attend: max_len must be between 0 and 2^30")
        if not batch:
            return out
        need = b.attend_workspace(pages, batch, heads, max_len)
        ws = q.new_empty(need, dtype=b.torch.uint8) if need else None
        if b.attend(pages, T, n, max_len, heads, 1.0 / math.sqrt(self.hd) if scale is None else scale, Q, O, code,
                    ws.data_ptr() if need else None, need, b.stream(self.device.index)) != 0:
            _failed(b)
        return out


def _settings(b, t, rows, device, dtype, name):
    """The address of one setting per row (None: off)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != (rows,) or t.device != device or not t.is_contiguous():
        raise JyError(f"sample: {name} must be {rows} contiguous {dtype} values on {device}")
    return t.data_ptr()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token id (int32) for each row of logits [rows][vocab] (float32, float16 or bfloat16) from
    the rows' random numbers u in [0, 1) and settings, device tensors of one value per row: float32
    temperature (<= 0: the largest logit; None: 1), int32 top_k (<= 0 or None: off), float32 top_p
    (>= 1 or None: off) and min_p (<= 0 or None: off), applied in this order.  -1 for a row without
    any logit above -infinity.  jyhip_sample in include/jieyu_amd.h says it to the letter."""
    b = _bind()
    torch, dev = b.torch, logits.device
    code = b.io.get(logits.dtype)
    if code is None or logits.dim() != 2 or not logits.is_cuda:
        raise JyError("sample: logits are a device tensor [rows][vocab] in float32, float16 or bfloat16")
    rows, vocab = logits.shape
    if vocab and logits.stride(1) != 1:
        raise JyError("sample: a row's logits must lie side by side")
    if out is None:
        out = logits.new_empty(rows, dtype=torch.int32)
    f = torch.float32
    args = [_settings(b, u, rows, dev, f, "u"), _settings(b, temperature, rows, dev, f, "temperature"),
            _settings(b, top_k, rows, dev, torch.int32, "top_k"), _settings(b, top_p, rows, dev, f, "top_p"),
            _settings(b, min_p, rows, dev, f, "min_p"), _settings(b, out, rows, dev, torch.int32, "out")]
    if not rows:
        return out
    need = b.sample_workspace(rows, vocab)
    ws = logits.new_empty(need, dtype=torch.uint8) if need else None
    if b.sample(logits.data_ptr(), code, rows, vocab, logits.stride(0), *args, ws.data_ptr() if need else None, need,
                dev.index, b.stream(dev.index)) != 0:
        _failed(b)
    return out


__all__ = ["PagePool", "sample"]
