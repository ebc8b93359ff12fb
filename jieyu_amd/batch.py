"""Operators of a step over several sequences at once (include/jieyu_amd.h), on torch tensors in device
memory: rotary positions, a paged key/value cache (down to 4 bits an element), attention of single rows and of
runs of rows over it, eviction from it, and sampling.

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

T_F32, T_F16, T_BF16, T_I8, T_I4 = 0, 1, 2, 3, 4


class _Pages(C.Structure):
    _fields_ = [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("num_pages", I), ("page_size", I),
                ("num_kv_heads", I), ("head_dim", I), ("type", I), ("device", I)]


class _Tables(C.Structure):
    _fields_ = [("tables", P), ("num_seqs", I), ("table_stride", I)]


class _Vectors(C.Structure):
    _fields_ = [("data", P), ("row_stride", LL), ("head_stride", LL)]


class _Rules(C.Structure):
    _fields_ = [("cap", C.c_float), ("slopes", P), ("first", P), ("last", P)]


_bound = None


class _Bound:
    """torch, its types by number, and the library's entry points with their prototypes."""

    def __init__(self):
        import torch
        L = lib()
        self.torch, self.int32 = torch, torch.int32
        self.io = {torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16}
        self.pool = {torch.uint8: T_I4, torch.int8: T_I8, torch.float16: T_F16, torch.bfloat16: T_BF16}
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
        rules, seen = ref(_Rules), (ref(_Vectors), ref(_Vectors), I)
        self.attend_ruled = proto("jyhip_pages_attend_ruled", I, ref(_Pages), ref(_Tables), P, I, I, C.c_float, rules, *seen, P,
                                  LL, LL, I, P, C.c_size_t, P)
        self.attend_ruled_workspace = proto("jyhip_pages_attend_ruled_workspace", C.c_size_t, ref(_Pages), I, I, I, I, I)
        self.attend_rows = proto("jyhip_pages_attend_rows", I, ref(_Pages), ref(_Tables), P, P, I, I, I, C.c_float, rules, *seen,
                                 P, C.c_size_t, P)
        self.attend_rows_workspace = proto("jyhip_pages_attend_rows_workspace", C.c_size_t, ref(_Pages), I, I, I, I, I)
        self.evict = proto("jyhip_pages_evict", I, ref(_Pages), ref(_Tables), ref(_Tables), P, P, I, I, I, P, LL, LL, I, P, LL, LL,
                           I, P, P)
        self.rope = proto("jyhip_rope", I, ref(_Vectors), ref(_Vectors), I, ref(_Vectors), ref(_Vectors), I, I, I, P, P, I, I,
                          C.c_float, I, I, P)
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


def _strided(t, shape, dtype, device, name):
    """A device tensor of vectors, for the library."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise JyError(f"{name}: a {dtype} tensor of {tuple(shape)} on {device} is needed")
    row, head, one = t.stride()
    if one != 1 and shape[2] > 1:
        raise JyError(f"{name}: a vector's elements must lie side by side")
    return _Vectors(t.data_ptr(), row, head)


def _groups4(hd):
    """groups of 32 elements that a 4-bit vector is laid out in"""
    return 2 if hd <= 64 else 4 if hd <= 128 else 8


class PagePool:
    """The pages of a key/value cache: k, v [layers][pages][kv heads][page size][head size] in int8
    (then with fp32 scales [layers][pages][kv heads][page size]), float16 or bfloat16, or in 4 bits:
    uint8 [layers][pages][kv heads][page size][16 groups], then with float16 scales [layers][pages]
    [kv heads][page size][groups][2], 2 groups for a head size up to 64, 4 up to 128, 8 up to 256 (the
    head size itself is `head_dim`, 32 groups unless given).  The tensors stay the caller's, and the
    pool keeps a reference to them.

    `tables` (int32 [sequences][pages of each]) says which page holds a sequence's positions; an id
    outside the pool is a hole: its positions are not written, read as zeros, and left out of the
    attention."""

    def __init__(self, k, v, k_scale=None, v_scale=None, head_dim=None):
        b = self._b = _bind()
        torch = b.torch
        if k.dim() != 5 or not k.is_cuda or k.dtype not in b.pool:
            raise JyError("pool: k and v are device tensors [layers][pages][kv heads][page size][head size] in int8, "
                          "4 bits (uint8), float16 or bfloat16")
        self.layers, self.pages, self.nkv, self.page_size, width = k.shape
        scales = None
        if k.dtype is torch.int8:
            scales = (torch.float32, k.shape[:4])
        elif k.dtype is torch.uint8:
            self.hd = 2 * width if head_dim is None else head_dim
            if width != 16 * _groups4(self.hd):
                raise JyError(f"pool: 4-bit vectors of {self.hd} elements take {16 * _groups4(self.hd)} bytes")
            scales = (torch.float16, (*k.shape[:4], width // 16, 2))
        if k.dtype is not torch.uint8:
            self.hd = width
            if head_dim not in (None, width):
                raise JyError("pool: head_dim is not the vectors' size")
        for t, shape, dtype, name in ((k, k.shape, k.dtype, "k"), (v, k.shape, k.dtype, "v")) + (() if scales is None else (
                (k_scale, scales[1], scales[0], "k_scale"), (v_scale, scales[1], scales[0], "v_scale"))):
            if t is None or t.shape != shape or t.dtype is not dtype or t.device != k.device or not t.is_contiguous():
                raise JyError(f"pool: {name} must be a contiguous {dtype} tensor of {tuple(shape)} on {k.device}")
        if scales is None and (k_scale is not None or v_scale is not None):
            raise JyError("pool: 16-bit pages have no scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        if not self.layers or not self.pages or not self.nkv:
            raise JyError("pool: no pages")

        def at(t, i):
            return None if t is None else t.data_ptr() + t.stride(0) * t.element_size() * i

        self._layers = [_Pages(at(k, i), at(v, i), at(k_scale, i), at(v_scale, i), self.pages, self.page_size, self.nkv,
                               self.hd, b.pool[k.dtype], k.device.index) for i in range(self.layers)]

    @classmethod
    def empty(cls, layers, pages, page_size, num_kv_heads, head_dim, dtype=None, device="cuda"):
        """A new pool, int8 unless `dtype` says otherwise (torch.uint8: 4 bits), without any contents of its own."""
        torch = _bind().torch
        dtype = dtype or torch.int8
        lead = (layers, pages, num_kv_heads, page_size)
        groups = _groups4(head_dim)
        new = lambda s, t: torch.empty(s, dtype=t, device=device)  # noqa: E731
        scales = [None, None]
        if dtype is torch.int8:
            scales = [new(lead, torch.float32) for _ in range(2)]
        if dtype is torch.uint8:
            scales = [new((*lead, groups, 2), torch.float16) for _ in range(2)]
        shape = (*lead, 16 * groups if dtype is torch.uint8 else head_dim)
        return cls(new(shape, dtype), new(shape, dtype), *scales, head_dim=head_dim)

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
        return _strided(t, shape, dtype, self.device, name)

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

    def _queries(self, q, out):
        """q's and out's vectors, their type and shape, and out"""
        code = self._b.io.get(q.dtype)
        if code is None or q.dim() != 3:
            raise JyError("q: float32, float16 or bfloat16 [rows][heads][head size]")
        rows, heads, _ = q.shape
        shape = (rows, heads, self.hd)
        if out is None:
            out = q.new_empty(shape)
        return self._vectors(q, shape, q.dtype, "q"), self._vectors(out, shape, q.dtype, "out"), code, rows, heads, out

    def _rules(self, rows, heads, cap, slopes, first, last=None):
        """The rules of a call, None without any."""
        if cap is None and slopes is None and first is None and last is None:
            return None
        b = self._b
        if slopes is not None and (slopes.dtype is not b.torch.float32 or slopes.shape != (heads,) or slopes.device != self.device
                                   or not slopes.is_contiguous()):
            raise JyError(f"slopes: {heads} contiguous float32 values on {self.device} are needed")
        if cap is not None and not C.c_float(cap).value > 0:  # (a smaller one than fp32 holds would count as none)
            raise JyError("cap: a positive number that float32 holds, or None")
        return _Rules(0.0 if cap is None else cap, None if slopes is None else slopes.data_ptr(),
                      None if first is None else _indices(b, first, rows, self.device, "first"),
                      None if last is None else _indices(b, last, rows, self.device, "last"))

    def attend(self, layer, q, tables, lens, max_len, scale=None, out=None, first=None, cap=None, slopes=None, weights=None):
        """Attention of q [sequences][heads][head size], one row per sequence, over the first lens[s]
        (int32) positions of each; zeros for a sequence without any.  `max_len`, an upper bound of
        lens, sizes the launch: a longer one is cut to it.  scale: 1 / sqrt(head size) unless given.

        first (int32): a sequence's positions before first[s] are left out, and max_len is an upper bound
        of lens - first.  cap: a score s becomes cap * tanh(s / cap).  slopes (float32 [heads]): slope times the
        distance to position lens[s] - 1 is taken off the scores.  weights (float32 [sequences][kv heads]
        [positions]): the weights of each position, summed over the query heads of a kv head, are added to it (past its
        last position they are not counted; each sequence and head has elements of its own)."""
        b = self._b
        pages, T = self._layer(layer), self._tables(tables)
        Q, O, code, batch, heads, out = self._queries(q, out)
        n = _indices(b, lens, batch, self.device, "lens")
        if T.num_seqs != batch:
            raise JyError("attend: one query row for each sequence of the tables")
        if not 0 <= max_len <= 1 << 30:
            raise JyError("attend: max_len must be between 0 and 2^30")
        rules = self._rules(batch, heads, cap, slopes, first)
        w = (None, 0, 0, 0) if weights is None else self._weights(weights, batch, "weights")
        if not batch:
            return out
        scale = 1.0 / math.sqrt(self.hd) if scale is None else scale
        stream = b.stream(self.device.index)
        if rules is None and weights is None:
            need = b.attend_workspace(pages, batch, heads, max_len)
            ws = q.new_empty(need, dtype=b.torch.uint8) if need else None
            rc = b.attend(pages, T, n, max_len, heads, scale, Q, O, code, ws.data_ptr() if need else None, need, stream)
        else:
            need = b.attend_ruled_workspace(pages, batch, heads, max_len, first is not None, weights is not None)
            ws = q.new_empty(need, dtype=b.torch.uint8) if need else None
            rc = b.attend_ruled(pages, T, n, max_len, heads, scale, rules, Q, O, code, *w, ws.data_ptr() if need else None, need,
                                stream)
        if rc != 0:
            _failed(b)
        return out

    def attend_rows(self, layer, q, tables, starts, pos, max_len, scale=None, out=None, first=None, last=None, cap=None,
                    slopes=None):
        """Attention of runs of rows (prompts, drafted tokens): sequence s has rows starts[s] .. starts[s + 1] - 1 of
        q [rows][heads][head size] (starts: int32 [sequences + 1], ascending), row r stands at position pos[r]
        (int32) and sees positions first[r] .. last[r] - 1 of its sequence (int32; 0 and pos[r] + 1 unless given),
        all of which are in the pages by then.  A row that sees nothing gives zeros; rows in no run are left as
        they are.  `max_len` bounds last (pos + 1): what lies past it is cut.  scale, cap, slopes: as in attend."""
        b = self._b
        pages, T = self._layer(layer), self._tables(tables)
        Q, O, code, rows, heads, out = self._queries(q, out)
        s = _indices(b, starts, T.num_seqs + 1, self.device, "starts")
        p = _indices(b, pos, rows, self.device, "pos")
        if not 0 <= max_len <= 1 << 30:
            raise JyError("attend_rows: max_len must be between 0 and 2^30")
        rules = self._rules(rows, heads, cap, slopes, first, last)
        if not rows:
            return out
        need = b.attend_rows_workspace(pages, T.num_seqs, rows, heads, max_len, code)
        ws = q.new_empty(need, dtype=b.torch.uint8) if need else None
        if b.attend_rows(pages, T, s, p, rows, max_len, heads, 1.0 / math.sqrt(self.hd) if scale is None else scale, rules, Q, O,
                         code, ws.data_ptr() if need else None, need, b.stream(self.device.index)) != 0:
            _failed(b)
        return out

    def _weights(self, t, batch, name):
        """Weights of positions, for the library: address, strides and length."""
        if (t.dtype is not self._b.torch.float32 or t.dim() != 3 or t.shape[:2] != (batch, self.nkv) or t.device != self.device
                or (t.stride(2) != 1 and t.shape[2] > 1)):
            raise JyError(f"{name}: a float32 tensor [sequences][kv heads][positions] on {self.device} is needed, positions "
                          "side by side")
        return (t.data_ptr(), *t.stride()[:2], t.shape[2])

    def evict(self, layer, weights, tables, lens, keep, recent, max_len, new_tables, new_weights=None):
        """Keep `keep` positions of each sequence and kv head: the last `recent` of its lens[s] (int32) and of the
        others those with the largest weights (float32 [sequences][kv heads][positions], as `attend` adds them up; equal
        ones by position).  What stays moves, in order, to the first positions of the pages that new_tables names, none
        of them a page of `tables`.  (kept, lens, weights): the old positions int32 [sequences][kv heads][keep], -1 behind
        them, the new lengths, and the weights of what stayed, zeros behind them, in new_weights (a new tensor unless
        given; it may be `weights`).  `max_len`, an upper bound of lens: a longer one is cut to it."""
        b = self._b
        pages, T, to = self._layer(layer), self._tables(tables), self._tables(new_tables)
        batch = T.num_seqs
        n = _indices(b, lens, batch, self.device, "lens")
        w = self._weights(weights, batch, "weights")
        if not (0 <= max_len <= 1 << 30 and 1 <= keep <= 1 << 30 and 0 <= recent <= keep):
            raise JyError("evict: max_len up to 2^30, 0 <= recent <= keep, keep from 1 to 2^30")
        if new_weights is None:
            new_weights = weights.new_empty(weights.shape)
        nw = self._weights(new_weights, batch, "new_weights")
        kept = tables.new_empty((batch, self.nkv, keep))
        new_lens = lens.new_empty(batch)
        if batch and b.evict(pages, T, to, n, new_lens.data_ptr(), max_len, keep, recent, *w, *nw, kept.data_ptr(),
                             b.stream(self.device.index)) != 0:
            _failed(b)
        return kept, new_lens, new_weights


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


def rope_frequencies(dim, theta=10000.0, scaling=None, factor=1.0, trained=None, low=1.0, high=4.0, device="cuda"):
    """The angle per position of each of dim / 2 pairs, float64: theta^(-2 i / dim), for `rope`.  For contexts
    `factor` times as long as the trained one, `scaling` is
      "linear"  every frequency over `factor`;
      "base"    theta times factor^(dim / (dim - 2)): the slowest pair alone turns `factor` times slower;
      "ramp"    over `factor` where a pair turns less than `low` times in the `trained` positions, as it is
                where it turns more than `high` times, in between the mix that rises with the turns."""
    torch = _bind().torch
    if dim < 2 or dim % 2 or not theta > 0 or not factor > 0:
        raise JyError("rope_frequencies: dim is even, theta and factor are positive")
    if scaling == "base":
        theta = theta * factor ** (dim / max(1, dim - 2))
    f = theta ** (-torch.arange(dim // 2, dtype=torch.float64, device=device) * 2 / dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        if trained is None or not high > low:
            raise JyError("rope_frequencies: the ramp needs the trained length and low < high")
        mix = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * mix + f / factor * (1.0 - mix)
    elif scaling not in (None, "base"):
        raise JyError('rope_frequencies: scaling is None, "linear", "base" or "ramp"')
    return f


def rope(q, k, pos, freq, layout="half", factor=1.0, out=None):
    """Rotary positions: (q, k) with the pairs of every head of q [rows][heads][head size] and k [rows][kv heads]
    [head size] (or None) turned by pos[r] * freq[i] (int32, one a row, and float64, one a pair); float32, float16
    or bfloat16.  layout "half" pairs element i with i + pairs, "interleaved" 2 i with 2 i + 1; elements from 2 pairs
    on stay.  `factor` multiplies cosines and sines.  out: a pair of tensors, which may be q and k themselves."""
    b = _bind()
    dtype, device = q.dtype, q.device
    code = b.io.get(dtype)
    if code is None or q.dim() != 3 or not q.is_cuda:
        raise JyError("rope: q is a device tensor [rows][heads][head size] in float32, float16 or bfloat16")
    if layout not in ("half", "interleaved"):
        raise JyError('rope: layout is "half" or "interleaved"')
    rows, heads, hd = q.shape
    if k is not None and k.dim() != 3:
        raise JyError("rope: k [rows][kv heads][head size]")
    qo, ko = out if out is not None else (q.new_empty(q.shape), None if k is None else k.new_empty(k.shape))
    if (k is None) != (ko is None):
        raise JyError("rope: an output for each input")
    Q, QO = _strided(q, q.shape, dtype, device, "q"), _strided(qo, q.shape, dtype, device, "out of q")
    K = KO = None
    if k is not None:
        shape = (rows, k.shape[1], hd)
        K, KO = _strided(k, shape, dtype, device, "k"), _strided(ko, shape, dtype, device, "out of k")
    p = _indices(b, pos, rows, device, "pos")
    if freq.dtype is not b.torch.float64 or freq.dim() != 1 or freq.device != device or not freq.is_contiguous():
        raise JyError(f"rope: freq must be a contiguous float64 tensor [pairs] on {device}")
    if b.rope(Q, QO, heads, K, KO, 0 if k is None else k.shape[1], rows, hd, p, freq.data_ptr(), freq.shape[0],
              layout == "interleaved", factor, code, device.index, b.stream(device.index)) != 0:
        _failed(b)
    return qo, ko


__all__ = ["PagePool", "rope", "rope_frequencies", "sample"]
