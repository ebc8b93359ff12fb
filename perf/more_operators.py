"""Performance cases of the operators that a served model needs around its batched attention: rotary
positions, a key/value cache held in 4 bits, attention with capped scores, distance biases and masks for
single tokens and for prompts, and the eviction of positions that get little attention.

A case is a plain dict.  Its "kind" says which operator runs:

  "rope"    rope of `rows` rows of query and key heads at positions below `longest`, `rot` of `hd`
            elements of each head rotated, pairs as `layout` says, frequencies by `scaling`.
  "append"  PagePool.write of `rows` new positions spread over `batch` sequences into pages of `pool`,
            then PagePool.read of the same positions (what the cache holds of them, as values).
  "attend"  PagePool.attend: one query row for each of `batch` sequences whose lengths lie in
            [`shortest`, `longest`]; `cap` (0: none) bounds the scores, `bias` adds the distance's,
            `window` (0: none) leaves out what is further back, `weights` adds up what each position got.
  "rows"    PagePool.attend_rows: `rows` query rows, the newest positions of `batch` sequences of up to
            `past` earlier ones each, under `mask`.
  "evict"   PagePool.evict of `batch` sequences of [`shortest`, `longest`] positions down to `keep`, the
            last `recent` among them, then PagePool.read of what stayed.

"io" is the type of queries, new keys and values and outputs, "pool" the cache's: "i4" (two 4-bit numbers a
byte; per 32 elements their step, of seven bits, and their lowest value in fp16), "i8" (one fp32 scale
per vector), "f16", "bf16".  `own` chooses between the operators' plain form and the package's kernels.
"""
import math
import random

import torch

own = False

IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# (query heads, key/value heads, head size) of the package's model shapes, then generic ones
HEADS = {"tiny-f32": (8, 2, 64), "qwen2.5-0.5b": (14, 2, 64), "llama3-8b": (32, 8, 128), "qwen2.5-7b": (28, 4, 128)}
MORE_HEADS = [(16, 16, 128), (10, 10, 64), (24, 1, 64), (10, 2, 112), (6, 3, 96), (8, 1, 256), (9, 3, 80)]


def listed():
    def heads(shape):
        return dict(zip(("nh", "nkv", "hd"), HEADS[shape]))

    def rope(name, shape, rows, longest, layout, scaling, io):
        return dict(name=name, kind="rope", **heads(shape), rot=HEADS[shape][2], rows=rows, longest=longest, layout=layout,
                    scaling=scaling, io=io)

    def append(name, shape, batch, rows, page, io):
        return dict(name=name, kind="append", **heads(shape), batch=batch, rows=rows, page=page, pool="i4", io=io)

    def attend(name, shape, batch, shortest, longest, page, pool, io, cap=0.0, bias=False, window=0, weights=False):
        return dict(name=name, kind="attend", **heads(shape), batch=batch, shortest=shortest, longest=longest, page=page,
                    pool=pool, io=io, cap=cap, bias=bias, window=window, weights=weights)

    def rows(name, shape, batch, n, past, page, pool, io, mask="causal", cap=0.0, bias=False):
        return dict(name=name, kind="rows", **heads(shape), batch=batch, rows=n, past=past, page=page, pool=pool, io=io,
                    mask=mask, cap=cap, bias=bias)

    def evict(name, shape, batch, shortest, longest, keep, recent, page, pool, io):
        return dict(name=name, kind="evict", **heads(shape), batch=batch, shortest=shortest, longest=longest, keep=keep,
                    recent=recent, page=page, pool=pool, io=io)

    return [
        # one chat's new token on the small model: latency
        rope("rope_one", "qwen2.5-0.5b", 1, 2048, "half", "none", "f32"),
        # the prompts of several requests, positions stretched for a long context
        rope("rope_prompts", "llama3-8b", 8191, 131072, "interleaved", "ramp", "bf16"),
        # the step's new positions of a large batch, into 4 bits
        append("append4_batch", "llama3-8b", 256, 256, 16, "bf16"),
        # the prompts of several new requests at once, into 4 bits
        append("append4_prompts", "llama3-8b", 7, 8191, 64, "bf16"),
        # one short chat with distance biases over a 4-bit cache: latency
        attend("attend4_one_short", "qwen2.5-0.5b", 1, 61, 61, 16, "i4", "f32", bias=True),
        # a full server with long contexts, the cache in 4 bits
        attend("attend4_many", "llama3-8b", 64, 200, 8190, 32, "i4", "bf16"),
        # a batch of long chats whose positions' weights are added up for a later eviction, scores capped
        attend("attend_weighed", "llama3-8b", 8, 1000, 16001, 16, "i8", "bf16", cap=50.0, weights=True),
        # a few drafted tokens for each sequence of a batch, checked in one pass
        rows("rows_drafts", "llama3-8b", 16, 77, 4000, 16, "i8", "bf16"),
        # several short prompts of documents packed one after the other, biased by distance
        rows("rows_documents", "qwen2.5-7b", 3, 2999, 0, 64, "f16", "f16", mask="documents", bias=True),
        # one long prompt, scores capped
        rows("rows_prompt", "llama3-8b", 1, 8191, 0, 64, "bf16", "bf16", cap=30.0),
        # a batch that has outgrown its share of the cache
        evict("evict_batch", "llama3-8b", 32, 1100, 4099, 1024, 128, 16, "i8", "bf16"),
        # one conversation over a long document, a cache of 4 bits
        evict("evict_long", "qwen2.5-7b", 1, 32769, 32769, 4097, 512, 64, "i4", "f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "rows", "rows", "evict"])
    nh, nkv, hd = rng.choice(list(HEADS.values()) + MORE_HEADS)
    c = dict(kind=kind, nh=nh, nkv=nkv, hd=hd, io=rng.choice(["f32", "f16", "bf16"]))
    if kind == "rope":
        return dict(c, rot=rng.choice([hd, hd, hd // 2, 2 * rng.randrange(1, hd // 2)]), rows=_log_int(rng, 1, 8191),
                    longest=_log_int(rng, 16, 1 << 20), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "ramp"]))
    c["page"] = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        n = _log_int(rng, 1, 8191)
        return dict(c, batch=_log_int(rng, 1, min(n, 256)), rows=n, pool="i4")
    c["pool"] = rng.choice(["i4", "i4", "i8", "f16", "bf16"])
    if kind == "evict":
        batch, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
        longest = min(longest, max(1, int(1.2e8 / (batch * nkv * hd))))
        keep = _log_int(rng, 1, max(1, longest // 2))
        return dict(c, batch=batch, shortest=_log_int(rng, 1, longest), longest=longest, keep=keep,
                    recent=rng.randrange(0, keep + 1))
    c["cap"], c["bias"] = rng.choice([0.0, 0.0, 20.0, 50.0]), rng.choice([False, False, True])
    if kind == "attend":
        batch, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
        longest = min(longest, max(1, int(2.5e8 / (batch * nkv * hd))))  # positions of all heads of a whole batch
        weights = rng.choice([False, True])
        if c["pool"] != "i4" and not c["cap"] and not c["bias"]:
            weights = True
        return dict(c, batch=batch, shortest=_log_int(rng, 1, longest), longest=longest, weights=weights,
                    window=rng.choice([0, 0, _log_int(rng, 1, 4096)]))
    n = _log_int(rng, 1, 4096)
    batch = _log_int(rng, 1, min(n, 32))
    past = rng.choice([0, _log_int(rng, 1, max(1, min(16384 // batch, 30000000 // n)))])
    return dict(c, batch=batch, rows=n, past=past, mask=rng.choice(["causal", "causal", "prefix", "documents", "window"]))


# ---------------------------------------------------------------- inputs

def _spread(rng, case):
    lo, hi = math.log(case["shortest"]), math.log(case["longest"])
    n = [max(1, int(round(math.exp(rng.uniform(lo, hi))))) for _ in range(case["batch"])]
    n[rng.randrange(len(n))] = case["longest"]
    return n


def _shares(rng, case):
    """new rows: at least one for each sequence, the rest shared out"""
    cuts = sorted(rng.sample(range(1, case["rows"]), case["batch"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]


def _groups(hd):
    """4-bit groups of a vector as it is laid out: 32 elements each, 2, 4 or 8 of them"""
    return 2 if hd <= 64 else 4 if hd <= 128 else 8


def _seven_bits(x):
    """fp32 numbers (not negative) rounded to seven significant bits, ties to even"""
    u = x.view(torch.int32)
    return ((u + 0xffff + ((u >> 17) & 1)) & ~0x1ffff).view(torch.float32)


def _quantise4(x):
    """(numbers, scale, lowest) of the groups of 32 of the last axis, [..., groups, 32] and [..., groups]"""
    hd = x.shape[-1]
    G = _groups(hd)
    room = x.new_full((*x.shape[:-1], 32 * G), math.nan)
    room[..., :hd] = x
    room = room.view(*x.shape[:-1], G, 32)
    there = ~torch.isnan(room)
    low = torch.where(there, room, torch.full_like(room, math.inf)).amin(-1)
    high = torch.where(there, room, torch.full_like(room, -math.inf)).amax(-1)
    some = there.any(-1)
    low = torch.where(some, low, torch.zeros_like(low)).half().float()
    scale = torch.where(some, (high - low) / torch.full_like(low, 15.0), torch.zeros_like(low))
    scale = _seven_bits(scale).half().float()
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    n = torch.round((room - low[..., None]) * inv[..., None]).clamp(0.0, 15.0)
    return torch.where(there, n, torch.zeros_like(n)), scale, low


def _pack4(n, scale, low):
    """bytes [..., 16 groups] (byte r groups + g: elements 32 g + 2 r, low half, and 32 g + 2 r + 1) and
    fp16 [..., groups, 2]"""
    G = n.shape[-2]
    pairs = n.to(torch.uint8).view(*n.shape[:-1], 16, 2).transpose(-3, -2)  # [..., 16, groups, 2]
    b = (pairs[..., 0] | (pairs[..., 1] << 4)).reshape(*n.shape[:-2], 16 * G)
    return b, torch.stack([scale, low], -1).half()


def _unpack4(b, s, hd):
    G = s.shape[-2]
    n = torch.stack([b & 15, b >> 4], -1).view(*b.shape[:-1], 16, G, 2).transpose(-3, -2).reshape(*b.shape[:-1], G, 32)
    s = s.float()
    return (n.float() * s[..., :1] + s[..., 1:]).reshape(*b.shape[:-1], 32 * G)[..., :hd]


def _quantise8(x):
    a = x.abs().amax(-1)
    on, top = a > 1e-8, torch.full_like(a, 127.0)
    inv = torch.where(on, top / a, torch.zeros_like(a))
    s = torch.where(on, a / top, torch.zeros_like(a))
    return torch.round((x * inv[..., None]).clamp(-127.0, 127.0)).to(torch.int8), s


def _held(x, pool):
    """a pool's two tensors for fp32 vectors x"""
    if pool == "i4":
        return _pack4(*_quantise4(x))
    return _quantise8(x) if pool == "i8" else (x.to(IO[pool]), None)


def _values(x, s, hd):
    """fp32 values of held vectors"""
    if s is None:
        return x.float()
    return _unpack4(x, s, hd) if x.dtype is torch.uint8 else x.float() * s[..., None]


def _tables(lens, page, g, dev, spare=3):
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare  # pages that belong to nobody
    order = torch.randperm(total, generator=g, device=dev)[:sum(need)].to(torch.int32).cpu()
    t = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t.to(dev), total


def _frequencies(case, dev):
    """radians per position of each pair, in 64 bits"""
    pairs, theta = case["rot"] // 2, 500000.0
    i = torch.arange(pairs, dtype=torch.float64, device=dev)
    if case["scaling"] == "base":
        theta *= 4.0 ** (pairs / max(1, pairs - 1))
    f = theta ** (-i / pairs)
    if case["scaling"] == "linear":
        f = f / 4.0
    if case["scaling"] == "ramp":  # pairs that turn less than once in the trained range are stretched, over 4 times not
        turns = ((8192 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * turns + f / 8.0 * (1.0 - turns)
    return f


def _inputs(case, seed):
    rng, dev = random.Random(int(seed)), "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    io, nh, nkv, hd = IO[case["io"]], case["nh"], case["nkv"], case["hd"]
    randn = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    d = {}
    if case["kind"] == "rope":
        # queries and keys of one fused projection: heads side by side, the values' behind them
        qkv = randn(case["rows"], nh + 2 * nkv, hd).to(io)
        d["q"], d["k"] = qkv[:, :nh], qkv[:, nh:nh + nkv]
        d["pos"] = torch.randint(0, case["longest"], (case["rows"],), generator=g, device=dev, dtype=torch.int32)
        d["freq"] = _frequencies(case, dev)
        return d
    page = case["page"]
    if case["kind"] in ("append", "rows"):
        new = _shares(rng, case)
        past = [rng.choice([0, rng.randrange(1, 500)]) if case["kind"] == "append" else rng.randrange(0, case["past"] + 1) for _ in new]
        lens = [a + b for a, b in zip(past, new)]
        seq = [b for b, n in enumerate(new) for _ in range(n)]
        pos = [i for n, a in zip(lens, past) for i in range(a, n)]
        d["seq"], d["pos"] = ints(seq), ints(pos)
    else:
        lens = _spread(rng, case)
    d["tables"], total = _tables(lens, page, g, dev)
    channels = [torch.exp(0.5 * randn(hd)) for _ in range(2)]  # channels that stand out, as trained models have them
    for n, c in zip("kv", channels):
        d[n + "p"], d[n + "s"] = _held(randn(1, total, nkv, page, hd) * c, case["pool"])
    if case["kind"] == "append":
        kv = (randn(len(pos), 2, nkv, hd) * channels[0]).to(io)
        d["k"], d["v"] = kv[:, 0], kv[:, 1]
        return d
    d["longest"] = max(lens)
    if case["kind"] == "evict":
        d["lens"] = ints(lens)
        w = torch.exp(2.0 * randn(len(lens), nkv, d["longest"])) / 100.0
        w[:, :, :4] += 5.0  # the first positions draw much of the weight
        w = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.1, torch.zeros_like(w), w)  # what nobody looked at: ties
        d["weights"] = w
        # pages of their own for what stays
        order = torch.arange(total, total + len(lens) * -(-case["keep"] // page), device=dev, dtype=torch.int32)
        d["new_tables"] = order.view(len(lens), -1)
        for n in ("kp", "ks", "vp", "vs"):
            if d[n] is not None:
                d[n] = torch.cat([d[n], d[n].new_zeros((1, order.numel(), *d[n].shape[2:]))], 1)
        width = min(case["keep"], d["longest"])  # the rows of new positions that are read back
        d["to"] = torch.arange(width, device=dev, dtype=torch.int32).repeat(len(lens))
        d["of"] = torch.arange(len(lens), device=dev, dtype=torch.int32).repeat_interleave(width)
        return d
    if case["bias"]:
        d["slopes"] = 2.0 ** (-8.0 * (torch.arange(nh, device=dev, dtype=torch.float32) + 1) / nh)
    if case["kind"] == "attend":
        d["lens"] = ints(lens)
        d["q"] = (1.5 * randn(len(lens), nh, hd)).to(io)
        if case["window"]:
            d["first"] = (d["lens"] - case["window"]).clamp(min=0)
        if case["weights"]:
            d["weights"] = torch.rand((len(lens), nkv, d["longest"]), generator=g, device=dev)
        return d
    d["q"] = (1.5 * randn(len(pos), nh, hd)).to(io)
    d["starts"] = ints([0] + [sum(new[:i + 1]) for i in range(len(new))])
    if case["mask"] == "window":
        d["first"] = (d["pos"] - 511).clamp(min=0)
    if case["mask"] == "documents":  # each row sees its own document, from where that starts
        starts = [0]
        while starts[-1] < d["longest"]:
            starts.append(starts[-1] + rng.randrange(20, 900))
        at = torch.tensor(starts, device=dev)
        d["first"] = at[torch.searchsorted(at, d["pos"].long(), right=True) - 1].int()
    if case["mask"] == "prefix":  # the first part of each sequence is seen by all of its rows
        share = ints([max(1, int(n * rng.uniform(0.05, 0.6))) for n in lens])
        d["last"] = torch.maximum(d["pos"] + 1, share[d["seq"].long()])
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"], d["io"] = case, IO[case["io"]]
    if own:
        import jieyu_amd as jy
        d["jy"] = jy
        if case["kind"] != "rope":
            d["pool"] = jy.PagePool(d["kp"], d["vp"], d["ks"], d["vs"], head_dim=case["hd"])
    return d


# ---------------------------------------------------------------- the operators' plain form

def _rope_plain(d):
    pairs = d["freq"].numel()
    a = d["pos"].double()[:, None, None] * d["freq"]
    c, s = torch.cos(a).float(), torch.sin(a).float()
    out = []
    for x in (d["q"], d["k"]):
        y = x.float().clone()
        r = y[..., :2 * pairs]
        i, j = (r[..., :pairs], r[..., pairs:]) if d["case"]["layout"] == "half" else (r[..., 0::2], r[..., 1::2])
        u, w = i * c - j * s, i * s + j * c
        i.copy_(u)
        j.copy_(w)
        out.append(y.to(d["io"]))
    return out


def _slots(d, tables, seq, pos):
    """(page, place in the page) of positions `pos` of sequences `seq`"""
    page = d["kp"].shape[3]
    return tables[seq, pos // page].long().clamp(min=0), pos % page


def _append_plain(d):
    page, slot = _slots(d, d["tables"], d["seq"].long(), d["pos"].long())
    out = []
    for n in "kv":
        x, s = _held(d[n].float(), d["case"]["pool"])
        d[n + "p"][0][page, :, slot] = x
        d[n + "s"][0][page, :, slot] = s
        out.append(_values(d[n + "p"][0][page, :, slot], d[n + "s"][0][page, :, slot], d["case"]["hd"]).to(d["io"]))
    return out


def _all_positions(d, n):
    """fp32 keys and values [batch][kv heads][n][hd] of every sequence's first n positions"""
    batch, pos = d["tables"].shape[0], torch.arange(n, device=d["kp"].device)
    page, slot = _slots(d, d["tables"], torch.arange(batch, device=pos.device)[:, None], pos[None])
    slot = slot.expand_as(page)
    return [_values(d[c + "p"][0][page, :, slot], None if d[c + "s"] is None else d[c + "s"][0][page, :, slot],
                    d["case"]["hd"]).permute(0, 2, 1, 3) for c in "kv"]


def _attention_plain(d, q, at, first, last):
    """out and weights of q [batch][rows][nh][hd] at positions `at`, each seeing positions first .. last - 1 ([batch][rows])"""
    B, R, nh, hd = q.shape
    k, v = _all_positions(d, d["longest"])
    n, per = k.shape[2], nh // k.shape[1]
    pos = torch.arange(n, device=q.device)
    live = (pos >= first[..., None]) & (pos < last[..., None])
    seen = live.any(1)[:, None, :, None]  # positions that nobody sees hold anything
    k, v = torch.where(seen, k, torch.zeros_like(k)), torch.where(seen, v, torch.zeros_like(v))
    q = q.float().view(B, R, nh // per, per, hd).permute(0, 2, 3, 1, 4).reshape(B, nh // per, per * R, hd)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, nh, R, n) / math.sqrt(hd)
    cap = d["case"]["cap"]
    if cap:
        s = cap * torch.tanh(s / cap)
    if d["case"]["bias"]:
        s = s - d["slopes"][:, None, None] * (at[..., None] - pos).abs()[:, None]
    s = s.masked_fill(~live[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.view(B, nh // per, per * R, n), v.contiguous()).view(B, nh, R, hd).permute(0, 2, 1, 3)
    return o.to(d["io"]), p


def _attend_plain(d):
    n = d["lens"].long()[:, None]
    first = d["first"].long()[:, None] if "first" in d else torch.zeros_like(n)
    o, p = _attention_plain(d, d["q"][:, None], n - 1, first, n)
    if "weights" not in d:
        return o[:, 0]
    nkv = d["case"]["nkv"]
    d["weights"] += p.view(p.shape[0], nkv, -1, p.shape[-1]).sum(2)
    return o[:, 0], d["weights"]


def _rows_plain(d):
    starts, seq = d["starts"].long(), d["seq"].long()
    place = torch.arange(seq.numel(), device=seq.device) - starts[seq]
    shape = (starts.numel() - 1, d["case"]["rows"] if starts.numel() == 2 else int(place.max()) + 1)

    def batched(x):
        y = x.new_zeros((*shape, *x.shape[1:]))
        y[seq, place] = x
        return y

    pos = d["pos"].long()
    first = d["first"].long() if "first" in d else torch.zeros_like(pos)
    last = d["last"].long() if "last" in d else pos + 1
    o, _ = _attention_plain(d, batched(d["q"]), batched(pos), batched(first), batched(last))
    return o[seq, place]


def _evict_plain(d):
    case, w, n = d["case"], d["weights"], d["lens"].long()
    pos = torch.arange(w.shape[-1], device=w.device)
    there = pos < n[:, None]
    late = pos >= n[:, None] - case["recent"]
    rank = torch.where(late[:, None], torch.full_like(w, math.inf), w)
    rank = torch.where(there[:, None], rank, torch.full_like(w, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices  # ties: the lowest position first
    left = torch.clamp(n, max=case["keep"])
    width = min(case["keep"], w.shape[-1])
    chosen = order[..., :width]
    alive = torch.arange(width, device=w.device) < left[:, None, None]
    chosen = torch.sort(torch.where(alive, chosen, torch.full_like(chosen, 1 << 40)), dim=-1).values
    alive = alive.expand_as(chosen)
    kept = torch.where(alive, chosen, torch.full_like(chosen, -1))
    new_w = torch.zeros_like(w)
    at = chosen.masked_fill(~alive, 0)
    new_w[..., :width] = torch.where(alive, w.gather(-1, at), torch.zeros_like(at, dtype=w.dtype))
    batch, head = torch.arange(w.shape[0], device=w.device), torch.arange(case["nkv"], device=w.device)
    page, slot = _slots(d, d["tables"], batch[:, None, None], at)
    to = torch.arange(width, device=w.device)
    to_page, to_slot = _slots(d, d["new_tables"], batch[:, None, None], to[None, None])
    to_page, to_slot, h = to_page.expand_as(at)[alive], to_slot.expand_as(at)[alive], head[None, :, None].expand_as(at)
    out = []
    for c in "kv":
        x = d[c + "p"][0][page, h, slot]
        d[c + "p"][0][to_page, h[alive], to_slot] = x[alive]
        s = None
        if d[c + "s"] is not None:
            s = d[c + "s"][0][page, h, slot]
            d[c + "s"][0][to_page, h[alive], to_slot] = s[alive]
        y = _values(x, s, case["hd"])
        y = torch.where(alive[..., None], y, torch.zeros_like(y))
        out.append(y.permute(0, 2, 1, 3).reshape(-1, case["nkv"], case["hd"]).to(d["io"]))
    full = kept.new_full((*kept.shape[:2], case["keep"]), -1)
    full[..., :width] = kept
    return dict(kept=full.int(), lens=left.int(), weights=new_w, k=out[0], v=out[1])


# ---------------------------------------------------------------- one pass

def _run_own(d):
    case, jy = d["case"], d["jy"]
    if case["kind"] == "rope":
        return list(jy.rope(d["q"], d["k"], d["pos"], d["freq"], layout=case["layout"]))
    pool = d["pool"]
    if case["kind"] == "append":
        pool.write(0, d["k"], d["v"], d["tables"], d["pos"], d["seq"])
        return list(pool.read(0, d["tables"], d["pos"], d["seq"], dtype=d["io"]))
    if case["kind"] == "evict":
        kept, lens, weights = pool.evict(0, d["weights"], d["tables"], d["lens"], case["keep"], case["recent"], d["longest"],
                                         d["new_tables"])
        k, v = pool.read(0, d["new_tables"], d["to"], d["of"], dtype=d["io"])
        return dict(kept=kept, lens=lens, weights=weights, k=k, v=v)
    cap, slopes, first = case["cap"] or None, d.get("slopes"), d.get("first")
    if case["kind"] == "attend":
        span = min(case["window"], d["longest"]) if case["window"] else d["longest"]
        out = pool.attend(0, d["q"], d["tables"], d["lens"], span, first=first, cap=cap, slopes=slopes, weights=d.get("weights"))
        return (out, d["weights"]) if "weights" in d else out
    return pool.attend_rows(0, d["q"], d["tables"], d["starts"], d["pos"], d["longest"], first=first, last=d.get("last"),
                            cap=cap, slopes=slopes)


def run(state):
    if own:
        return _run_own(state)
    plain = dict(rope=_rope_plain, append=_append_plain, attend=_attend_plain, rows=_rows_plain, evict=_evict_plain)
    return plain[state["case"]["kind"]](state)


def _vector_bytes(case):
    """of one key or value vector as held"""
    hd, pool = case["hd"], case["pool"]
    return hd / 2 + 4 * ((hd + 31) // 32) if pool == "i4" else hd + 4 if pool == "i8" else 2 * hd


def work(case):
    io = 4 if case["io"] == "f32" else 2
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["kind"] == "rope":
        n = case["rows"] * (nh + nkv)
        return dict(bytes=2 * n * hd * io + 4 * case["rows"], flops=3 * n * case["rot"])
    per = nkv * _vector_bytes(case)
    if case["kind"] == "append":
        values = 2 * case["rows"] * nkv * hd
        return dict(bytes=4 * case["rows"] * per + 2 * values * io, flops=4 * values)
    if case["kind"] == "rows":
        # rows a sequence, earlier positions, and the positions that a row sees, all in the mean
        new, past = case["rows"] / case["batch"], case["past"] / 2
        seen = past + new / 2
        seen = min(seen, 512) if case["mask"] == "window" else min(seen, 230) if case["mask"] == "documents" else seen
        seen = 1.1 * seen if case["mask"] == "prefix" else seen
        return dict(bytes=2 * case["batch"] * (new + past) * per + 2 * case["rows"] * nh * hd * io,
                    flops=4 * case["rows"] * max(1, seen) * nh * hd)
    # the lengths' mean: they are spread evenly over their logarithm, and one is the longest
    a, b = case["shortest"], case["longest"]
    n = (b - a) / math.log(b / a) if b > a else a
    if case["kind"] == "evict":
        total, kept = n * (case["batch"] - 1) + b, case["batch"] * min(case["keep"], n)
        moved = kept * (2 * 3 * per + 2 * nkv * hd * io)
        return dict(bytes=4 * nkv * (total + case["batch"] * b + kept) + moved, flops=total * nkv)
    if case["window"]:
        n, b = min(n, case["window"]), min(b, case["window"])
    n = n * (case["batch"] - 1) + b
    return dict(bytes=2 * n * per + 2 * case["batch"] * nh * hd * io + (8 * n * nkv if case["weights"] else 0),
                flops=4 * n * nh * hd)


# ---------------------------------------------------------------- the definition in 64 bits

def _held64(x, pool):
    """what the cache holds of one tensor of vectors, from the format's rule: its roundings (to fp16, of fp32
    differences and quotients) are part of the definition"""
    lead, hd = x.shape[:-1], x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for i in range(0, hd, 32):
        part = x[..., i:i + 32].double()
        low = part.amin(-1, keepdim=True).half().double()
        m, e = torch.frexp(((part.amax(-1, keepdim=True) - low).float().double() / 15).float().double())
        step = torch.ldexp(torch.round(m * 128), e - 7).half().double()  # seven bits
        back = torch.where(step > 0, 1 / step, 0.0).float().double()
        n = torch.round(((part - low).float().double() * back).float().double()).clamp(0, 15)
        out[..., i:i + 32] = (n * step + low).float().double()
    return out.view(*lead, hd)


def _sequence64(d, case, c, s, n):
    """keys or values of sequence s's first n positions, [kv heads][n][hd]"""
    page, hd = case["page"], case["hd"]
    ids = d["tables"][s, :-(-n // page)].long()
    x = d[c + "p"][0][ids]
    if case["pool"] == "i4":
        t = d[c + "s"][0][ids].double()
        G = t.shape[-2]
        y = torch.zeros(*x.shape[:-1], 32 * G, dtype=torch.float64, device=x.device)
        for g in range(G):
            for r in range(16):
                byte = x[..., r * G + g]
                y[..., 32 * g + 2 * r] = (byte % 16).double() * t[..., g, 0] + t[..., g, 1]
                y[..., 32 * g + 2 * r + 1] = (byte // 16).double() * t[..., g, 0] + t[..., g, 1]
        y = y[..., :hd]
    elif case["pool"] == "i8":
        y = x.double() * d[c + "s"][0][ids].double()[..., None]
    else:
        y = x.double()
    return y.permute(1, 0, 2, 3).reshape(case["nkv"], -1, hd)[:, :n]


def _attention64(case, k, v, q, pos, first, last, slope):
    """(out, weights) of one head: q [rows][hd], k and v [n][hd]"""
    s = q.double() @ k.T / math.sqrt(case["hd"])
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    j = torch.arange(k.shape[0], device=k.device)
    if slope is not None:
        s = s - slope.double() * (pos[:, None] - j).abs()
    s[(j < first[:, None]) | (j >= last[:, None])] = -math.inf
    s = torch.softmax(s, -1).nan_to_num(0.0)
    return s @ v, s


def exact(case, seed):
    d = _inputs(case, seed)
    nh, nkv = case["nh"], case["nkv"]
    per = nh // nkv
    if case["kind"] == "rope":
        n, out = d["freq"].numel(), []
        turn = torch.polar(torch.ones(case["rows"], 1, n, dtype=torch.float64, device="cuda"), d["pos"].double()[:, None, None] * d["freq"])
        for x in (d["q"], d["k"]):
            x = x.double()
            half = case["layout"] == "half"
            at = torch.arange(n, device=x.device)
            i, j = (at, at + n) if half else (2 * at, 2 * at + 1)
            z = torch.complex(x[..., i], x[..., j]) * turn
            x[..., i], x[..., j] = z.real, z.imag
            out.append(x)
        return out
    if case["kind"] == "append":
        return [_held64(d["k"].float(), case["pool"]), _held64(d["v"].float(), case["pool"])]
    if case["kind"] == "rows":
        out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
        first = d["first"] if "first" in d else torch.zeros_like(d["pos"])
        last = d["last"] if "last" in d else d["pos"] + 1
        starts = d["starts"].tolist()
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            n = int(max(d["pos"][b - 1] + 1, last[a:b].max()))
            k, v = _sequence64(d, case, "k", s, n), _sequence64(d, case, "v", s, n)
            for h in range(nh):
                out[a:b, h], _ = _attention64(case, k[h // per], v[h // per], d["q"][a:b, h], d["pos"][a:b], first[a:b], last[a:b],
                                              d["slopes"][h] if case["bias"] else None)
        return out
    if case["kind"] == "attend":
        out, w = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda"), d["weights"].double() if case["weights"] else None
        for s, n in enumerate(d["lens"].tolist()):
            k, v = _sequence64(d, case, "k", s, n), _sequence64(d, case, "v", s, n)
            last = torch.tensor([n], device="cuda")
            first = d["first"][s:s + 1] if "first" in d else torch.zeros_like(last)
            for h in range(nh):
                o, p = _attention64(case, k[h // per], v[h // per], d["q"][s, h:h + 1], last - 1, first, last,
                                    d["slopes"][h] if case["bias"] else None)
                out[s, h] = o[0]
                if w is not None:
                    w[s, h // per, :n] += p[0]
        return out if w is None else (out, w)
    # what stays is settled by comparisons: the values are those of the positions that do
    width = min(case["keep"], d["longest"])
    out = {n: torch.zeros(case["batch"], width, nkv, case["hd"], dtype=torch.float64, device="cuda") for n in "kv"}
    new_w = torch.zeros(d["weights"].shape, dtype=torch.float64, device="cuda")
    for s, n in enumerate(d["lens"].tolist()):
        both = {c: _sequence64(d, case, c, s, n) for c in "kv"}
        for h in range(nkv):
            w = d["weights"][s, h, :n].tolist()
            old = max(0, n - case["recent"])
            best = sorted(range(old), key=lambda i: (-w[i], i))[:max(0, min(case["keep"], n) - (n - old))]
            at = torch.tensor(sorted(best) + list(range(old, n)), device="cuda")
            for c in "kv":
                out[c][s, :len(at), h] = both[c][h, at]
            new_w[s, h, :len(at)] = d["weights"][s, h, at].double()
    return dict(kept=None, lens=None, weights=new_w, **{c: out[c].view(-1, nkv, case["hd"]) for c in "kv"})
