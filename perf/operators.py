"""Performance cases of the batched decode operators: a paged key/value cache written and read
back, attention of one new token per sequence over it, and sampling.

A case is a plain dict.  Its "kind" says which operator runs:

  "attend"  PagePool.attend: one query row for each of `batch` sequences whose lengths lie in
            [`shortest`, `longest`], over pages of `page` positions held as `pool`.
  "append"  PagePool.write of `rows` new positions spread over `batch` sequences, then
            PagePool.read of the same positions (what the cache holds of them, as values).
  "read"    PagePool.read of `rows` positions of `batch` sequences.
  "sample"  sample: one token for each of `batch` rows of `vocab` logits, with the filters
            that `filters` names.

"io" is the type of queries, new keys and values, outputs and logits; "pool" the cache's type
(int8 with one fp32 scale per position and head, or 16 bits).  `own` chooses between the
operators' plain form and the package's kernels.
"""
import math
import random

import torch

own = False

IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
POOL = {"i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}

# (query heads, key/value heads, head size) of the package's model shapes, then generic ones:
# no sharing, one shared head, and head sizes that are neither 64 nor 128
HEADS = {"tiny-f32": (8, 2, 64), "qwen2.5-0.5b": (14, 2, 64), "llama3-8b": (32, 8, 128), "qwen2.5-7b": (28, 4, 128)}
MORE_HEADS = [(16, 16, 128), (10, 10, 64), (24, 1, 64), (10, 2, 112), (6, 3, 96), (8, 1, 256), (9, 3, 80)]


def listed():
    def attend(name, shape, batch, shortest, longest, page, pool, io):
        nh, nkv, hd = HEADS[shape]
        return dict(name=name, kind="attend", nh=nh, nkv=nkv, hd=hd, batch=batch, shortest=shortest, longest=longest,
                    page=page, pool=pool, io=io)

    def rows(name, kind, shape, batch, n, page, pool, io):
        _, nkv, hd = HEADS[shape]
        return dict(name=name, kind=kind, nkv=nkv, hd=hd, batch=batch, rows=n, page=page, pool=pool, io=io)

    def sample(name, batch, vocab, io, filters):
        return dict(name=name, kind="sample", batch=batch, vocab=vocab, io=io, filters=filters)

    return [
        # one short chat on the small model: latency
        attend("attend_one_short", "qwen2.5-0.5b", 1, 61, 61, 16, "i8", "f32"),
        # a served batch in the middle of its answers, lengths of every kind
        attend("attend_batch", "llama3-8b", 32, 1, 1500, 16, "i8", "bf16"),
        # one conversation over a long document
        attend("attend_long", "qwen2.5-7b", 1, 32769, 32769, 64, "i8", "f32"),
        # a full server with long contexts, the cache kept in 16 bits
        attend("attend_many_bf16", "llama3-8b", 64, 200, 8190, 32, "bf16", "bf16"),
        # the step's new position of one sequence on the small model
        rows("append_one", "append", "qwen2.5-0.5b", 1, 1, 16, "i8", "f32"),
        # the step's new positions of a large batch
        rows("append_batch", "append", "llama3-8b", 256, 256, 16, "i8", "bf16"),
        # the prompts of several new requests at once
        rows("append_prompts", "append", "llama3-8b", 7, 8191, 64, "i8", "bf16"),
        # a cached prefix read back for a prompt's attention, or to be moved
        rows("read_prefix", "read", "qwen2.5-0.5b", 3, 1999, 16, "i8", "f32"),
        rows("read_long", "read", "qwen2.5-7b", 2, 32770, 128, "i8", "bf16"),
        # one chat's next token with the usual filters
        sample("sample_one", 1, 151936, "f32", "chat"),
        # a served batch whose requests each bring their own settings
        sample("sample_batch", 64, 128256, "f32", "mixed"),
        # a large batch, nucleus sampling over every logit
        sample("sample_large", 256, 152064, "bf16", "nucleus"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "read", "sample"])
    io = rng.choice(["f32", "f16", "bf16"])
    if kind == "sample":
        vocab = _log_int(rng, 100, 152064)
        return dict(kind=kind, batch=_log_int(rng, 1, 256), vocab=vocab, io=io,
                    filters=rng.choice(["chat", "mixed", "nucleus", "minp", "none", "greedy"]))
    nh, nkv, hd = rng.choice(list(HEADS.values()) + MORE_HEADS)
    page, pool = rng.choice([16, 32, 64, 128, 256]), rng.choice(["i8", "i8", "f16", "bf16"])
    if kind == "attend":
        batch, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
        longest = min(longest, max(1, int(2.5e8 / (batch * nkv * hd))))  # positions of all heads of a whole batch
        return dict(kind=kind, nh=nh, nkv=nkv, hd=hd, batch=batch, shortest=_log_int(rng, 1, longest),
                    longest=longest, page=page, pool=pool, io=io)
    n = _log_int(rng, 1, 16384)
    return dict(kind=kind, nkv=nkv, hd=hd, batch=_log_int(rng, 1, min(n, 256)), rows=n, page=page, pool=pool, io=io)


# ---------------------------------------------------------------- inputs

def _lengths(case, rng):
    if case["kind"] == "attend":
        lo, hi = math.log(case["shortest"]), math.log(case["longest"])
        n = [max(1, int(round(math.exp(rng.uniform(lo, hi))))) for _ in range(case["batch"])]
        n[rng.randrange(len(n))] = case["longest"]
        return n, None
    # new rows: at least one for each sequence, the rest shared out; each after some earlier positions
    cuts = sorted(rng.sample(range(1, case["rows"]), case["batch"] - 1))
    new = [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]
    past = [0 if case["kind"] == "read" else rng.choice([0, rng.randrange(1, 500)]) for _ in new]
    return [a + b for a, b in zip(past, new)], past


def _pool_values(case, pages, g, dev):
    """A pool's tensors [1][pages][nkv][page][hd] (and scales): keys and values of unit size with
    channels that stand out, as trained models have them."""
    shape = (1, pages, case["nkv"], case["page"], case["hd"])
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
        x *= torch.exp(0.5 * torch.randn(case["hd"], generator=g, device=dev))
        if case["pool"] == "i8":
            q, s = _quantise(x)
            out += [q.to(torch.int8), s]
        else:
            out += [x.to(POOL[case["pool"]]), None]
        del x
    return out


def _inputs(case, seed):
    rng, dev = random.Random(int(seed)), "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    io = IO[case["io"]]
    if case["kind"] == "sample":
        B, V = case["batch"], case["vocab"]
        x = 2.0 * torch.randn((B, V), generator=g, device=dev)
        # some tokens that the context makes likely
        hot = torch.rand((B, V), generator=g, device=dev) < 60.0 / V
        x = torch.where(hot, 6.0 + 1.5 * x, x)
        settings = dict(chat=[(0.8, 50, 0.95, 0.0)], nucleus=[(1.0, 0, 0.9, 0.0)], minp=[(1.2, 0, 1.0, 0.05)],
                        none=[(1.0, 0, 1.0, 0.0)], greedy=[(0.0, 0, 1.0, 0.0)],
                        mixed=[(0.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (1.3, 0, 1.0, 0.02),
                               (1.0, 0, 1.0, 0.0), (0.6, 1000, 0.99, 0.01), (0.9, 5, 1.0, 0.0)])[case["filters"]]
        rows = [settings[b % len(settings)] for b in range(B)]
        T, k, p, m = (list(c) for c in zip(*rows))
        f = lambda v, t=torch.float32: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
        return dict(logits=x.to(io), u=torch.rand(B, generator=g, device=dev), temperature=f(T),
                    top_k=f(k, torch.int32), top_p=f(p), min_p=f(m))
    lens, past = _lengths(case, rng)
    page = case["page"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3  # pages that belong to nobody
    order = torch.randperm(total, generator=g, device=dev)[:sum(need)].to(torch.int32).cpu()
    tables = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    d = dict(tables=tables.to(dev))
    d["kp"], d["ks"], d["vp"], d["vs"] = _pool_values(case, total, g, dev)
    if case["kind"] == "attend":
        d["lens"], d["longest"] = torch.tensor(lens, dtype=torch.int32, device=dev), max(lens)
        d["q"] = torch.randn((len(lens), case["nh"], case["hd"]), generator=g, device=dev).to(io)
        return d
    seq = [b for b, (n, a) in enumerate(zip(lens, past)) for _ in range(n - a)]
    pos = [i for n, a in zip(lens, past) for i in range(a, n)]
    d["seq"] = torch.tensor(seq, dtype=torch.int32, device=dev)
    d["pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
    if case["kind"] == "append":
        # the rows of one fused projection: keys and values side by side
        kv = torch.randn((len(pos), 2, case["nkv"], case["hd"]), generator=g, device=dev)
        kv *= torch.exp(0.5 * torch.randn(case["hd"], generator=g, device=dev))
        kv = kv.to(io)
        d["k"], d["v"] = kv[:, 0], kv[:, 1]
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["kind"], d["io"] = case["kind"], IO[case["io"]]
    if own:
        import jieyu_amd as jy
        d["jy"] = jy
        if case["kind"] != "sample":
            d["pool"] = jy.PagePool(d["kp"], d["vp"], d["ks"], d["vs"])
    return d


# ---------------------------------------------------------------- the operators' plain form

def _quantise(x):
    """int8 values (as floats) and scales of the last axis, by the package's cache rule."""
    a = x.float().abs().amax(-1)
    on, top = a > 1e-8, torch.full_like(a, 127.0)  # (a tensor: division by a number is a product with its reciprocal)
    inv = torch.where(on, top / a, torch.zeros_like(a))
    s = torch.where(on, a / top, torch.zeros_like(a))
    return torch.round((x.float() * inv[..., None]).clamp(-127.0, 127.0)), s


def _slots(d, page):
    seq, pos = d["seq"].long(), d["pos"].long()
    return d["tables"][seq, pos // page].long(), pos % page


def _append_plain(d):
    page, slot = _slots(d, d["kp"].shape[3])
    for name, scale, x in (("kp", "ks", d["k"]), ("vp", "vs", d["v"])):
        if d[scale] is not None:
            q, s = _quantise(x)
            d[name][0][page, :, slot] = q.to(torch.int8)
            d[scale][0][page, :, slot] = s
        else:
            d[name][0][page, :, slot] = x.to(d[name].dtype)


def _read_plain(d):
    page, slot = _slots(d, d["kp"].shape[3])
    out = []
    for name, scale in (("kp", "ks"), ("vp", "vs")):
        x = d[name][0][page, :, slot].float()
        if d[scale] is not None:
            x = x * d[scale][0][page, :, slot][..., None]
        out.append(x.to(d["io"]))
    return out


def _attend_plain(d):
    q, n = d["q"].float(), d["lens"].long()
    B, nh, hd = q.shape
    nkv, page = d["kp"].shape[2:4]
    pos = torch.arange(d["longest"], device=q.device)
    live = pos[None] < n[:, None]
    at = d["tables"][:, pos // page].long().clamp(min=0)
    slot = (pos % page)[None].expand_as(at)
    k, v = d["kp"][0][at, :, slot].float(), d["vp"][0][at, :, slot].float()  # [B][positions][nkv][hd]
    if d["ks"] is not None:
        k, v = k * d["ks"][0][at, :, slot][..., None], v * d["vs"][0][at, :, slot][..., None]
    s = torch.matmul(q.view(B, nkv, nh // nkv, hd), k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(hd)
    s = s.masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = v.masked_fill(~live[..., None, None], 0.0).permute(0, 2, 1, 3).contiguous()
    return torch.matmul(p, v).reshape(B, nh, hd).to(d["io"])


def _sample_plain(d):
    x, T = d["logits"].double(), d["temperature"].double()[:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / torch.where(T > 0, T, torch.ones_like(T)))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices  # ties: the lowest index first
    es = e.gather(1, order)
    rank = torch.arange(x.shape[1], device=x.device)[None]
    k = d["top_k"].long()[:, None]
    keep = (rank < k) | (k <= 0)
    cum = torch.cumsum(es * keep, -1)
    p = d["top_p"].double()[:, None]
    keep &= (cum - es * keep < p * cum[:, -1:]) | (p >= 1)
    keep &= es >= d["min_p"].double()[:, None]
    keep |= rank == 0
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    cum = torch.cumsum(e * kept, -1)
    hit = cum > d["u"].double()[:, None] * cum[:, -1:]
    return torch.where(T[:, 0] > 0, hit.int().argmax(-1), order[:, 0]).int()


# ---------------------------------------------------------------- one pass

def run(state):
    d = state
    if own:
        if d["kind"] == "attend":
            return d["pool"].attend(0, d["q"], d["tables"], d["lens"], d["longest"])
        if d["kind"] == "sample":
            return d["jy"].sample(d["logits"], d["u"], d["temperature"], d["top_k"], d["top_p"], d["min_p"])
        if d["kind"] == "append":
            d["pool"].write(0, d["k"], d["v"], d["tables"], d["pos"], d["seq"])
        return d["pool"].read(0, d["tables"], d["pos"], d["seq"], dtype=d["io"])
    if d["kind"] == "attend":
        return _attend_plain(d)
    if d["kind"] == "sample":
        return _sample_plain(d)
    if d["kind"] == "append":
        _append_plain(d)
    return _read_plain(d)


def work(case):
    io = 4 if case["io"] == "f32" else 2
    if case["kind"] == "sample":
        n = case["batch"] * case["vocab"]
        return dict(bytes=n * io + 24 * case["batch"], flops=2 * n)
    per = case["nkv"] * (case["hd"] + 4 if case["pool"] == "i8" else 2 * case["hd"])  # one position of K or V
    if case["kind"] == "attend":
        # the lengths' mean: they are spread evenly over their logarithm, and one is the longest
        a, b = case["shortest"], case["longest"]
        mean = (b - a) / math.log(b / a) if b > a else a
        n = mean * (case["batch"] - 1) + b
        rows = 2 * case["batch"] * case["nh"] * case["hd"] * io
        return dict(bytes=2 * n * per + rows, flops=4 * n * case["nh"] * case["hd"])
    values = 2 * case["rows"] * case["nkv"] * case["hd"]
    if case["kind"] == "read":
        return dict(bytes=2 * case["rows"] * per + values * io, flops=values)
    return dict(bytes=4 * case["rows"] * per + 2 * values * io, flops=4 * values)


# ---------------------------------------------------------------- the definition in 64 bits

def _held(x, case):
    """What the cache holds of vectors x (float64 values of the input's type), in float64.  The
    int8 rule's two roundings to fp32 before the one to whole numbers are part of the format."""
    if case["pool"] != "i8":
        return x.to(POOL[case["pool"]]).double()
    a = x.abs().amax(-1, keepdim=True)
    inv = (127.0 / a).float().double()
    q = torch.round((x * inv).float().double()).clamp(-127, 127)
    q, s = torch.where(a > 1e-8, q, 0.0), torch.where(a > 1e-8, (a / 127.0).float().double(), 0.0)
    return q * s


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "sample":
        return None  # whole numbers
    if case["kind"] == "append":
        return [_held(d["k"].double(), case), _held(d["v"].double(), case)]
    ids, page = d["tables"].cpu(), case["page"]

    def positions(pool, scale, s, n):  # the first n positions of sequence s: [nkv][n][hd]
        x = pool[0][ids[s, :-(-n // page)].long().to(pool.device)].double()
        if scale is not None:
            x = x * scale[0][ids[s, :-(-n // page)].long().to(pool.device)].double()[..., None]
        return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n]

    if case["kind"] == "read":
        counts = torch.bincount(d["seq"].long()).tolist()
        return [torch.cat([positions(p, s, b, n).permute(1, 0, 2) for b, n in enumerate(counts)])
                for p, s in ((d["kp"], d["ks"]), (d["vp"], d["vs"]))]
    out, per = [], case["nh"] // case["nkv"]
    for b, n in enumerate(d["lens"].tolist()):
        k, v = positions(d["kp"], d["ks"], b, n), positions(d["vp"], d["vs"], b, n)
        rows = []
        for h in range(case["nh"]):
            s = (k[h // per] @ d["q"][b, h].double()) / math.sqrt(case["hd"])
            rows.append(torch.softmax(s, 0) @ v[h // per])
        out.append(torch.stack(rows))
    return torch.stack(out)
