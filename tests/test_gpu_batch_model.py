"""A model's pass over sequences in pages, and sampled session steps: the batched operators where the
framework's own paths call them."""
import math
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))

import quant_models as QM  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda"
TOL = 1e-3  # max|gpu - reference| <= 1e-3 max|reference|, as for the package's tolerance modes


@pytest.fixture(scope="module")
def jy():
    import jieyu_amd
    if jieyu_amd.device_count() < 1:
        pytest.fail("no HIP device visible")
    return jieyu_amd


def spec(wtype, **over):
    d = dict(hidden=256, heads=8, kv=2, hd=64, inter=512, vocab=300, theta=10000.0, bias=True,
             layers=[{s: wtype for s in QM.SLOTS}] * 2, embed=wtype, lm=wtype, tied=False)
    d.update(over)
    return d


def build(sp, seed=5):
    QM.SPECS["batch"] = sp
    try:
        return QM.build_model("batch", seed)
    finally:
        del QM.SPECS["batch"]


def dense(tw, out, inn):
    """a weight [out][in] in float64"""
    t, a = tw
    a = np.asarray(a)
    if t == QM.JY_F32:
        return a.reshape(inn, out).T.astype(np.float64)
    if t == QM.JY_F16:
        return a.view(np.float16).reshape(inn, out).T.astype(np.float64)
    b = a.view(np.uint8).reshape(out, inn // 32, 34)
    d = b[..., :2].copy().view(np.float16).astype(np.float64)
    return (b[..., 2:].view(np.int8).astype(np.float64) * d).reshape(out, inn)


class Reference:
    """The decoder in float64, keys and values held as the pool holds them."""

    def __init__(self, m, pool):
        H, nh, nkv, hd, F = m["hidden"], m["heads"], m["kv"], m["hd"], m["inter"]
        self.m, self.pool = m, pool
        dims = dict(Wq=(nh * hd, H), Wk=(nkv * hd, H), Wv=(nkv * hd, H), Wo=(H, nh * hd), W1=(F, H), W2=(H, F), W3=(F, H))
        self.w = [{s: dense(L[s], *dims[s]) for s in dims} for L in m["layers"]]
        self.cache = {}

    def held(self, x):
        if self.pool == "i8":
            x = x.astype(np.float32)
            a = np.abs(x).max(-1, keepdims=True)
            with np.errstate(divide="ignore"):
                inv = np.where(a > 1e-8, np.float32(127) / a, np.float32(0))
            return (np.rint(x * inv).astype(np.float64)) * (a / np.float32(127))
        t = torch.from_numpy(x.astype(np.float32)).to(torch.float16 if self.pool == "f16" else torch.bfloat16)
        return t.double().numpy()

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean() + 1e-5) * w.astype(np.float64)

    def rope(self, x, pos):
        hd = x.shape[-1]
        f = self.m["theta"] ** (-np.arange(0, hd, 2) / hd) * pos
        a, b = x[:, 0::2], x[:, 1::2]
        y = np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = a * np.cos(f) - b * np.sin(f), a * np.sin(f) + b * np.cos(f)
        return y

    def token(self, seq, pos, x):
        m, x = self.m, x.astype(np.float64)
        nh, nkv, hd = m["heads"], m["kv"], m["hd"]
        for l, (L, W) in enumerate(zip(m["layers"], self.w)):
            h = self.norm(x, L["rms1"])
            q, k, v = (W[s] @ h + (L[b].astype(np.float64) if b in L else 0) for s, b in (("Wq", "bq"), ("Wk", "bk"), ("Wv", "bv")))
            q, k, v = self.rope(q.reshape(nh, hd), pos), self.rope(k.reshape(nkv, hd), pos), v.reshape(nkv, hd)
            c = self.cache.setdefault((seq, l), {})
            c[pos] = (self.held(k), self.held(v))
            K, V = (np.stack([c[p][i] for p in range(pos + 1)]) for i in (0, 1))
            o = np.empty((nh, hd))
            for i in range(nh):
                s = K[:, i // (nh // nkv)] @ q[i] / math.sqrt(hd)
                p = np.exp(s - s.max())
                o[i] = p / p.sum() @ V[:, i // (nh // nkv)]
            x = x + W["Wo"] @ o.reshape(-1)
            h = self.norm(x, L["rms2"])
            g = W["W1"] @ h
            x = x + W["W2"] @ (g / (1 + np.exp(-g)) * (W["W3"] @ h))
        return self.norm(x, m["final"])


def near(got, want):
    off = np.abs(got - want).max() / np.abs(want).max()
    assert off <= TOL, f"off by {off:.2e} of the largest"


@pytest.mark.parametrize("wtype,mode", [(QM.JY_F32, 0), (QM.JY_Q8_0, 0), (QM.JY_Q8_0, 7), (QM.JY_F16, 0)])
@pytest.mark.parametrize("pool", ["i8", "bf16"])
def test_prompts_and_steps_of_several_sequences(jy, wtype, mode, pool):
    """three sequences: their prompts in one call, then steps of all of them, one of them idle for
    a while; every row against the model in 64 bits"""
    m = build(spec(wtype))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 128)
    g.mode = mode
    ref = Reference(m, pool)
    p = jy.PagePool.empty(2, 14, 16, 2, 64, dtype={"i8": torch.int8, "bf16": torch.bfloat16}[pool], device=DEV)
    tables = np.array([[3, 9, 1, 0], [2, 13, 5, 7], [8, 6, 4, 11]], np.int32)
    rng = np.random.default_rng(1)
    at = [37, 1, 20]
    seq = [s for s in range(3) for _ in range(at[s])]
    pos = [i for s in range(3) for i in range(at[s])]
    X = rng.standard_normal((len(seq), 256)).astype(np.float32)
    near(g.forward_paged(p, X, tables, pos, seq), np.stack([ref.token(s, i, x) for s, i, x in zip(seq, pos, X)]))
    for step in range(6):
        live = [s for s in range(3) if not (s == 1 and step in (2, 3))]
        X = rng.standard_normal((len(live), 256)).astype(np.float32)
        now = [at[s] for s in live]
        near(g.forward_paged(p, X, tables, now, live), np.stack([ref.token(s, i, x) for s, i, x in zip(live, now, X)]))
        for s in live:
            at[s] += 1
    X = rng.standard_normal((1, 256)).astype(np.float32)  # one row, without seq: sequence 0
    near(g.forward_paged(p, X, tables, [at[0]]), ref.token(0, at[0], X[0])[None])
    g.close()


def test_the_first_layers_bytes_are_the_contiguous_caches(jy):
    """keys and values of the first layer come from the same products: the same bytes"""
    m = build(spec(QM.JY_Q8_0))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 64)
    X = np.random.default_rng(2).standard_normal((30, 256)).astype(np.float32)
    kv = g.kv(64)
    g.forward_cached(kv, X, 0)
    k, ks, v, vs = kv.read(0, 0, 30)
    p = jy.PagePool.empty(2, 4, 16, 2, 64, device=DEV)
    g.forward_paged(p, X, np.array([[2, 0]], np.int32), np.arange(30), np.zeros(30, np.int32))
    for a, s, pk, psc in ((k, ks, p.k, p.k_scale), (v, vs, p.v, p.v_scale)):
        got = torch.cat([pk[0, 2], pk[0, 0]], 1)[:, :30].permute(1, 0, 2).cpu().numpy()
        assert np.array_equal(got, a)
        assert np.array_equal(torch.cat([psc[0, 2], psc[0, 0]], 1)[:, :30].t().cpu().numpy(), s)
    kv.close()
    g.close()


def test_refusals(jy):
    m = build(spec(QM.JY_F32))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 40)
    p = jy.PagePool.empty(2, 6, 16, 2, 64, device=DEV)
    x = np.zeros((2, 256), np.float32)
    t = np.array([[0, 1, 2], [3, -1, 6]], np.int32)
    p.k.zero_(), p.v.zero_(), p.k_scale.zero_(), p.v_scale.zero_()
    for args, text in [((t, [40, 0]), "RoPE"), ((t, [-1, 0]), "RoPE"), ((t, [0, 16]), "no page"), ((t, [0, 39]), "no page"),
                       ((t[:, :1], [16, 0]), "past the page table"), ((t, [0, 0], [0, 2]), "out of range"),
                       ((t, [0, 0], [-1, 0]), "out of range"), ((t, [5, 5], [0, 0]), "same slot"),
                       ((np.array([[0], [0]], np.int32), [3, 3]), "same slot"), ((t[:1], [0, 1]), "more rows")]:
        with pytest.raises(jy.JyError, match=text):
            g.forward_paged(p, x, *args)
    with pytest.raises(jy.JyError, match="heads are not"):
        g.forward_paged(jy.PagePool.empty(2, 6, 16, 1, 64, device=DEV), x, t, [0, 0])
    with pytest.raises(jy.JyError, match="fewer layers"):
        g.forward_paged(jy.PagePool.empty(1, 6, 16, 2, 64, device=DEV), x, t, [0, 0])
    assert not p.k.any() and not p.k_scale.any()  # nothing was written
    g.close()


# ---------------------------------------------------------------- sampled sessions

def allowed(logits, u, T, k, p, mp, slack):
    """ids that the definition allows when the logits are off a little"""
    x = torch.from_numpy(logits).double()
    e = torch.exp((x - x.max()) / T)
    order = torch.sort(x, descending=True, stable=True).indices
    es = e[order][:k] if k > 0 else e[order]
    cum = torch.cumsum(es, 0)
    got = set()
    for dp in (-slack, 0, slack):
        n = max(1, int((cum - es < (p + dp) * cum[-1]).sum())) if p < 1 else len(es)
        for dm in (-slack, 0, slack):
            keep = torch.zeros(len(x), dtype=torch.bool)
            keep[order[:n]] = True
            keep &= e >= mp * (1 + dm)
            c = torch.cumsum(e * keep, 0)
            for du in (-slack, 0, slack):
                hit = torch.nonzero((c > (u + du) * c[-1]) & keep)
                if len(hit):
                    got.add(int(hit[0]))
    return got


SETTINGS = [(0.8, 20, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.3, 0, 0.7, 0.0), (1.0, 0, 1.0, 0.1), (0.5, 5, 1.0, 0.0)]


@pytest.mark.parametrize("wtype,mode", [(QM.JY_F32, 0), (QM.JY_Q8_0, 0), (QM.JY_Q8_0, 7)])
@pytest.mark.parametrize("T,k,p,mp", SETTINGS)
def test_sampled_steps(jy, wtype, mode, T, k, p, mp):
    m = build(spec(wtype))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 64)
    g.mode = mode
    prompt = QM.prompt_of(m, 6)
    u = np.random.default_rng(3).random(12).astype(np.float32)
    s = g.session(prompt, 13, temperature=T)
    assert s.step_sampled(u[:7], k, p, mp) == 7 and s.step_sampled(u[7:], k, p, mp) == 5 and s.remaining == 0
    ids = s.ids()
    s.close()
    s = g.session(prompt, 13, temperature=T)  # one at a time: the same
    for x in u:
        assert s.step_sampled([x], k, p, mp) == 1
    assert s.ids().tolist() == ids.tolist()
    s.close()
    # each token against the logits after what stood before it (from a prompt pass: off by its own rounding)
    for i, x in enumerate(u):
        _, _, logits = g.generate(ids[:7 + i], 1, want_logits=True)
        assert int(ids[7 + i]) in allowed(logits, float(x), T, k, p, mp, 2e-3), i
    g.close()


def test_sampled_steps_stop_and_refuse(jy):
    m = build(spec(QM.JY_Q8_0))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 64)
    prompt = QM.prompt_of(m, 6)
    u = np.random.default_rng(3).random(20).astype(np.float32)
    s = g.session(prompt, 21, temperature=1.0)
    assert s.step_sampled(u) == 20
    ids = s.ids()
    s.close()
    eos = int(ids[12])
    n = ids[6:].tolist().index(eos) + 1
    s = g.session(prompt, 21, temperature=1.0, eos=[eos])
    assert len(s) == 7 and (n == 1 or s.step_sampled(u) == n - 1) and s.remaining == 0
    assert s.ids().tolist() == ids[:6 + n].tolist()
    assert s.step_sampled(u) == 0
    s.close()
    s = g.session(prompt, 5, temperature=0.0)
    with pytest.raises(jy.JyError, match="greedy"):
        s.step_sampled(u)
    s.close()
    s = g.session(prompt, 5, temperature=1.0, repetition_penalty=1.2)
    with pytest.raises(jy.JyError, match="penalty"):
        s.step_sampled(u)
    s.close()
    # host-drawn and device-drawn steps may follow one another
    s = g.session(prompt, 9, temperature=1.0)
    assert s.step(2) == 2 and s.step_sampled(u[:3]) == 3 and s.step(3) == 3 and s.remaining == 0
    assert all(0 <= i < 300 for i in s.ids())
    s.close()
    g.close()


@pytest.mark.parametrize("wtype,mode", [(QM.JY_F32, 0), (QM.JY_Q8_0, 0), (QM.JY_Q8_0, 7)])
def test_a_first_pass_of_one_row_and_passes_between_a_sessions_steps(jy, wtype, mode):
    """a new model's first call is one row; a session whose workspace a longer pass replaces goes on
    with the tokens it would have drawn"""
    m = build(spec(wtype))
    d, keep = QM.desc_of(m)
    rng = np.random.default_rng(4)
    X = rng.standard_normal((40, 256)).astype(np.float32)
    u = rng.random(12).astype(np.float32)
    prompt = QM.prompt_of(m, 6)
    runs = []
    for between in (False, True):
        g = jy.GpuModel(d, 64)
        g.mode = mode
        p = jy.PagePool.empty(2, 6, 16, 2, 64, device=DEV)
        tables = np.array([[4, 2, 0], [1, 5, 3]], np.int32)
        near(g.forward_paged(p, X[:1], tables, [0]), Reference(m, "i8").token(0, 0, X[0])[None])
        s = g.session(prompt, 13, temperature=1.0)
        for i in range(0, 12, 4):
            if between:
                g.forward_paged(p, X[:13 + i], tables, np.arange(13 + i), np.ones(13 + i, np.int32))
            assert s.step_sampled(u[i:i + 4], top_p=0.9) == 4
        runs.append(s.ids().tolist())
        s.close()
        g.close()
    assert runs[0] == runs[1]


@pytest.mark.parametrize("eos", [None, [298]])
def test_sampled_steps_without_any_number(jy, eos):
    """a step whose logits are all NaN ends the session with an error, and gives no token"""
    m = build(spec(QM.JY_F32))
    np.asarray(m["lm"][1])[:] = np.nan
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 64)
    prompt = QM.prompt_of(m, 6)
    s = g.session(prompt, 9, temperature=1.0, eos=eos)
    n, ids = len(s), s.ids().tolist()
    if s.remaining:  # (the first token is the host's)
        with pytest.raises(jy.JyError, match="no number"):
            s.step_sampled(np.full(4, 0.5, np.float32), top_k=5)
    assert s.remaining == 0 and len(s) == n and s.ids().tolist() == ids
    assert s.step_sampled([0.5]) == 0
    s.close()
    g.close()


def test_batched_loop_from_pages_to_tokens(jy):
    """the operators as a server uses them: a pass of all sequences, logits, a token for each by its own
    settings, the next pass; the run is the same twice, and a sequence alone draws the same tokens"""
    m = build(spec(QM.JY_F32))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 64)
    E = dense(m["embed"], 300, 256) if m["embed"][0] != QM.JY_F32 else np.asarray(m["embed"][1]).reshape(300, 256)
    head = torch.from_numpy(np.asarray(m["lm"][1]).reshape(256, 300).astype(np.float32)).to(DEV)
    settings = [torch.tensor(v, device=DEV) for v in ([0.0, 0.9, 1.2], [0.5, 0.95, 1.0], [0.0, 0.05, 0.0])]
    top_k = torch.tensor([0, 30, 0], dtype=torch.int32, device=DEV)

    def run(which):
        p = jy.PagePool.empty(2, 12, 16, 2, 64, device=DEV)
        tables = np.arange(12, dtype=np.int32).reshape(3, 4)[which]
        ids, out = np.array([[5, 6, 7], [8, 9, 10], [11, 12, 13]])[which], []
        n = len(which)
        h = g.forward_paged(p, E[ids.reshape(-1)], tables, np.tile(np.arange(3), n), np.repeat(np.arange(n), 3))[2::3]
        for t in range(10):
            u = torch.tensor(np.random.default_rng(t).random(3).astype(np.float32)[which], device=DEV)
            T, P, mp = (s[which].contiguous() for s in settings)
            tok = jy.sample(torch.from_numpy(h).to(DEV) @ head, u, T, top_k[which].contiguous(), P, mp).cpu().numpy()
            out.append(tok)
            h = g.forward_paged(p, E[tok], tables, np.full(n, 3 + t))
        return np.stack(out, 1)

    a = run([0, 1, 2])
    assert np.array_equal(a, run([0, 1, 2]))
    assert (a >= 0).all() and (a < 300).all()
    g.close()


@pytest.mark.parametrize("wtype,mode", [(QM.JY_F32, 0), (QM.JY_Q8_0, 0), (QM.JY_Q8_0, 7)])
def test_a_sequence_of_a_batch_and_alone(jy, wtype, mode):
    """each sequence of a batched loop run by itself, fed the batch's tokens: the same states (to the
    products' rounding, which may go by the number of rows), and the batch's token is among those that
    its own state and settings allow; so no row reads another's table, settings or random number"""
    m = build(spec(wtype))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 64)
    g.mode = mode
    rng = np.random.default_rng(6)
    E = rng.standard_normal((300, 256)).astype(np.float32)
    W = (rng.standard_normal((256, 300)) / 8).astype(np.float32)
    head = torch.from_numpy(W).to(DEV)
    T, P, mp, top_k = [0.0, 0.9, 1.2], [0.5, 0.95, 1.0], [0.0, 0.05, 0.0], [0, 30, 0]
    settings = [torch.tensor(v, device=DEV) for v in (T, P, mp)]
    ks = torch.tensor(top_k, dtype=torch.int32, device=DEV)
    prompts = [[5, 6, 7, 8, 9], [10], [11, 12, 13]]
    n = [len(p) for p in prompts]
    tables = np.array([[7, 2, 5], [1, 9, 0], [8, 4, 3]], np.int32)
    p = jy.PagePool.empty(2, 10, 16, 2, 64, device=DEV)
    seq = [s for s in range(3) for _ in range(n[s])]
    h = g.forward_paged(p, E[sum(prompts, [])], tables, [i for s in range(3) for i in range(n[s])], seq)[np.cumsum(n) - 1]
    states, tokens, us = [], [], []
    for t in range(14):
        u = rng.random(3).astype(np.float32)
        tok = jy.sample(torch.from_numpy(h).to(DEV) @ head, torch.from_numpy(u).to(DEV), settings[0], ks, *settings[1:]).cpu().numpy()
        states.append(h), tokens.append(tok), us.append(u)
        h = g.forward_paged(p, E[tok], tables, [a + t for a in n])
    for s in range(3):
        p = jy.PagePool.empty(2, 3, 16, 2, 64, device=DEV)
        table = np.array([[1, 2, 0]], np.int32)
        h = g.forward_paged(p, E[prompts[s]], table, np.arange(n[s]), np.zeros(n[s], np.int32))[-1:]
        for t in range(14):
            near(h, states[t][s:s + 1])
            logits = (h[0].astype(np.float64) @ W).astype(np.float32)
            tok = int(tokens[t][s])
            if T[s] > 0:
                assert tok in allowed(logits, float(us[t][s]), T[s], top_k[s], P[s], mp[s], 2e-3), (s, t)
            else:
                assert logits[tok] >= logits.max() - 2 * TOL * np.abs(logits).max(), (s, t)
            h = g.forward_paged(p, E[[tok]], table, [n[s] + t])
    g.close()
