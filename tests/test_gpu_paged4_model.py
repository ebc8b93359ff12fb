"""A model's pass over sequences whose keys and values are pages in 4 bits, alone and beside layers of another type."""
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))

import quant_models as QM  # noqa: E402
from test_gpu_batch_model import Reference, build, jy, near, spec  # noqa: E402, F401

pytestmark = pytest.mark.gpu

DEV = "cuda"
# The pass turns queries and keys in eights of pairs and leaves both in that order: in every 16 elements of a key the
# second and third four have changed places (an order of its own inverse; scores do not see it)
ORDER = np.arange(64).reshape(4, 4, 4)[:, [0, 2, 1, 3]].reshape(-1)


class Pools:
    """A pool whose layers are of the given types, as GpuModel.forward_paged takes one."""

    def __init__(self, jy, dtypes, pages, page):
        self.pools = [jy.PagePool.empty(1, pages, page, 2, 64, dtype=t, device=DEV) for t in dtypes]
        self.layers, self.device = len(dtypes), self.pools[0].device
        self._layers = [p._layers[0] for p in self.pools]

    def held(self, layer, tables, seq, pos):
        """what the layer holds of one token: (keys, values) [kv heads][hd]"""
        t = torch.from_numpy(np.ascontiguousarray(tables[seq:seq + 1])).to(DEV)
        k, v = self.pools[layer].read(0, t, torch.tensor([pos], dtype=torch.int32, device=DEV), dtype=torch.float32)
        return k[0].double().cpu().numpy()[:, ORDER], v[0].double().cpu().numpy()


class Held(Reference):
    """The decoder in float64 over the values that the pools hold after the call, each checked against its own.

    A group of 32 numbers is off by half a step, by what the seven bits of the step cut off the largest (15 steps of 2^-7
    at most, 0.12 of one), by the rounding of the low to fp16, and, like every state of the call, by 1e-3 of the largest."""

    def __init__(self, m, pools, tables):
        super().__init__(m, "f16")
        self.pools, self.tables = pools, tables

    def token(self, seq, pos, x):
        self.at, self.calls = (seq, pos), 0
        return super().token(seq, pos, x)

    def held(self, x):
        layer, which = divmod(self.calls, 2)
        self.calls += 1
        got = self.pools.held(layer, self.tables, *self.at)[which]
        if self.pools.pools[layer].k.dtype is torch.uint8:
            part = x.reshape(2, 2, 32)
            low, top = part.min(-1, keepdims=True), part.max(-1, keepdims=True)
            room = (0.62 * (top - low) / 15 * (1 + 2.0**-6) + 2.0**-11 * np.abs(low) + 2.0**-25) * np.ones_like(part)
            room = room.reshape(2, 64)
        elif self.pools.pools[layer].k.dtype is torch.int8:
            room = 0.51 / 127 * np.abs(x).max(-1, keepdims=True)
        else:
            room = 2.0**-8 * np.abs(x)
        assert (np.abs(got - x) <= room + 2e-3 * np.abs(x).max()).all()
        return got


@pytest.mark.parametrize("dtypes", [[torch.uint8] * 2, [torch.bfloat16, torch.uint8], [torch.uint8, torch.bfloat16]])
@pytest.mark.parametrize("wtype,mode", [(QM.JY_F32, 0), (QM.JY_Q8_0, 7)])
def test_prompts_and_steps(jy, dtypes, wtype, mode):  # noqa: F811
    m = build(spec(wtype))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 128)
    g.mode = mode
    tables = np.array([[3, 9, 1, 0], [2, 13, 5, 7], [8, 6, 4, 11]], np.int32)
    p = Pools(jy, dtypes, 14, 16)
    ref = Held(m, p, tables)
    rng = np.random.default_rng(1)
    at = [37, 1, 20]
    seq = [s for s in range(3) for _ in range(at[s])]
    pos = [i for s in range(3) for i in range(at[s])]
    X = rng.standard_normal((len(seq), 256)).astype(np.float32)
    got = g.forward_paged(p, X, tables, pos, seq)
    near(got, np.stack([ref.token(s, i, x) for s, i, x in zip(seq, pos, X)]))
    for step in range(3):
        X = rng.standard_normal((3, 256)).astype(np.float32)
        got = g.forward_paged(p, X, tables, at)
        near(got, np.stack([ref.token(s, i, x) for s, i, x in zip(range(3), at, X)]))
        at = [a + 1 for a in at]
    g.close()


@pytest.mark.parametrize("dtypes", [[torch.bfloat16, torch.uint8], [torch.uint8, torch.int8], [torch.uint8] * 2])
def test_a_long_sequence_over_layers_of_two_types(jy, dtypes):  # noqa: F811
    """thousands of positions, whose chunks are joined: each layer's attention has the workspace that its type needs"""
    m = build(spec(QM.JY_F32))
    d, keep = QM.desc_of(m)
    g = jy.GpuModel(d, 4200)
    n = 4100
    tables = np.arange(66, dtype=np.int32)[None]
    p = Pools(jy, dtypes, 66, 64)
    ref = Held(m, p, tables)
    gen = torch.Generator()
    gen.manual_seed(3)
    where = torch.arange(n, dtype=torch.int32, device=DEV)
    t = torch.from_numpy(tables).to(DEV)
    for layer, pool in enumerate(p.pools):
        k, v = (torch.randn((n, 2, 64), generator=gen).to(DEV) for _ in range(2))
        pool.write(0, k, v, t, where, seq=torch.zeros(n, dtype=torch.int32, device=DEV))
        hk, hv = pool.read(0, t, where, seq=torch.zeros(n, dtype=torch.int32, device=DEV), dtype=torch.float32)
        hk, hv = hk.double().cpu().numpy()[..., ORDER], hv.double().cpu().numpy()
        ref.cache[(0, layer)] = {i: (hk[i], hv[i]) for i in range(n)}
    X = np.random.default_rng(2).standard_normal((1, 256)).astype(np.float32)
    got = g.forward_paged(p, X, tables, [n])
    near(got, ref.token(0, n, X[0])[None])
    g.close()
