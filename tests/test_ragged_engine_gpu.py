"""Layer-stack models of window attention: engines against the model written out in 64 bits.

Tolerances.  The 32-bit engine: a dozen fp32 products of up to 256 terms a layer, each off by at most 256 * 2^-24 of its absolute sum, which
is up to ten times the result: three layers stay inside 2^-10 of the largest logit.  The bf16 engine rounds about eight intermediate
results a layer and its weights' products' inputs, 2^-8 each and independent: sqrt(3 * 8) 2^-8 = 0.02 of the logits' norm, of which the
check takes twice."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
V, W = 300, 192


def config():
    from ds41rt_b200.config import RopeConfig
    from ds41rt_b200.stack_config import LayerSpec, StackConfig, WindowAttentionSpec
    rope = RopeConfig(theta=10000.0)
    mixers = [WindowAttentionSpec(8, 2, 40, 24, 40 ** -0.5, window=37, first=3, rot_dim=32, rope=rope, head_gate=True),
              WindowAttentionSpec(6, 3, 64, 64, 0.125, rot_dim=64, rope=rope, sink=True),
              WindowAttentionSpec(4, 1, 32, 48, 0.2, window=70, head_norm=False)]
    cfg = StackConfig("windows", V, W, tuple(LayerSpec(m, None) for m in mixers), 1e-6, norm="rms", post_norm=False, residual_gate=False,
                      depth_average=False)
    cfg.validate()
    return cfg


class Model:
    def __init__(self, cfg, seed=3):
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s: (torch.randn(s, generator=gen) * s[-1] ** -0.5).bfloat16().float()
        self.cfg, self.layers = cfg, []
        for spec in cfg.layers:
            m = spec.mixer
            t = {"norm1": 1 + rnd(W), "mix.q": rnd(m.heads * m.dim, W) * 2, "mix.k": rnd(m.kv_heads * m.dim, W), "mix.v": rnd(m.kv_heads * m.vdim, W),
                 "mix.o": rnd(W, m.heads * m.vdim) * 2}
            if m.head_norm:
                t.update({"mix.q.norm": 1 + rnd(m.dim), "mix.k.norm": 1 + rnd(m.dim)})
            if m.head_gate:
                t["mix.g"] = rnd(m.heads, W)
            if m.sink:
                t["mix.sink"] = rnd(m.heads) * 3
            self.layers.append(t)
        self.top = {"embed": torch.randn(V, W, generator=gen).bfloat16().float(), "final.norm": 1 + rnd(W), "head": rnd(V, W)}

    def weights(self, dtype):
        from ds41rt_b200.models.stack import StackWeights
        return StackWeights(self.cfg, lambda l: self.layers[l], self.top, "cuda", dtype)

    def logits(self, tokens):
        """Of every position of one request, in 64 bits."""
        from ds41rt_b200.config import rope_inv_freq
        d = lambda x: x.double().cuda()
        rms = lambda x, w: x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        n = len(tokens)
        at = torch.arange(n, device="cuda")
        x = d(self.top["embed"])[torch.tensor(tokens, device="cuda")]
        for spec, t in zip(self.cfg.layers, self.layers):
            m, t = spec.mixer, {k: d(v) for k, v in t.items()}
            h = rms(x, t["norm1"])
            q, k, v = ((h @ t[f"mix.{n}"].T).unflatten(1, (-1, s)) for n, s in (("q", m.dim), ("k", m.dim), ("v", m.vdim)))
            if m.head_norm:
                q, k = rms(q, t["mix.q.norm"]), rms(k, t["mix.k.norm"])
            if m.rot_dim:
                half = m.rot_dim // 2
                a = at[:, None, None] * torch.tensor(rope_inv_freq(m.rope, m.rot_dim), dtype=torch.float32).double().cuda()

                def turn(y):
                    u, w = y[..., :half], y[..., half:m.rot_dim]
                    return torch.cat([u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin(), y[..., m.rot_dim:]], -1)

                q, k = turn(q), turn(k)
            g = m.heads // m.kv_heads
            z = torch.einsum("nhd,mhd->hnm", q, k.repeat_interleave(g, 1)) * m.scale
            seen = at[None] <= at[:, None]
            if m.window:
                seen &= (at[None] > at[:, None] - m.window) | (at[None] < m.first)
            z = z.masked_fill(~seen, -math.inf)
            if m.sink:
                z = torch.cat([z, t["mix.sink"][:, None, None].expand(-1, n, 1)], -1)
            o = torch.einsum("hnm,mhv->nhv", torch.softmax(z, -1)[..., :n], v.repeat_interleave(g, 1))
            if m.head_gate:
                o = o * torch.sigmoid(h @ t["mix.g"].T)[..., None]
            x = x + o.flatten(1) @ t["mix.o"].T
        return rms(x, d(self.top["final.norm"])) @ d(self.top["head"]).T


@pytest.fixture(scope="module")
def model():
    return Model(config())


def engine(model, dtype, **kw):
    from ds41rt_b200.models.stack import StackEngine
    return StackEngine(model.cfg, model.weights(dtype), **{**dict(max_rows=96, slots=4, max_ctx=512, page_tokens=32), **kw})


def tokens(n, seed):
    return torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def close(got, want, dtype):
    if dtype == "f32":
        return ((got.double() - want).abs().max() <= want.abs().max() * 2 ** -10).item()
    return ((got.double() - want).norm() <= want.norm() * 0.04).item()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_passes_of_several_requests(model, dtype):
    """Portions of three prompts and a row without a slot in one pass, then their next portions in another order."""
    e = engine(model, dtype)
    prompts = {0: tokens(150, 1), 2: tokens(61, 2), 3: tokens(90, 3)}
    for s in prompts:
        assert e.cache.ensure(s, 200)
    done = {s: 0 for s in prompts}
    for portions in ([(0, 50), (2, 1), (3, 44)], [(3, 40), (None, 2), (0, 30)], [(2, 60), (0, 35)], [(0, 35), (3, 6)]):
        rows = []
        for s, n in portions:
            if s is None:
                rows += [(5, 0, -1)] * n
            else:
                rows += [(prompts[s][i], i, s) for i in range(done[s], done[s] + n)]
                done[s] += n
        e.set_rows(*(list(x) for x in zip(*rows)))
        e.forward_rows(len(rows), head=False)
        got = e.logits_at(range(len(rows)))
        for i, (_, pos, s) in enumerate(rows):
            if s >= 0:
                assert close(got[i], model.logits(prompts[s][:pos + 1])[-1], dtype), (portions, i, pos, s)
    assert done == {s: len(p) for s, p in prompts.items()}
    e.check_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sessions(model, dtype):
    """A prompt in passes, long ones among them, then captured decode steps, by the host and by the device, of two requests that join."""
    from ds41rt_b200.runtime.session import DecodeSession
    e = engine(model, dtype, max_rows=80)
    session = DecodeSession(e)
    text = {0: tokens(190, 5), 1: tokens(33, 6)}
    for s, t in text.items():
        assert e.cache.ensure(s, 300)
        nxt = e.prefill(s, t)
        want = model.logits(t)[-1]
        assert close(e.logits[e.last_head_row], want, dtype) and (dtype == "bf16" or nxt == int(want.argmax()))
        t.append(nxt)
    for _ in range(4):
        out = session.step([t[-1] for t in text.values()], [len(t) - 1 for t in text.values()], list(text))
        logits = e.logits_rows(2)
        for i, (t, o) in enumerate(zip(text.values(), out)):
            assert close(logits[i], model.logits(t)[-1], dtype)
            t.append(o)
    session.step([t[-1] for t in text.values()], [len(t) - 1 for t in text.values()], list(text))
    first = e.chosen[:2].tolist()
    e.set_rows([t[-1] for t in text.values()], [len(t) - 1 for t in text.values()], list(text))
    session.run_device_loop(2, 3)
    torch.cuda.synchronize()
    for i, t in enumerate(text.values()):
        t.append(first[i])
    if dtype == "f32":
        for i, t in enumerate(text.values()):
            for _ in range(2):
                t.append(int(model.logits(t)[-1].argmax()))
            assert close(e.logits_rows(2)[i], model.logits(t[:-1])[-1], dtype)
    e.check_status()


def test_a_snapshot_continues(model):
    """Another slot goes on from a request's pages."""
    e = engine(model, "f32")
    t = tokens(75, 8)
    e.cache.ensure(0, 100)
    e.prefill(0, t)
    snap = e.cache.snapshot(0, 75)
    assert e.cache.restore(1, snap) and e.cache.ensure(1, 100)
    more = tokens(20, 9)
    e.set_rows(more, range(75, 95), [1] * 20)
    e.forward_rows(20, head=False)
    assert close(e.logits_at([19])[0], model.logits(t + more)[-1], "f32")


def test_rows_that_cannot_be(model):
    """A position that no page table reaches, and a slot that there is not: zeros from the attention, and told by the status."""
    from ds41rt_b200.ops.lib import KernelError
    e = engine(model, "f32")
    e.cache.ensure(0, 100)
    for pos, slot in ((100000, 0), (3, 9)):
        e.set_rows([1, 2], [0, pos], [1 - min(slot, 1), slot])
        e.forward_rows(2, head=False)
        with pytest.raises(KernelError, match="1 requests"):
            e.check_status()
    e.set_rows([5, 6], [0, 1], [0, 0])
    e.forward_rows(2, head=False)
    e.check_status()
    assert close(e.logits_at([1])[0], model.logits([5, 6])[-1], "f32")
