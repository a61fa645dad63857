"""Engines whose passes read the pages that requests share once for all of them, against the plain CPU statement: prompts in
portions, requests that continue one snapshot and decode together through captured graphs, changing company, reused slots."""
import pytest
import torch

import test_belasun_gpu as belasun
import test_stack_gpu as genesun
from test_stack_gpu import close, feed, limit

pytestmark = pytest.mark.gpu
FAMILIES = {"belasun": belasun, "genesun": genesun}


def engine(family, name, **kw):
    e = FAMILIES[family].engine(name, "bf16", shared_prefix=True, **kw)
    e.tags = set()
    launch = e._run

    def run(tag, *a, **k):
        e.tags.add(tag)
        return launch(tag, *a, **k)
    e._run = run
    return e


def reference(family, name, toks):
    return FAMILIES[family].reference(name, toks, "bf16")[:2] if family == "belasun" else genesun.reference(name, toks)[:2]


@pytest.mark.parametrize("family,name", [("belasun", "odd"), ("belasun", "plain"), ("belasun", "tiles"), ("genesun", "odd"),
                                         ("genesun", "tiles")])
def test_portions_match_the_oracle(family, name):
    e = engine(family, name)
    toks = FAMILIES[family].tokens(name, 230)
    want, spread = reference(family, name, toks)
    for sizes in ([1024], [2], [70, 2, 3, 61, 64, 5, 65, 2, 130], [90, 1]):
        close(feed(e, 0, toks, 0, sizes), want, "bf16", spread)
        e.cache.release(0)
    assert "prefix_attend" in e.tags and not e.tags & {"group_attend", "latent_attend"}


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("family,name,page", [("belasun", "tiles", 64), ("belasun", "odd", 16), ("belasun", "plain", 32),
                                              ("genesun", "tiles", 64), ("genesun", "odd", 32)])
def test_requests_that_share_a_snapshot_decode_together(family, name, page, graphs):
    """Three requests continue one prompt, a fourth has its own; rows leave, change places and come back on a reused slot."""
    from ds41rt_b200.runtime.session import DecodeSession
    f = FAMILIES[family]
    e = engine(family, name, page_tokens=page)
    ses = DecodeSession(e, use_graphs=graphs)
    common = f.tokens(name, 140, seed=5)
    ends = [f.tokens(name, 60, seed=20 + i) for i in range(5)]
    toks = [common + ends[0], common + ends[1], common + ends[2], f.tokens(name, 100, seed=6) + ends[3], common + ends[4]]
    at = [140, 140, 140, 100, 140]
    want = [reference(family, name, t) for t in toks]
    feed(e, 0, common, 0, [90, 1024])
    snap = e.cache.snapshot(0, 140)
    assert e.cache.restore(1, snap) and e.cache.restore(2, snap)
    feed(e, 3, toks[3][:100], 0, [1024])
    slot = [0, 1, 2, 3, None]
    for s in range(4):
        assert e.cache.ensure(s, 210)

    def step(who):
        ses.step([toks[i][at[i]] for i in who], [at[i] for i in who], [slot[i] for i in who])
        got = e.logits_rows(len(who)).cpu().double()
        for k, i in enumerate(who):
            close(got[k:k + 1], want[i][0][at[i]:at[i] + 1], "bf16", want[i][1][at[i]:at[i] + 1])
            at[i] += 1

    for _ in range(6):
        step([0, 1, 2, 3])
    tokens = 140 // page * page
    for p in e.prefix_plans.values():                    # rows at 146 see nothing of the prefix where their chunk begins behind it
        low = 145 // p.chunk * p.chunk // page * page if p.chunk else 0
        assert p.shared == ([([0, 1, 2], tokens)] if tokens - low >= 64 else [])
    for who in ([3, 2, 0, 1], [2, 1], [0, 3, 2], [1], [3, 1, 2, 0]):
        for _ in range(2):
            step(who)
    e.cache.release(2)                                   # request 2 ends; another one continues the snapshot on its slot
    assert e.cache.restore(2, snap) and e.cache.ensure(2, 210)
    slot[4] = 2
    for who in ([4, 0, 1], [0, 4, 3, 1]):
        for _ in range(3):
            step(who)
    # a pass of one request between two steps, then the same rows again
    e.cache.release(3)
    feed(e, 3, toks[3][:40], 0, [33, 7])
    for _ in range(2):
        step([0, 4, 1])
    e.check_status()
    e.cache.drop_snapshot(snap)
    assert "prefix_attend" in e.tags and not e.tags & {"group_attend", "latent_attend"}


def test_graphs_of_a_device_loop_follow_the_requests_as_they_grow():
    """A captured step feeds itself across several pages; the tokens are those of an engine that reads every row's pages alone."""
    from ds41rt_b200.runtime.session import DecodeSession
    got = []
    for shared in (False, True):
        e = belasun.engine("tiles", "f32", shared_prefix=shared)
        assert not e.prefix_plans                        # 32-bit passes read row by row
        e = belasun.engine("tiles", "bf16", shared_prefix=shared, page_tokens=32)
        common = belasun.tokens("tiles", 130, seed=8)
        feed(e, 0, common, 0, [1024])
        snap = e.cache.snapshot(0, 130)
        assert e.cache.restore(1, snap) and all(e.cache.ensure(s, 300) for s in (0, 1))
        e.set_rows([3, 200], [130, 130], [0, 1])
        DecodeSession(e).run_device_loop(2, 1)
        e.check_status()
        got.append(e.logits_rows(2).cpu().double())
        ses = DecodeSession(e)
        e.set_rows([3, 200], [130, 130], [0, 1])
        ses.run_device_loop(2, 120)
        torch.cuda.synchronize()
        e.check_status()
        assert e.row_pos[:2].tolist() == [250, 250] and torch.isfinite(e.logits_rows(2)).all()
    for i, first in enumerate((3, 200)):
        want, spread = (x[130] for x in belasun.reference("tiles", common + [first], "bf16")[:2])
        err = float((got[0][i] - got[1][i]).pow(2).mean().sqrt() / want.std())
        assert err < 2 * limit("bf16", float(spread))    # either is within one of the exact values


def test_the_scheduler_serves_requests_that_share_a_prompt():
    """Requests that extend one prompt continue its snapshot together: every token's logit is the largest one, within what rounding may
    move two of them (a logit is off by at most sqrt(vocabulary) times the root mean square that `limit` bounds)."""
    from ds41rt_b200.serving.engine import GenRequest, NativeBackend
    from ds41rt_b200.serving.protocol import Sampling
    e = engine("belasun", "tiles", max_rows=256, slots=4, page_tokens=32)
    seen = set()
    describe = e.describe

    def watched(*a):
        describe(*a)
        seen.update(len(p.shared[0][0]) for p in e.prefix_plans.values() if p.shared)
    e.describe = watched
    be = NativeBackend(e, eos=-1, concurrency=3, prefill_chunk=128)
    try:
        def submit(p, n):
            r = GenRequest(prompt_ids=p, max_tokens=n, sampling=Sampling(temperature=0.0))
            be.submit(r)
            return r

        def collect(r):
            toks = []
            while True:
                ev = r.events.get(timeout=60)
                assert ev.kind != "error", ev.message
                toks += ev.tokens
                if ev.kind == "finish":
                    return toks

        first = belasun.tokens("tiles", 120, seed=31)
        common = first + collect(submit(first, 8))[:7]
        prompts = [common + belasun.tokens("tiles", 5 + i, seed=40 + i) for i in range(3)]
        outs = [collect(r) for r in [submit(p, 24) for p in prompts]]
        assert be.error is None and seen & {2, 3}
        for p, o in zip(prompts, outs):
            assert len(o) == 24
            want, spread = belasun.reference("tiles", p + o, "bf16")[:2]
            for i, tok in enumerate(o):
                z, at = want[len(p) + i - 1], len(p) + i - 1
                room = 2 * len(z) ** 0.5 * limit("bf16", float(spread[at])) * float(z.std())
                assert float(z.max() - z[tok]) <= room
    finally:
        be.close()
    e.check_status()


def test_prompts_between_steps_leave_the_plan_of_the_steps():
    """A long prompt pass takes no plan; the same rows as a short pass, eager or by a captured step, do."""
    from ds41rt_b200.runtime.session import DecodeSession
    e = engine("belasun", "tiles", page_tokens=32)
    sets, plans = [0], list(e.prefix_plans.values())
    real = plans[0].set

    def counted(*a):
        sets[0] += 1
        real(*a)
    plans[0].set = counted
    ses = DecodeSession(e)
    a, b, c = (belasun.tokens("tiles", n, seed=50 + n) for n in (90, 100, 150))
    want = [belasun.reference("tiles", t, "bf16")[:2] for t in (a, b, c)]
    feed(e, 0, a[:70], 0, [1024])
    feed(e, 1, b[:80], 0, [1024])
    assert all(e.cache.ensure(s, 200) for s in range(3))
    assert sets[0] == 0
    for i in range(4):
        ses.step([a[70 + i], b[80 + i]], [70 + i, 80 + i], [0, 1])
        got = e.logits_rows(2).cpu().double()
        for r, at in enumerate((70 + i, 80 + i)):
            close(got[r:r + 1], want[r][0][at:at + 1], "bf16", want[r][1][at:at + 1])
        if i == 1:
            n = sets[0]
            close(feed(e, 2, c[:70], 0, [1024]), want[2][0][:70], "bf16", want[2][1][:70])
    assert n == sets[0] == 1
    for _ in range(2):                                   # once as a prompt's pass, then as any other over the same rows
        e.set_rows(c[:80], list(range(80)), [2] * 80)
        e.forward_rows(80, head=False)
        e.forward_rows(80, head=False)
        got = e.logits_at(list(range(80))).cpu().double()
        close(got, want[2][0][:80], "bf16", want[2][1][:80])
    assert sets[0] == 2
    e.check_status()
