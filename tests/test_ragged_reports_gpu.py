"""What descriptions report stays until somebody asks, whatever passes come in between."""
import pytest
import torch

from test_ragged_engine_gpu import Model, close, config, engine
from test_ragged_gpu import I32, Batch, ragged

pytestmark = pytest.mark.gpu


def error():
    from ds41rt_b200.ops.lib import KernelError
    return KernelError


def test_a_bad_description_and_a_good_one():
    b = Batch([(3, 10), (2, 60), (4, 0)])
    b.describe()
    b.p.check_status()
    kept = b.d_slots.clone()
    b.d_slots[1:] = 7                           # two slots that there are not
    b.describe()
    b.d_slots.copy_(kept)
    b.describe()
    b.d_new[0] = -1
    b.describe()
    b.d_new[0] = 3
    b.describe()
    with pytest.raises(error(), match="3 requests of the description cannot be, the first of them number 1"):
        b.p.check_status()
    b.p.check_status()
    b.describe()
    b.p.check_status()
    b.check(b.attend())


def test_replays():
    b = Batch([(3, 10), (2, 60), (4, 0)])
    b.describe()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.describe()
    kept = b.d_slots.clone()
    for n in range(6):
        b.d_slots[2] = 9 if n in (1, 2) else kept[2]
        graph.replay()
    with pytest.raises(error(), match="2 requests of the description cannot be, the first of them number 2"):
        b.p.check_status()
    graph.replay()
    b.p.check_status()


@pytest.fixture(scope="module")
def model():
    return Model(config())


def test_passes_of_an_engine(model):
    e = engine(model, "f32")
    e.cache.ensure(0, 100)
    e.cache.ensure(1, 100)
    for bad in ((100000, 0), (3, 9)):
        e.set_rows([1, 2], [0, bad[0]], [1, bad[1]])
        e.forward_rows(2, head=False)
        for n in range(3):
            e.set_rows([5, 6], [0, 1], [0, 0])
            e.forward_rows(2, head=False)
        with pytest.raises(error(), match="1 requests"):
            e.check_status()
        e.check_status()
    assert close(e.logits_at([1])[0], model.logits([5, 6])[-1], "f32")


def test_an_engine_asks_once(model, monkeypatch):
    """However many shapes of attention it has: one copy to the host, and one wait."""
    e = engine(model, "f32")
    assert len(e.ragged) > 1
    asked = []
    real = torch.Tensor.tolist
    monkeypatch.setattr(torch.Tensor, "tolist", lambda t: asked.append(t) or real(t))
    e.check_status()
    assert len(asked) == 1
    e.status[:4] = torch.tensor([1, 600, 2, 3], dtype=I32)
    with pytest.raises(error(), match="timed out at site 600, block 2, detail 3"):
        e.check_status()
    assert all(p.status.data_ptr() == e.status.data_ptr() == p.args.status for p in e.ragged.values())


def test_kernel_classes_have_their_work(model):
    """Every class of launches of a pass is one that utils/stack_bench.py counts the work of, and the other way round."""
    from ds41rt_b200.utils.stack_bench import work
    e = engine(model, "bf16")
    e.cache.ensure(0, 100)
    for n, decode in ((70, False), (1, True)):
        e.set_rows(list(range(n)), range(n), [0] * n)
        e.timeline = []
        e.forward_rows(n, head=True)
        tags = {tag for tag, _, _ in e.timeline}
        e.timeline = None
        assert tags == set(work(model.cfg, n, n, 0, decode))
