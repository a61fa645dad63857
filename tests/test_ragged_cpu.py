"""What passes of ragged requests refuse before anything is launched, and what their workspace is (no GPU)."""
import pytest
import torch

from ds41rt_b200.ops import ragged
from ds41rt_b200.ops.ragged import RaggedPass

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
SIZES = dict(rows=16, requests=4, heads=8, kv_heads=2, dim=64, vdim=64, page_tokens=64, device="cpu")


def make(**kw):
    return RaggedPass(**{**SIZES, **kw})


@pytest.mark.parametrize("kw", [dict(rows=0), dict(requests=0), dict(kv_heads=3), dict(dim=72), dict(vdim=8), dict(dim=272), dict(vdim=512),
                                dict(rows=1 << 19), dict(requests=5000), dict(window=-1), dict(first=-1), dict(window=1 << 31),
                                dict(page_tokens=0), dict(page_tokens=1 << 24), dict(dtype=torch.float16), dict(heads=4096, kv_heads=2),
                                dict(rows=1 << 18, heads=128, kv_heads=1)])
def test_sizes_that_no_pass_has(kw):
    with pytest.raises(ValueError):
        make(**kw)


def test_forms():
    """Which sizes take the tensor-core form."""
    assert make().tiled and make(dim=256, vdim=128).tiled and make(page_tokens=16).tiled and make(page_tokens=256).tiled
    assert make(vdim=256).tiled and not make(vdim=240).tiled
    assert not make(dtype=F32).tiled and not make(page_tokens=24).tiled and not make(page_tokens=8).tiled
    assert not make(heads=400, kv_heads=2).tiled


def test_workspace():
    p = make(rows=1000, requests=30, heads=32, kv_heads=8, dim=128, vdim=128)
    assert p.unit_tokens == 64 and p.max_blocks >= 1000 // 64 + 30 and p.max_units >= p.max_blocks * 8
    assert p.turn_rows * 4 * 128 <= 2 * 16384
    assert p.nbytes() == sum(t.numel() * 4 for t in (p.header, p.units, p.counters, p.row_pos, p.row_slot, p.row_place, p.part_o, p.part_ml,
                                                    p.status))
    assert make(rows=4).nbytes() < 1 << 21


def ints(*x):
    return torch.tensor(x, dtype=I32)


@pytest.mark.parametrize("slots,new,lengths", [
    (ints(0).long(), ints(1), ints(1)), (ints(0), ints(1, 1), ints(1)), (ints(0), ints(1), ints(1).float()),
    (ints(0).view(1, 1), ints(1), ints(1)), (ints(0, 1, 2, 3)[::2], ints(1, 1), ints(1, 1)), (ints(*range(5)), ints(*[1] * 5), ints(*[1] * 5))])
def test_descriptions_refuse(slots, new, lengths):
    with pytest.raises(ValueError):
        make().describe(slots, new, lengths, torch.zeros(4, 3, dtype=I32), 5)


@pytest.mark.parametrize("pos,slot", [(ints(*range(17)), ints(*range(17))), (ints(1), ints(1, 2)), (ints(1).long(), ints(1)),
                                      (ints(1, 2, 3)[::2], ints(1, 2))])
def test_descriptions_by_rows_refuse(pos, slot):
    with pytest.raises(ValueError):
        make().describe_rows(pos, slot, torch.zeros(4, 3, dtype=I32), 5)


@pytest.mark.parametrize("table,pages", [(torch.zeros(4, 3, dtype=torch.int64), 5), (torch.zeros(4, dtype=I32), 5), (torch.zeros(0, 3, dtype=I32), 5),
                                         (torch.zeros(3, 4, dtype=I32).T, 5), (torch.zeros(4, 3, dtype=I32), 0),
                                         (torch.zeros(4, 3, dtype=I32), 1 << 25)])
def test_page_tables_refuse(table, pages):
    with pytest.raises(ValueError):
        make()._table(table, pages, 0)


def attend_arguments(p, **kw):
    R, H, D, V = p.rows, p.heads, p.dim, p.vdim
    a = dict(q=torch.zeros(R, H, D, dtype=p.dtype), pool=torch.zeros(5 * 64, p.columns, dtype=p.dtype), page_table=torch.zeros(4, 3, dtype=I32),
             described=p, scale=0.1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(15, 8, 64, dtype=BF16)), dict(q=torch.zeros(16, 8, 64)), dict(q=torch.zeros(16, 8, 128, dtype=BF16)[..., ::2]),
    dict(q=torch.zeros(16, 8, 68, dtype=BF16)[..., :64]), dict(pool=torch.zeros(5 * 64, 256)), dict(pool=torch.zeros(5 * 64, 128, dtype=BF16)),
    dict(pool=torch.zeros(4 * 64, 256, dtype=BF16)), dict(pool=torch.zeros(5 * 64, 512, dtype=BF16)[:, ::2]), dict(scale=0.0),
    dict(scale=float("nan")), dict(page_table=torch.zeros(4, 4, dtype=I32)), dict(page_table=torch.zeros(4, 3)),
    dict(out=torch.zeros(16, 8, 64)), dict(out=torch.zeros(16, 8, 32, dtype=BF16)), dict(out=torch.zeros(16, 8, 72, dtype=BF16)[..., :64]),
    dict(out=torch.zeros(16, 8 * 64 + 4, dtype=BF16)[:, :512].unflatten(1, (8, 64))), dict(sink=torch.zeros(7)), dict(sink=torch.zeros(8).double()),
    dict(gate=torch.zeros(16, 7)), dict(gate=torch.zeros(16, 16)[:, ::2]), dict(gate=torch.zeros(16, 8, dtype=BF16)),
    dict(gate=torch.zeros(8).expand(16, 8))])
def test_attention_refuses(kw):
    p = make()
    p.table_shape, p.n_pages = (4, 3), 5
    with pytest.raises(ValueError):
        ragged.attend(**attend_arguments(p, **kw))


def test_attention_wants_a_description():
    with pytest.raises(ValueError, match="described"):
        ragged.attend(**attend_arguments(make()))


def heads_arguments(**kw):
    a = dict(q=torch.zeros(6, 4, 32), k=torch.zeros(6, 2, 32), v=torch.zeros(6, 2, 16), row_pos=ints(*range(6)), row_place=ints(*range(6)),
             pool=torch.zeros(8, 96))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(6, 128)), dict(q=torch.zeros(6, 4, 32).half()), dict(k=torch.zeros(5, 2, 32)), dict(k=torch.zeros(6, 2, 16)),
    dict(v=torch.zeros(6, 3, 16)), dict(q=torch.zeros(6, 4, 64)[..., ::2]), dict(q=torch.zeros(6, 8, 32)[:, ::2]), dict(row_pos=ints(1, 2)),
    dict(row_place=ints(*range(6)).long()), dict(pool=torch.zeros(8, 95)), dict(pool=torch.zeros(8, 96).half()), dict(pool=torch.zeros(0, 96)),
    dict(pool=torch.zeros(8, 192)[:, ::2]), dict(q_norm=torch.zeros(16)), dict(q_norm=torch.zeros(32).double()), dict(k_norm=torch.zeros(4, 32)),
    dict(freq=torch.zeros(17)), dict(freq=torch.zeros(8).double()), dict(freq=torch.zeros(16)[::2]), dict(width=33), dict(width=-1), dict(eps=-1.0),
    dict(eps=float("nan")), dict(out=torch.zeros(6, 4, 16)), dict(out=torch.zeros(6, 4, 32).bfloat16()), dict(out=torch.zeros(1, 4, 32).expand(6, 4, 32))])
def test_heads_refuse(kw):
    with pytest.raises(ValueError):
        ragged.heads_to_cache(**heads_arguments(**kw))


@pytest.mark.parametrize("kw", [dict(window=-1), dict(first=-2), dict(kv_heads=3), dict(dim=300), dict(rot_dim=7), dict(rot_dim=48)])
def test_window_layers_that_cannot_be(kw):
    from ds41rt_b200.stack_config import ConfigError, LayerSpec, StackConfig, WindowAttentionSpec
    sizes = dict(heads=8, kv_heads=2, dim=32, vdim=32, scale=0.1, window=5, first=1)
    StackConfig("w", 10, 32, (LayerSpec(WindowAttentionSpec(**sizes), None),), 1e-6).validate()
    with pytest.raises(ConfigError):
        StackConfig("w", 10, 32, (LayerSpec(WindowAttentionSpec(**{**sizes, **kw}), None),), 1e-6).validate()


@pytest.mark.parametrize("name", ["HeadsArgs", "AttendArgs"])
def test_arguments_as_bytes(name):
    """The packed form is the structure, byte for byte but for what lies between two fields and behind the last."""
    import ctypes as C
    from ds41rt_b200.ops import ragged, stack
    form = getattr(ragged, name)
    values, n = [], [0]

    def fill(a):
        for field, t in a._fields_:
            n[0] += 1
            if t is stack.ProjArgs:
                setattr(a, field, fill(t()))
            else:
                values.append(n[0] * 0.5 if t is C.c_float else n[0])
                setattr(a, field, values[-1])
        return a

    want = bytes(fill(form()))
    got = ragged.packed(form).pack(*values)
    assert len(got) <= len(want) and got == want[:len(got)] and len(want) - len(got) < 8
