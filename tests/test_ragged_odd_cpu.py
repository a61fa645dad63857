"""What the heads' call and the other calls of ragged passes refuse at their limits (no GPU)."""
import pytest
import torch

from ds41rt_b200.ops import ragged

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.mark.parametrize("H,G,D", [(64, 3, 768), (49, 1, 1024), (396, 1, 128), (4001, 224, 12)])
def test_rows_of_too_many_head_values(H, G, D):
    at = torch.zeros(1, dtype=I32)
    with pytest.raises(ValueError, match="50688"):
        ragged.heads_to_cache(torch.zeros(1, H, D), torch.zeros(1, G, D), torch.zeros(1, G, 1), at, at, torch.zeros(1, G * (D + 1)))


def test_cache_rows_of_too_many_values():
    """A row of 2^31 values: numbers of columns are 32-bit."""
    at, G, V = torch.zeros(1, dtype=I32), 1024, (1 << 21) - 1
    with pytest.raises(ValueError, match="values of a row"):
        ragged.heads_to_cache(torch.zeros(1, 1, 1), torch.zeros(1, G, 1), torch.empty(1, G, V, device="meta"), at, at,
                              torch.empty(1, G * (1 + V), device="meta"))


def test_reports_in_words():
    assert ragged.told([0, 0, 0, 0]) == "" and ragged.told([0, 5, 0, 0]) == ""
    assert ragged.told([2, 5, 0, 0]) == "2 requests of the description cannot be, the first of them number 5"
    assert ragged.told([0, 0, 3, 2 ** 31 - 1 - 70]) == "3 new tokens are on pages that are not leased, the lowest row of them 70"
    assert ragged.told([1, 2, 1, 2 ** 31 - 1]) == "1 requests of the description cannot be, the first of them number 2; " \
        "1 new tokens are on pages that are not leased, the lowest row of them 0"


def test_reports_go_where_they_are_sent():
    p = ragged.RaggedPass(rows=16, requests=4, heads=8, kv_heads=2, dim=64, vdim=64, page_tokens=64, device="cpu")
    assert p.args.report == p.report.data_ptr() == p.header.data_ptr() + 16 and p.args.status == p.status.data_ptr()
    from ds41rt_b200.ops.lib import KernelError
    p.report[0], p.report[1] = 1, 3
    with pytest.raises(KernelError, match="1 requests .* number 3"):
        p.check_status()
    p.check_status()
    there = torch.zeros(8, dtype=I32)
    p.tell(there[:4], there[4:])
    there[4] = 1
    with pytest.raises(KernelError, match="number 0"):
        p.check_status()
    assert not there.any()


@pytest.mark.parametrize("name", ["row_pos", "row_slot", "row_place"])
@pytest.mark.parametrize("first", [0, 1, 5])
def test_descriptions_made_from_themselves(name, first, monkeypatch):
    """From the beginning of what they write or from within it, of rows and of requests."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)             # where CPU tensors are
    p = ragged.RaggedPass(rows=16, requests=4, heads=8, kv_heads=2, dim=64, vdim=64, page_tokens=64, device="cpu")
    own, other, table = getattr(p, name)[first:first + 3], torch.zeros(3, dtype=I32), torch.zeros(4, 3, dtype=I32)
    for pair in ((own, other), (other, own)):
        with pytest.raises(ValueError, match="copies"):
            p.describe_rows(*pair, table, 5)
    for three in ((own, other, other), (other, own, other), (other, other, own)):
        with pytest.raises(ValueError, match="copies"):
            p.describe(*three, table, 5)
    p._apart(3, own.clone().data_ptr(), other.data_ptr(), p.header.data_ptr())


def test_attention_in_place_of_queries_that_are_read_twice():
    p = ragged.RaggedPass(rows=4, requests=4, heads=4, kv_heads=2, dim=256, vdim=256, page_tokens=64, device="cpu")
    p.table_shape, p.n_pages = (4, 3), 5
    q = torch.zeros(4, 4, 256, dtype=BF16)
    with pytest.raises(ValueError, match="out cannot be q"):
        ragged.attend(q, torch.zeros(5 * 64, 1024, dtype=BF16), torch.zeros(4, 3, dtype=I32), p, scale=0.1, out=q)


@pytest.mark.parametrize("dtype,rows,fits", [(F32, 4, True), (F32, 2, False), (F32, 1, False), (BF16, 8, True), (BF16, 4, False)])
def test_attention_takes_rows_at_16_bytes(dtype, rows, fits, monkeypatch):
    """Queries, heads of queries, and results whose rows are so many values more than their own apart."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)              # not where CPU tensors are
    p = ragged.RaggedPass(rows=4, requests=4, heads=4, kv_heads=2, dim=64, vdim=64, page_tokens=64, device="cpu", dtype=dtype)
    p.table_shape, p.n_pages = (4, 3), 5
    whole, pool, table = torch.zeros(4, 4, 64, dtype=dtype), torch.zeros(5 * 64, 256, dtype=dtype), torch.zeros(4, 3, dtype=I32)
    apart = torch.zeros(4, 256 + rows, dtype=dtype)[:, :256].unflatten(1, (4, 64))
    heads = torch.zeros(4, 4, 64 + rows, dtype=dtype)[..., :64]
    for q, out in ((apart, whole), (heads, whole), (whole, apart)):
        with pytest.raises(ValueError) as error:              # the device is looked at last
            ragged.attend(q, pool, table, p, scale=0.1, out=out)
        assert ("16 bytes" in str(error.value)) != fits


def test_tensor_memory_before_the_next_kernel_may_begin():
    """A CTA that lets the next kernel's begin beside it has its tensor memory by then: else either could wait for the other."""
    from pathlib import Path
    text = (Path(ragged.__file__).parents[2] / "csrc/kernels/ragged_attend.cu").read_text()
    body = text[text.index("ragged_tiled_kernel(const __grid_constant__"):text.index("inline int tiled_smem")]
    assert body.count("pdl_launch_dependents()") == 1 and body.index("tmem_alloc(") < body.index("pdl_launch_dependents()") < body.index("pdl_wait()")


@pytest.mark.parametrize("kv_heads,vdim,fits", [(818, 64, True), (819, 64, False), (409, 256, True), (410, 256, False)])
def test_as_many_units_as_a_pass_has(kv_heads, vdim, fits):
    """Fewer than 2^22 = 4194304, the host says so and not the first call: 5120 blocks to a head (two parts of it) and 1184 more."""
    sizes = dict(rows=1 << 18, requests=4096, heads=kv_heads, kv_heads=kv_heads, dim=64, vdim=vdim, page_tokens=64, device="meta")
    if fits:
        assert ragged.RaggedPass(**sizes).max_units < 1 << 22
    else:
        with pytest.raises(ValueError, match="more than a pass divides"):
            ragged.RaggedPass(**sizes)


@pytest.mark.parametrize("kw,fits", [
    (dict(), True), (dict(scale=0.0), False), (dict(scale=-0.1), False), (dict(scale=float("nan")), False), (dict(scale=float("inf")), False),
    (dict(rot_dim=8), False), (dict(window=1 << 31), False), (dict(first=1 << 31), False), (dict(heads=2048, kv_heads=1), False),
    (dict(heads=1024, kv_heads=1), True), (dict(heads=196, kv_heads=2, dim=250), True), (dict(heads=198, kv_heads=2, dim=250), False)])
def test_window_layers_that_an_engine_could_not_run(kw, fits):
    """The configuration says so, not the engine's first pass."""
    from ds41rt_b200 import stack_config
    assert stack_config.MOST_HEAD_VALUES == ragged.MOST_HEAD_VALUES
    spec = stack_config.WindowAttentionSpec(**{**dict(heads=8, kv_heads=2, dim=32, vdim=32, scale=0.1), **kw})
    cfg = stack_config.StackConfig("w", 10, 32, (stack_config.LayerSpec(spec, None),), 1e-6)
    if fits:
        cfg.validate()
    else:
        with pytest.raises(stack_config.ConfigError):
            cfg.validate()
