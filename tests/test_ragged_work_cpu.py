"""What a pass of a stack with window attention has to read, write and compute, against a count of every position (no GPU)."""
import pytest

from ds41rt_b200.stack_config import LayerSpec, MLSTMSpec, StackConfig, WindowAttentionSpec
from ds41rt_b200.utils.stack_bench import work

SPECS = [WindowAttentionSpec(8, 2, 40, 24, 0.1, window=37, first=3, head_gate=True), WindowAttentionSpec(6, 3, 64, 64, 0.1),
         WindowAttentionSpec(4, 1, 32, 48, 0.2, window=70, first=90)]


def config(*mixers):
    return StackConfig("w", 100, 32, tuple(LayerSpec(m, None) for m in mixers), 1e-6, residual_gate=False, depth_average=False)


def visible(m, p):
    return {j for j in range(p + 1) if not m.window or j > p - m.window or j < m.first}


@pytest.mark.parametrize("m", SPECS)
@pytest.mark.parametrize("R,n_keys,first,decode", [(5, 200, 0, True), (5, 1, 0, True), (80, 33, 0, True), (150, 150, 0, False), (60, 160, 100, False)])
def test_window_attention(m, R, n_keys, first, decode):
    got = work(config(m), R, n_keys, first, decode)
    assert {t for t in got if t.startswith("ragged")} == {"ragged_describe", "ragged_heads", "ragged_attend"}
    assert not any("mlstm" in t or t == "head_norm_gate" for t in got)
    rows = [n_keys - 1] * R if decode else range(first, n_keys)
    pairs = sum(len(visible(m, p)) for p in rows)
    keys = pairs if decode else len(set().union(*(visible(m, p) for p in rows)))
    per = m.dim + m.vdim
    assert got["ragged_attend"] == (2 * keys * m.kv_heads * per + 2 * R * m.heads * per, 2 * pairs * m.heads * per)
    cols, size = m.heads * m.dim + m.kv_heads * per, 2 if R >= 64 else 4
    assert got["ragged_heads"] == (R * cols * (size + 2), 0)
    wide = cols + (m.heads if m.head_gate else 0)
    assert got["gemm_mix_in"] == (2 * wide * 32 + R * (2 * 32 + size * wide), 2 * R * wide * 32)


def test_one_description_to_a_shape():
    one, two = work(config(SPECS[0]), 5, 200, 0, True), work(config(SPECS[0], SPECS[1], SPECS[0]), 5, 200, 0, True)
    assert two["ragged_describe"][0] == 2 * one["ragged_describe"][0]
    assert two["ragged_attend"][0] == 2 * one["ragged_attend"][0] + work(config(SPECS[1]), 5, 200, 0, True)["ragged_attend"][0]


def test_others_are_what_they_were():
    got = work(config(MLSTMSpec(4, 32, 32, 15.0, 1e-6)), 5, 200, 0, True)
    assert "mlstm_step" in got and "head_norm_gate" in got and not any(t.startswith("ragged") for t in got)
