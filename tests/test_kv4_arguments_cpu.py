"""Numbers that the C ABI of the 4-bit cache cannot hold are refused by its Python face, not cut to 32 bits."""
import pytest
import torch

from riftco_transformer_b200 import kv4

TOO_LARGE = 2 ** 32 + 16   # its lower half is an ordinary length


@pytest.mark.parametrize("value", [TOO_LARGE, -1])
def test_bounds_are_not_cut_to_32_bits(value):
    pool = kv4.PagedKv4Pool.empty(4, 2, 16, 128, device="cpu")
    tables, lens, starts = (torch.zeros(s, dtype=torch.int32) for s in ((1, 4), (1,), (2,)))
    q = torch.zeros((1, 4, 128))
    with pytest.raises(ValueError, match="max_seq_len"):
        kv4.paged_decode_attention_kv4(q, pool, tables, lens, torch.empty_like(q), value)
    for max_chunk, max_len, what in ((1, value, "max_seq_len"), (value, 16, "max_chunk")):
        with pytest.raises(ValueError, match=what):
            kv4.paged_chunk_attention_kv4(q, pool, tables, lens, starts, q.bfloat16(), max_chunk, max_len)
    for at in range(5):
        with pytest.raises(ValueError):
            kv4.paged_decode_kv4_workspace_bytes(*[value if i == at else n for i, n in enumerate((1, 4, 2, 128, 16))])
    for at in range(7):
        with pytest.raises(ValueError):
            kv4.paged_chunk_kv4_workspace_bytes(*[value if i == at else n for i, n in enumerate((1, 4, 4, 2, 128, 4, 16))])


@pytest.mark.parametrize("softcap", [1e-50, 1e-45, -1e-50, 9e-7, 1.1e18, 1e300, float("inf"), float("nan"), -5.0])
def test_score_caps_are_not_rounded_to_none(softcap):
    with pytest.raises(ValueError, match="score cap"):
        kv4._rules(softcap, 0, None, 4, 0)


@pytest.mark.parametrize("window", [-1, TOO_LARGE])
def test_windows_are_not_cut_to_32_bits(window):
    with pytest.raises(ValueError, match="window"):
        kv4._rules(5.0, window, None, 4, 0)


def test_ordinary_rules_are_taken():
    assert kv4._rules(0.0, 0, None, 4, 0) is None
    rules = kv4._rules(1e-6, 2 ** 32 - 1, None, 4, 0)._obj
    assert rules.softcap == pytest.approx(1e-6) and rules.window == 2 ** 32 - 1 and rules.alibi_slopes is None
