"""The 4-bit paged cache without a GPU: the restated format, and what the Python face refuses."""
import numpy as np
import pytest
import torch

import kv4_cases


def test_format_restatement_round_trips_and_bounds_its_error():
    rng = np.random.default_rng(1)
    k = rng.standard_normal((3, 2, 32, 128)).astype(np.float32) * np.float32(3)
    v = rng.standard_normal((3, 2, 32, 128)).astype(np.float32)
    pages = kv4_cases.pack(k, v)
    assert pages.shape == (3, 2, 2, 18 * 128)
    for x, back in zip((k, v), kv4_cases.unpack(pages, 128)):
        codes, scale, base = kv4_cases.quantize(x)
        assert (back == kv4_cases.values(codes, scale, base)).all()
        # half a step, and at the top of the range what rounding the scale to 11 bits may cut off
        step = np.repeat(scale.astype(np.float64), 64, -1)
        slack = 15 * step * 2.0 ** -11 + np.repeat(np.abs(base.astype(np.float64)), 64, -1) * 2.0 ** -11
        assert (np.abs(x - back.astype(np.float64)) <= 0.5 * step + slack + 1e-6).all()


def test_format_places_a_known_value():
    """Byte positions by hand: token 5 of tile 1, head 1, channel 70 of the values."""
    v = np.zeros((1, 2, 32, 128), np.float32)
    v[0, 1, 16 + 5, 64:] = -1.0      # the group's base
    v[0, 1, 16 + 5, 70] = 2.0        # its largest value: code 15, scale 3 / 15
    pages = kv4_cases.pack(np.zeros_like(v), v)
    d = 128
    row = 9 * d + (70 // 32) * 256 + 5 * 16
    assert pages[0, 1, 1, row + (70 % 32) // 2] == 0x0F
    pair = pages[0, 1, 1, 9 * d + 8 * d + (5 * 2 + 1) * 4:][:4].view(np.float16)
    assert pair[0] == np.float16(0.2) and pair[1] == -1.0


@pytest.mark.parametrize("bad", [
    dict(head_width=96), dict(head_width=0), dict(block_size=24), dict(block_size=0), dict(dtype=torch.int8),
    dict(bytes=18 * 128 - 1), dict(tiles=2), dict(transposed=True), dict(dims=3)])
def test_pool_refuses_what_the_format_does_not_hold(bad):
    from riftco_transformer_b200 import PagedKv4Pool
    shape = [4, 2, bad.get("tiles", 1), bad.get("bytes", 18 * 128)]
    pages = torch.zeros(shape, dtype=bad.get("dtype", torch.uint8))
    if bad.get("transposed"):
        pages = torch.zeros([2, 4, 1, 18 * 128], dtype=torch.uint8).transpose(0, 1)
    if bad.get("dims") == 3:
        pages = pages[0]
    with pytest.raises((ValueError, RuntimeError)):
        PagedKv4Pool(pages, bad.get("block_size", 16), bad.get("head_width", 128))


def test_calls_refuse_host_tensors():
    from riftco_transformer_b200 import PagedKv4Pool, paged_decode_attention_kv4
    pool = PagedKv4Pool.empty(4, 2, 16, 128, device="cpu")
    assert pool.physical_blocks == 4 and pool.kv_heads == 2 and pool.bytes_per_token() == 2 * 144
    tables = torch.zeros((1, 1), dtype=torch.int32)
    q = torch.zeros((1, 4, 128))
    with pytest.raises(ValueError):
        paged_decode_attention_kv4(q, pool, tables, torch.ones(1, dtype=torch.int32), torch.empty_like(q), 16)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_no_cpu_fallback():
    from riftco_transformer_b200 import _lib
    lib = _lib.lib
    unavailable = _lib.STATUS_BACKEND_UNAVAILABLE
    assert lib.b2_rope_append_kv4(None, None, None, None, None, None, None, 1, 1, 1e4, None, None) == unavailable
    assert lib.b2_kv4_dequantize(None, None, None, 1, None, None, None, None) == unavailable
    assert lib.b2_paged_decode_attention_kv4(None, None, None, None, None, None, 1, 1, None, 0, None, None) == unavailable
    assert lib.b2_paged_chunk_attention_kv4(None, None, None, None, None, None, None, 1, 1, 1, 1, None, 0, None,
                                            None) == unavailable
    assert lib.b2_paged_decode_kv4_workspace_bytes(1, 4, 2, 128, 100000) == 0


def test_struct_layouts_match_the_header():
    import ctypes as C

    from riftco_transformer_b200._lib import Kv4CacheStruct, Kv4ScoreRulesStruct
    assert C.sizeof(Kv4CacheStruct) == 48 and Kv4CacheStruct.reserved.offset == 44
    assert C.sizeof(Kv4ScoreRulesStruct) == 16 and Kv4ScoreRulesStruct.alibi_slopes.offset == 8
