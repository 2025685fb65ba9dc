"""The 4-bit paged K/V cache on the GPU: append, read-back and attention against the numpy restatement
(bytes exactly, attention in 64 bits).

Tolerances. FP32 contexts: each product of q (integers, off by at most 2^-22 of their head's largest) with
exact codes is summed in FP32, so a score is off by about 2^-22 * sum |q k| / sqrt(d), with sums around 40 here 1e-5; a weight is off by
as much relative to itself, and the context by at most twice that relative to the values it averages:
rel-L2 2e-5. bf16 contexts: half a step of the rounding, 2^-8 of each value, and the fp16 operands of the
tile kernel, 2^-11 on keys, queries, weights and values: a score of up to 16 then moves by up to
2 * 16 * 2^-11 / sqrt(64) = 2e-3, so rel-L2 2^-8 + 3 * 2^-11 + 2e-3 < 8e-3."""
import numpy as np
import pytest
import torch

import kv4_cases
from conftest import Guarded, rel_l2

pytestmark = pytest.mark.gpu

F32_TOL = 2e-5
BF16_TOL = 8e-3


def cuda(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def guarded_bf16(shape):
    """A bf16 tensor inside a larger one, and the check that the rest kept its pattern."""
    n = int(np.prod(shape))
    raw = torch.full((n + 8192,), 0x7FAB, dtype=torch.int16, device="cuda")

    def check():
        torch.cuda.synchronize()
        assert bool((raw[:4096] == 0x7FAB).all()) and bool((raw[4096 + n:] == 0x7FAB).all())
    return raw[4096:4096 + n].view(torch.bfloat16).view(*shape), check


def decode(case, max_len=None, seq_lens=None, bf16=False, workspace=None, **rules):
    import riftco_transformer_b200 as b2
    if rules.pop("bias", False):
        rules["alibi_slopes"] = cuda(case.slopes)
    pool = b2.PagedKv4Pool(cuda(case.pages), case.bs, case.d)
    out = Guarded(case.q.shape)
    out.tensor.fill_(float("nan"))
    ctx16, check16 = guarded_bf16(case.q.shape)
    status = status_word()
    lens = cuda(np.array(case.lens if seq_lens is None else seq_lens, np.uint32))
    b2.paged_decode_attention_kv4(cuda(case.q), pool, cuda(case.tables), lens, out.tensor,
                                  max(1, max(case.lens)) if max_len is None else max_len, status=status,
                                  context_bf16=ctx16 if bf16 else None, workspace=workspace, **rules)
    out.check()
    check16()
    if bf16:
        assert torch.equal(ctx16, out.tensor.to(torch.bfloat16))
    return out.tensor.cpu().numpy(), int(status.item())


def chunk(case, new, max_len=None, extra_rows=0, tiles=True, max_chunk=None, **rules):
    """`tiles`: rows that are nobody's make the call large enough for the tile kernel, whatever its chunks."""
    import riftco_transformer_b200 as b2
    if rules.pop("bias", False):
        rules["alibi_slopes"] = cuda(case.slopes)
    if "prefix" in rules:
        rules["prefix_lens"] = cuda(np.array(rules.pop("prefix"), np.uint32))
    pool = b2.PagedKv4Pool(cuda(case.pages), case.bs, case.d)
    starts = np.concatenate(([0], np.cumsum(new))).astype(np.uint32)
    assert starts[-1] + extra_rows == case.q.shape[0]
    rows = case.q.shape[0]
    q = case.q
    if tiles:
        q = np.concatenate((q, np.full((max(6000 // (11 * pool.kv_heads), 3 * len(new)), *q.shape[1:]), np.nan, np.float32)))
    ctx, check = guarded_bf16(q.shape)
    ctx.fill_(7.0)
    status = status_word()
    b2.paged_chunk_attention_kv4(cuda(q), pool, cuda(case.tables), cuda(np.array(case.lens, np.uint32)),
                                 cuda(starts), ctx, max(new) if max_chunk is None else max_chunk,
                                 max(case.lens) if max_len is None else max_len,
                                 status=status, **rules)
    check()
    assert not tiles or b2.last_route() == "attention_kv4_tiles"
    assert bool((ctx[rows:] == 7.0).all())
    return ctx[:rows].float().cpu().numpy(), int(status.item())


# ---- append and read-back ---------------------------------------------------------------------

def append(pages, tables, q, k, v, positions, token_seq, bs, theta=1e4, in_place=False):
    import riftco_transformer_b200 as b2
    d = q.shape[2]
    pool = b2.PagedKv4Pool(cuda(pages), bs, d)
    qd = cuda(q)
    out = qd if in_place else torch.full_like(qd, float("nan"))
    status = status_word()
    b2.rope_append_kv4(qd, cuda(k), cuda(v), cuda(positions), pool, cuda(tables), theta,
                       token_seq=None if token_seq is None else cuda(token_seq),
                       queries_out=None if in_place else out, status=status)
    return out.cpu().numpy(), pool, int(status.item())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv,bs,tokens", [(2, 2, 16, 1), (8, 2, 32, 7), (5, 5, 48, 33), (32, 8, 64, 300),
                                              (1, 1, 16, 9500)])
def test_append_stores_the_defined_bytes(d, hq, hkv, bs, tokens):
    """q's first kv_heads heads carry the same data as k, so q_out is the rotated k the cache has to
    hold: its bytes are then exact whatever the last bit of a sine."""
    rng = np.random.default_rng(d + tokens)
    seqs = min(3, tokens)
    owner = np.sort(rng.integers(0, seqs, tokens)).astype(np.uint32)
    owner[:seqs] = np.arange(seqs)
    owner.sort()
    positions = np.empty(tokens, np.uint32)
    for s in range(seqs):
        positions[owner == s] = rng.choice(5 * tokens, (owner == s).sum(), replace=False)   # any order
    positions[0] = 0
    first = np.flatnonzero(owner == owner[0])
    positions[first] = np.concatenate(([0], 1 + rng.choice(5 * tokens, first.size - 1, replace=False)))
    blocks = -(-(5 * tokens + 1) // bs)
    tables = rng.permutation(seqs * blocks + 3)[:seqs * blocks].reshape(seqs, blocks).astype(np.uint32)
    q = rng.standard_normal((tokens, hq, d)).astype(np.float32)
    k = (q[:, :hkv] if hq >= hkv else rng.standard_normal((tokens, hkv, d))).astype(np.float32).copy()
    v = rng.standard_normal((tokens, hkv, d)).astype(np.float32)
    v[0, 0, :64] = 1.5                       # a constant group: scale 0
    v[-1, -1, -1] = 400.0                    # an outlier
    pages = rng.integers(0, 256, (seqs * blocks + 3, hkv, bs // 16, 18 * d), dtype=np.uint8)
    out, pool, status = append(pages, tables, q, k, v, positions, owner, bs)
    assert status == 0
    # rotation: cosines and sines to an FP32 rounding (2^-24 each, angles below 2^12 in double), two
    # products and a sum, each rounded: 2^-22 of the pair's size is above their sum
    half = d // 2
    angle = positions[:, None].astype(np.float64) * 1e4 ** (-2.0 * np.arange(half) / d)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = q[..., :half].astype(np.float64), q[..., half:].astype(np.float64)
    want = np.concatenate((a * cos - b * sin, b * cos + a * sin), -1)
    size = np.concatenate((np.abs(a) + np.abs(b),) * 2, -1)
    assert (np.abs(out - want) <= 2.0 ** -22 * size).all()
    # bytes: exactly the restated ones at the tokens' slots, untouched everywhere else
    want_pages = pages.copy()
    for t in range(tokens):
        block, slot = tables[owner[t], positions[t] // bs], positions[t] % bs
        one = np.zeros((1, hkv, 16, d), np.float32)
        kk, vv = one.copy(), one.copy()
        kk[0, :, slot % 16], vv[0, :, slot % 16] = out[t, :hkv], v[t]
        packed = kv4_cases.pack(kk, vv)[0, :, 0]
        for at in (0, 9 * d):
            src = packed[:, at:at + 8 * d].reshape(hkv, d // 32, 16, 16)[:, :, slot % 16]
            want_pages[block, :, slot // 16, at:at + 8 * d].reshape(hkv, d // 32, 16, 16)[:, :, slot % 16] = src
            src = packed[:, at + 8 * d:at + 9 * d].reshape(hkv, 16, -1)[:, slot % 16]
            want_pages[block, :, slot // 16, at + 8 * d:at + 9 * d].reshape(hkv, 16, -1)[:, slot % 16] = src
    assert (pool.pages.cpu().numpy() == want_pages).all()
    # read-back: base + scale * code, one rounding
    import riftco_transformer_b200 as b2
    kb, vb = Guarded((tokens, hkv, d)), Guarded((tokens, hkv, d))
    b2.dequantize_kv4(pool, cuda(tables), cuda(positions), kb.tensor, vb.tensor, token_seq=cuda(owner))
    kb.check()
    vb.check()
    for got, x in ((kb.tensor, out[:, :hkv]), (vb.tensor, v)):
        assert (got.cpu().numpy() == kv4_cases.values(*kv4_cases.quantize(x))).all()


def test_append_far_positions_keep_the_phase():
    """Angles of 10^5 radians: FP32 would have lost them."""
    rng = np.random.default_rng(5)
    d, positions = 128, np.array([131071, 1 << 20], np.uint32)
    q = rng.standard_normal((2, 1, d)).astype(np.float32)
    tables = np.zeros((2, (1 << 20) // 4096 + 1), np.uint32)
    tables[1] = 1
    pages = np.zeros((2, 1, 256, 18 * d), np.uint8)
    out, _, status = append(pages, tables, q, q.copy(), q.copy(), positions, None, 4096, theta=5e5)
    assert status == 0
    angle = positions[:, None].astype(np.float64) * 5e5 ** (-2.0 * np.arange(d // 2) / d)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = q[..., :64].astype(np.float64), q[..., 64:].astype(np.float64)
    want = np.concatenate((a * cos - b * sin, b * cos + a * sin), -1)
    # the angle itself is good to 2^20 * 2^-52
    assert (np.abs(out - want) <= 2.0 ** -22 * np.concatenate((np.abs(a) + np.abs(b),) * 2, -1)).all()


def test_append_in_place_padding_and_tokens_outside_the_cache():
    from riftco_transformer_b200 import _lib
    rng = np.random.default_rng(6)
    d, hq, hkv, bs = 128, 4, 2, 16
    q = rng.standard_normal((5, hq, d)).astype(np.float32)
    k = rng.standard_normal((5, hkv, d)).astype(np.float32)
    v = rng.standard_normal((5, hkv, d)).astype(np.float32)
    tables = np.array([[0, 1], [2, 9]], np.uint32)          # block 9 is not there
    pages = np.full((3, hkv, 1, 18 * d), 0xAB, np.uint8)
    pad = 0xFFFFFFFF
    want_q, _, _ = append(pages, tables, q, k, v, np.array([3, 17, 8, 4, 3], np.uint32),
                          np.array([0, 1, 0, 0, 0], np.uint32), bs)
    cases = [(np.array([3, 17, pad, 32, 3], np.uint32), np.array([0, 1, 0, 0, 2], np.uint32))]
    for positions, owner in cases:   # stored; bad block; padding; past the table; no such sequence
        out, pool, status = append(pages, tables, q, k, v, positions, owner, bs, in_place=True)
        assert status == _lib.ATTN_STATUS_BAD_BLOCK
        assert (out[2] == q[2]).all()                        # padding: left as it was
        assert (out[[0, 1, 4]] == want_q[[0, 1, 4]]).all()   # the rest is rotated all the same
        got = pool.pages.cpu().numpy()
        changed = (got != pages).any(axis=(1, 2, 3))
        assert changed.tolist() == [True, False, False]
        import riftco_transformer_b200 as b2
        kb = torch.full((5, hkv, d), 9.0, device="cuda")
        vb = torch.full((5, hkv, d), 9.0, device="cuda")
        st = status_word()
        b2.dequantize_kv4(pool, cuda(tables), cuda(positions), kb, vb, token_seq=cuda(owner), status=st)
        assert int(st.item()) == _lib.ATTN_STATUS_BAD_BLOCK
        assert bool((kb[1:] == 9.0).all()) and bool((vb[1:] == 9.0).all()) and not bool((kb[0] == 9.0).any())


def test_append_of_many_padding_tokens_between_real_ones():
    """Runs of tokens share a CTA and its angle buffers."""
    rng = np.random.default_rng(8)
    n, d, hq, hkv, bs = 12000, 64, 2, 1, 16
    real = rng.random(n) < 0.4
    positions = np.full(n, 0xFFFFFFFF, np.uint32)
    positions[real] = np.arange(real.sum())
    blocks = -(-n // bs)
    tables = np.arange(blocks, dtype=np.uint32).reshape(1, blocks)
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    k = q[:, :1].copy()
    pages = np.zeros((blocks, hkv, 1, 18 * d), np.uint8)
    out, pool, status = append(pages, tables, q, k, k.copy(), positions, np.zeros(n, np.uint32), bs, in_place=True)
    assert status == 0 and (out[~real] == q[~real]).all()
    angle = positions[real][:, None].astype(np.float64) * 1e4 ** (-2.0 * np.arange(32) / 64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = q[real][..., :32].astype(np.float64), q[real][..., 32:].astype(np.float64)
    want = np.concatenate((a * cos - b * sin, b * cos + a * sin), -1)
    assert (np.abs(out[real] - want) <= 2.0 ** -22 * np.concatenate((np.abs(a) + np.abs(b),) * 2, -1)).all()
    rk, _ = kv4_cases.unpack(pool.pages.cpu().numpy(), d)
    got = rk.transpose(1, 0, 2, 3).reshape(-1, d)[:real.sum()]
    assert (got == kv4_cases.values(*kv4_cases.quantize(out[real][:, 0]))).all()


def test_append_of_values_the_format_cannot_hold():
    """NaN, infinities and magnitudes above 65000 store a group of NaN; attention over it says so."""
    import riftco_transformer_b200 as b2
    from riftco_transformer_b200 import _lib
    d, hkv = 128, 1
    rng = np.random.default_rng(7)
    for bad in (np.nan, np.inf, -np.inf, 65001.0, -1e30, 3e38):
        k = rng.standard_normal((1, hkv, d)).astype(np.float32)
        k[0, 0, 65] = bad                    # second group (position 0: not rotated)
        v = k.copy()
        pages = np.zeros((1, hkv, 1, 18 * d), np.uint8)
        _, pool, status = append(pages, np.zeros((1, 1), np.uint32), k, k, v, np.zeros(1, np.uint32), None, 16)
        assert status == 0
        kb, vb = torch.empty((1, hkv, d), device="cuda"), torch.empty((1, hkv, d), device="cuda")
        b2.dequantize_kv4(pool, cuda(np.zeros((1, 1), np.uint32)), cuda(np.zeros(1, np.uint32)), kb, vb)
        assert bool(kb[0, 0, 64:].isnan().all()) and bool(vb[0, 0, 64:].isnan().all()), bad
        # the other group is stored; of the key it is the rotation's partner, and infinity * sin 0 is NaN
        assert bool(vb[0, 0, :64].isfinite().all()), bad
        assert bool(kb[0, 0, :64].isfinite().all()) == bool(np.isfinite(bad)), bad
        ctx, st = torch.empty((1, 1, d), device="cuda"), status_word()
        q = torch.ones((1, 1, d), device="cuda")
        b2.paged_decode_attention_kv4(q, pool, cuda(np.zeros((1, 1), np.uint32)), cuda(np.ones(1, np.uint32)), ctx, 1,
                                      status=st)
        assert int(st.item()) & _lib.ATTN_STATUS_NAN_OR_POS_INF
    # the largest magnitudes it does hold
    k = np.full((1, hkv, d), 65000.0, np.float32)
    k[0, 0, ::2] = -65000.0
    pages = np.zeros((1, hkv, 1, 18 * d), np.uint8)
    _, pool, _ = append(pages, np.zeros((1, 1), np.uint32), k, k, k.copy(), np.zeros(1, np.uint32), None, 16)
    rk, rv = kv4_cases.unpack(pool.pages.cpu().numpy(), d)
    assert (rk[0, 0, 0] == kv4_cases.values(*kv4_cases.quantize(k[0, 0]))).all() and np.isfinite(rv[0, 0, 0]).all()


# ---- single-token attention ---------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (6, 2), (8, 2), (10, 2), (16, 2), (9, 1), (24, 2)])
def test_decode_head_layouts(d, hq, hkv):
    case = kv4_cases.Case(d + hq, [1, 16, 17, 75, 300], hq, hkv, d, 16)
    got, status = decode(case, bf16=True)
    assert status == 0
    assert rel_l2(got, case.decode()) <= F32_TOL


@pytest.mark.parametrize("bs", [16, 32, 48, 128])
@pytest.mark.parametrize("poison", [0x00, 0x7C, 0xFF])
def test_decode_block_sizes_and_what_unused_slots_hold(bs, poison):
    """0x7C7C is a large scale, 0xFFFF a NaN: slots behind the last token must not count."""
    case = kv4_cases.Case(bs, [1, 15, 31, 33, 127, 129, 1000], 8, 2, 128, bs, poison=poison)
    got, status = decode(case)
    assert status == 0
    assert rel_l2(got, case.decode()) <= F32_TOL


@pytest.mark.parametrize("rules", [dict(softcap=5.0), dict(softcap=1e-6), dict(softcap=1e18), dict(window=1), dict(window=16), dict(window=33),
                                   dict(window=100000), dict(bias=True), dict(softcap=2.0, window=200, bias=True)])
@pytest.mark.parametrize("hq", [8, 16])
def test_decode_score_rules(rules, hq):
    case = kv4_cases.Case(31, [1, 33, 700, 2100], hq, 2, 128, 16)
    got, status = decode(case, **rules)
    assert status == 0
    want = {("slopes" if k == "bias" else k): (case.slopes if k == "bias" else v) for k, v in rules.items()}
    assert rel_l2(got, case.decode(**want)) <= F32_TOL


@pytest.mark.parametrize("max_len", [5000, 40000])
def test_decode_long_contexts_are_split_and_joined(max_len):
    case = kv4_cases.Case(max_len, [max_len, 1, max_len // 2 + 3, 0], 4, 1, 128, 16)
    got, status = decode(case, bf16=True)
    assert status == 0
    assert rel_l2(got, case.decode()) <= F32_TOL
    assert (got[3] == 0).all()
    again, _ = decode(case)
    assert (again.view(np.uint32) == got.view(np.uint32)).all()   # no order of arrival in the result


@pytest.mark.parametrize("strength", [1e-4, 30.0])
def test_decode_of_flat_and_of_peaked_scores(strength):
    case = kv4_cases.Case(3, [64, 999], 8, 2, 128, 16, strength=strength)
    got, status = decode(case)
    assert status == 0
    want = case.decode()
    if strength < 1:
        assert rel_l2(got, want) <= F32_TOL
    else:   # scores in the hundreds: 2^-22 of sum |q k| / sqrt(d), now about 1500, and twice that in the context
        assert rel_l2(got, want) <= 2 * 1500 * 2.0 ** -22


def test_decode_of_query_and_value_magnitudes_beyond_fp16():
    """q is scaled to fp16's range by a power of two per head, p * scale by one per warp."""
    for factor in (1e-30, 1e-6, 1e6, 1e20):
        case = kv4_cases.Case(11, [200], 8, 2, 64, 16, strength=min(1.0, 1 / factor) if factor <= 1e4 else 1e-3)
        case.q = (case.q * np.float32(factor)).astype(np.float32) if factor < 1 else case.q
        got, status = decode(case)
        assert status == 0
        assert rel_l2(got, case.decode()) <= F32_TOL
    case = kv4_cases.Case(12, [200], 8, 2, 64, 16, strength=1e-3)
    case.q[0, ::2] *= np.float32(1e4)
    got, status = decode(case)
    assert status == 0 and rel_l2(got, case.decode()) <= F32_TOL


@pytest.mark.parametrize("hq", [4, 12])
def test_decode_of_long_sums_that_cancel(hq):
    """Values of zero mean over 30000 tokens: the context is 1/170 of what it is summed from, so that whatever the tensor
    core cuts off its partial sums instead of rounding would show. The weights' own errors, 2^-22 * sum |q k| / sqrt(d) of
    random sign, stay relative to the context: 2 * 10^-6 for sums of 10."""
    rng = np.random.default_rng(hq)
    case = kv4_cases.Case(hq, [30000], hq, 1, 128, 16)
    table = case.tables[0]
    k, _ = kv4_cases.unpack(case.pages[table], 128)
    v = rng.standard_normal(k.shape).astype(np.float32)
    case.pages[table] = kv4_cases.pack(np.nan_to_num(k), v)
    k, v = kv4_cases.unpack(case.pages[table], 128)
    case.k, case.v = ([a.transpose(1, 0, 2, 3).reshape(1, -1, 128)[:, :30000]] for a in (k, v))
    got, status = decode(case)
    assert status == 0 and rel_l2(got, case.decode()) <= 4e-6


def test_decode_values_whose_scale_varies_by_orders_of_magnitude():
    rng = np.random.default_rng(14)
    case = kv4_cases.Case(14, [640], 4, 1, 128, 16)
    k, v = kv4_cases.unpack(case.pages[case.tables[0]], 128)
    v = v * np.exp(rng.uniform(-9, 9, v.shape[:3]))[..., None].astype(np.float32)
    k = np.nan_to_num(k)
    case.pages[case.tables[0]] = kv4_cases.pack(k, np.nan_to_num(v))
    k, v = kv4_cases.unpack(case.pages[case.tables[0]], 128)
    case.k = [k.transpose(1, 0, 2, 3).reshape(1, -1, 128)[:, :640]]
    case.v = [v.transpose(1, 0, 2, 3).reshape(1, -1, 128)[:, :640]]
    got, status = decode(case)
    assert status == 0 and rel_l2(got, case.decode()) <= F32_TOL


def test_decode_reports_what_it_meets():
    from riftco_transformer_b200 import _lib
    base = kv4_cases.Case(21, [100, 40], 8, 2, 128, 16)
    want = base.decode()
    # NaN keys: the row is flagged, the other is right
    case = kv4_cases.Case(21, [100, 40], 8, 2, 128, 16)
    case.pages[case.tables[0, 2], :, 0, 8 * 128:9 * 128] = 0xFF
    got, status = decode(case)
    assert status == _lib.ATTN_STATUS_NAN_OR_POS_INF
    assert rel_l2(got[1], want[1]) <= F32_TOL
    # a query with a NaN or an infinity
    for bad in (np.nan, np.inf, -np.inf):
        case = kv4_cases.Case(21, [100, 40], 8, 2, 128, 16)
        case.q[1, 3, 5] = bad
        got, status = decode(case)
        assert status == _lib.ATTN_STATUS_NAN_OR_POS_INF
        assert rel_l2(got[0], want[0]) <= F32_TOL and rel_l2(got[1, :3], want[1, :3]) <= F32_TOL
    # a block id outside the pool is not dereferenced
    case = kv4_cases.Case(21, [100, 40], 8, 2, 128, 16)
    case.tables[0, 1] = 0xFFFFFFF0
    got, status = decode(case)
    assert status & _lib.ATTN_STATUS_BAD_BLOCK
    assert rel_l2(got[1], want[1]) <= F32_TOL
    # a length above max_seq_len is cut to it
    case = kv4_cases.Case(21, [100, 40], 8, 2, 128, 16)
    got, status = decode(case, max_len=64)
    assert status == _lib.ATTN_STATUS_BAD_BLOCK
    case.lens[0] = 64
    assert rel_l2(got, case.decode()) <= F32_TOL


def test_decode_offsets_past_32_bits():
    import riftco_transformer_b200 as b2
    case = kv4_cases.Case(23, [48], 4, 1, 128, 16)
    blocks = (1 << 32) // (18 * 128) + 1000
    pool = b2.PagedKv4Pool.empty(blocks, 1, 16, 128)
    pages = cuda(case.pages)
    tables = np.array([[blocks - 1, 5, blocks - 700]], np.uint32)
    for i in range(3):
        pool.pages[int(tables[0, i])] = pages[int(case.tables[0, i])]
    ctx, status = torch.empty(case.q.shape, device="cuda"), status_word()
    b2.paged_decode_attention_kv4(cuda(case.q), pool, cuda(tables), cuda(np.array([48], np.uint32)), ctx, 48,
                                  status=status)
    assert int(status.item()) == 0 and rel_l2(ctx.cpu().numpy(), case.decode()) <= F32_TOL
    # the append at the far end
    q = np.ones((1, 1, 128), np.float32)
    b2.rope_append_kv4(cuda(q), cuda(q), cuda(q), cuda(np.array([1], np.uint32)), pool, cuda(tables), 1e4, status=status)
    kb, vb = torch.empty((1, 1, 128), device="cuda"), torch.empty((1, 1, 128), device="cuda")
    b2.dequantize_kv4(pool, cuda(tables), cuda(np.array([1], np.uint32)), kb, vb, status=status)
    assert int(status.item()) == 0 and bool((vb == 1.0).all())


# ---- several new tokens ---------------------------------------------------------------------------

@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 8, 2), (128, 6, 3), (128, 5, 1), (128, 2, 2), (256, 4, 2)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([3, 1, 5], [40, 0, 17]), ([130, 40], [0, 300]), ([33, 1, 0, 200], [5, 77, 9, 0])])
@pytest.mark.parametrize("tiles", [False, True])
def test_chunk_is_causal_over_the_cache(d, hq, hkv, new, past, tiles):
    lens = [p + m for p, m in zip(past, new)]
    case = kv4_cases.Case(d + sum(new), lens, hq, hkv, d, 16, rows=sum(new))
    got, status = chunk(case, new, tiles=tiles)
    assert status == 0
    assert rel_l2(got, case.chunk(new)) <= BF16_TOL


@pytest.mark.parametrize("rules", [dict(softcap=4.0), dict(window=1), dict(window=50), dict(bias=True),
                                   dict(prefix=[100, 30]), dict(prefix=[1000, 0], window=40, softcap=3.0, bias=True)])
@pytest.mark.parametrize("new,past", [([5, 2], [90, 20]), ([150, 260], [33, 0])])
@pytest.mark.parametrize("d,tiles", [(128, True), (256, True), (128, False)])
def test_chunk_score_rules(rules, new, past, d, tiles):
    lens = [p + m for p, m in zip(past, new)]
    case = kv4_cases.Case(77, lens, 8, 2, d, 32, rows=sum(new))
    got, status = chunk(case, new, tiles=tiles, **rules)
    assert status == 0
    want = {("slopes" if k == "bias" else k): (case.slopes if k == "bias" else v) for k, v in rules.items()}
    assert rel_l2(got, case.chunk(new, **want)) <= BF16_TOL


@pytest.mark.parametrize("d,hq,hkv,new,past,route", [
    (128, 8, 8, [2] * 4, 4000, "attention_kv4"), (128, 8, 8, [3] * 4, 4000, "attention_kv4_tiles"),
    (256, 8, 8, [1, 1, 1, 13], 4000, "attention_kv4_tiles"), (64, 96, 8, [2] * 4, 6000, "attention_kv4_tiles"),
    (64, 8, 2, [40, 20], 100, "attention_kv4"), (64, 2, 2, [129, 640], 30, "attention_kv4_tiles")])
def test_chunk_routes(d, hq, hkv, new, past, route):
    """Tiles from three lists a sequence on, and not for very little work."""
    import riftco_transformer_b200 as b2
    case = kv4_cases.Case(9, [m + past for m in new], hq, hkv, d, 16, rows=sum(new))
    got, status = chunk(case, new, tiles=False)
    assert status == 0 and b2.last_route() == route
    assert rel_l2(got, case.chunk(new)) <= BF16_TOL


@pytest.mark.parametrize("new,past", [([20, 3], [5000, 64]), ([300], [6000]), ([1, 1, 1], [4000, 0, 63])])
@pytest.mark.parametrize("d", [128, 256])
def test_chunk_splits_long_contexts(new, past, d):
    """Few rows over many tokens: several CTAs, and both row tiles of one, share a row's tokens."""
    case = kv4_cases.Case(sum(new), [p + m for p, m in zip(past, new)], 32, 2, d, 16, rows=sum(new), poison=0x7C)
    got, status = chunk(case, new)
    assert status == 0 and rel_l2(got, case.chunk(new)) <= BF16_TOL
    again, _ = chunk(case, new)
    assert (again == got).all()


def test_chunk_scores_near_and_beyond_the_cap():
    """Both forms of the tanh: scores well below the cap, and far beyond it."""
    for strength, cap in ((1.0, 50.0), (3.0, 2.0), (20.0, 30.0)):
        case = kv4_cases.Case(91, [260], 4, 2, 128, 16, rows=90, strength=strength)
        got, status = chunk(case, [90], softcap=cap)
        assert status == 0
        # fp16 keys and queries move a score by 2 * 2^-11 * |s| at most, a capped one by no more than that of the cap
        tol = BF16_TOL + 2 * 2.0 ** -11 * min(cap, 16.0 * strength)
        assert rel_l2(got, case.chunk([90], softcap=cap)) <= tol


@pytest.mark.parametrize("new,at,window", [(100, 90, 20), (20, 137, 5)])
@pytest.mark.parametrize("d", [128, 256])
def test_chunk_of_values_that_are_not_finite(d, new, at, window):
    """A NaN group of token `at` makes the context NaN for the rows that see it, and for no other."""
    from riftco_transformer_b200 import _lib
    position = np.arange(150 - new, 150)
    for half in (0, 9 * d):   # keys, values
        case = kv4_cases.Case(17, [150], 4, 1, d, 16, rows=new)
        tile = case.pages[case.tables[0, at // 16], 0, 0]
        tile[half + 8 * d:half + 9 * d].reshape(16, -1)[at % 16] = 0xFF
        got, status = chunk(case, [new])
        assert status == _lib.ATTN_STATUS_NAN_OR_POS_INF
        sees = position >= at
        assert np.isnan(got[sees]).all()
        assert rel_l2(got[~sees], case.chunk([new])[~sees]) <= BF16_TOL
        # rows whose window has passed the token do not see it either
        got, status = chunk(case, [new], window=window)
        sees = (position >= at) & (position < at + window)
        assert np.isnan(got[sees]).all()
        assert rel_l2(got[~sees], case.chunk([new], window=window)[~sees]) <= BF16_TOL


def test_chunk_leaves_rows_behind_the_last_sequence():
    for new, d, tiles in (([4, 3], 128, True), ([140, 60], 128, True), ([140, 60], 256, True), ([4, 3], 64, False)):
        lens = [20 + m for m in new]
        case = kv4_cases.Case(5, lens, 8, 2, d, 16, rows=sum(new) + 9)
        got, status = chunk(case, new, extra_rows=9, tiles=tiles)
        assert status == 0 and (got[sum(new):] == 7.0).all()
        assert rel_l2(got[:sum(new)], case.chunk(new)) <= BF16_TOL


@pytest.mark.parametrize("tiles", [False, True])
def test_chunk_longer_than_the_bound_is_flagged(tiles):
    from riftco_transformer_b200 import _lib
    new = [30, 9]
    case = kv4_cases.Case(8, [50, 40], 8, 2, 128, 16, rows=39)
    got, status = chunk(case, new, max_chunk=10, tiles=tiles)
    assert status == _lib.ATTN_STATUS_BAD_BLOCK
    want = case.chunk(new)
    assert rel_l2(got[:10], want[:10]) <= BF16_TOL and rel_l2(got[30:], want[30:]) <= BF16_TOL


@pytest.mark.parametrize("tiles", [False, True])
def test_chunk_longer_than_its_sequence_is_flagged(tiles):
    from riftco_transformer_b200 import _lib
    for new, lens, d in (([6, 2], [4, 30], 128), ([200, 2], [150, 230], 128), ([200, 2], [150, 230], 256)):
        case = kv4_cases.Case(6, lens, 8, 2, d, 16, rows=sum(new))
        got, status = chunk(case, new, max_len=max(lens), tiles=tiles)
        assert status == _lib.ATTN_STATUS_BAD_BLOCK
        short = new[0] - lens[0]
        assert (got[:short] == 0).all()
        case.q = case.q[short:]
        assert rel_l2(got[short:], case.chunk([lens[0], new[1]])) <= BF16_TOL


# ---- a run of them together -------------------------------------------------------------------------

def test_prompt_then_tokens_against_the_fp32_cache():
    """A prompt goes in as a chunk, then tokens one by one; the FP32 cache's own attention over the
    read-back keys and values gives the same contexts."""
    import riftco_transformer_b200 as b2
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    hq, hkv, d, bs, prompt, more = 8, 2, 128, 16, [70, 9], 5
    total = [p + more for p in prompt]
    blocks = [-(-t // bs) for t in total]
    tables = torch.randperm(sum(blocks) + 1, device="cuda", generator=g)[:sum(blocks)].to(torch.int32)
    table = torch.zeros((2, max(blocks)), dtype=torch.int32, device="cuda")
    table[0, :blocks[0]], table[1, :blocks[1]] = tables[:blocks[0]], tables[blocks[0]:]
    pool = b2.PagedKv4Pool.empty(sum(blocks) + 1, hkv, bs, d)
    flat = b2.PagedKvPool(torch.zeros((sum(blocks) + 1, hkv, bs, d), device="cuda"),
                          torch.zeros((sum(blocks) + 1, hkv, bs, d), device="cuda"))
    status = status_word()

    def mirror(positions, owner):
        n = positions.shape[0]
        k, v = torch.empty((n, hkv, d), device="cuda"), torch.empty((n, hkv, d), device="cuda")
        b2.dequantize_kv4(pool, table, positions, k, v, token_seq=owner, status=status)
        page = table[owner.long(), positions.long() // bs].long()
        flat.key_pages[page, :, positions.long() % bs] = k
        flat.value_pages[page, :, positions.long() % bs] = v

    n = sum(prompt)
    rows = [torch.randn((n, h, d), device="cuda", generator=g) for h in (hq, hkv, hkv)]
    positions = torch.cat([torch.arange(p, device="cuda", dtype=torch.int32) for p in prompt])
    owner = torch.repeat_interleave(torch.arange(2, device="cuda", dtype=torch.int32),
                                    torch.tensor(prompt, device="cuda"))
    b2.rope_append_kv4(*rows, positions, pool, table, 1e4, token_seq=owner, status=status)
    mirror(positions, owner)
    ctx = torch.empty((n, hq, d), dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, prompt[0], n], dtype=torch.int32, device="cuda")
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    b2.paged_chunk_attention_kv4(rows[0], pool, table, lens, starts, ctx, max(prompt), max(prompt), status=status)
    want = torch.empty((n, hq, d), device="cuda")
    b2.paged_decode_attention(rows[0], flat, table[owner.long()].contiguous(), positions + 1, want, max(prompt),
                              status=status)
    assert rel_l2(ctx.float().cpu().numpy(), want.cpu().numpy()) <= BF16_TOL
    for step in range(more):
        rows = [torch.randn((2, h, d), device="cuda", generator=g) for h in (hq, hkv, hkv)]
        positions = torch.tensor([p + step for p in prompt], dtype=torch.int32, device="cuda")
        b2.rope_append_kv4(*rows, positions, pool, table, 1e4, status=status)
        mirror(positions, torch.arange(2, device="cuda", dtype=torch.int32))
        got, ref = torch.empty((2, hq, d), device="cuda"), torch.empty((2, hq, d), device="cuda")
        b2.paged_decode_attention_kv4(rows[0], pool, table, positions + 1, got, max(total), status=status)
        b2.paged_decode_attention(rows[0], flat, table, positions + 1, ref, max(total), status=status)
        assert rel_l2(got.cpu().numpy(), ref.cpu().numpy()) <= 2 * F32_TOL
    assert int(status.item()) == 0


@pytest.mark.parametrize("batch,context", [(3, 300), (32, 40)])
def test_decode_step_on_4_bit_pages(batch, context):
    """DecodeStep takes 4-bit pools: two steps give the logits of a step on FP32 pages that hold what the 4-bit ones do,
    the new token's keys and values included. Contexts differ by FP32 rounding; above 16 rows the linears round them
    to bf16, where that flips one in some thousands by half a step of 2^-8: far below 5e-3 in the logits."""
    import riftco_transformer_b200 as b2
    from riftco_transformer_b200.decode import CudaOps, DecodeStep, DecoderConfig, synthetic_step
    cfg = DecoderConfig(layers=2, d_model=512, q_heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=2048)
    dev = torch.device("cuda", 0)
    step, inputs = synthetic_step(cfg, batch, context, device=dev, kv4=True)
    lens = inputs["seq_lens"]

    class Mirror(CudaOps):
        """Appends to a copy of the 4-bit pool and keeps FP32 pages of what it then holds."""

        def rope_append(self, q, k, v, positions, tables, pool, theta, status):
            small = self.small[id(pool)]
            b2.rope_append_kv4(q, k, v, positions, small, tables, theta, status=status)
            kb, vb = torch.empty_like(k), torch.empty_like(v)
            b2.dequantize_kv4(small, tables, positions, kb, vb, status=status)
            page = tables[torch.arange(batch, device=dev), positions.long() // cfg.block_size].long()
            pool.key_pages[page, :, positions.long() % cfg.block_size] = kb
            pool.value_pages[page, :, positions.long() % cfg.block_size] = vb

    ops = Mirror(dev)
    flats, ops.small = [], {}
    for pool in step.pools:
        k, v = (torch.from_numpy(a).to(dev) for a in kv4_cases.unpack(pool.pages.cpu().numpy(), cfg.head_dim))
        flat = b2.PagedKvPool(k, v)
        flats.append(flat)
        ops.small[id(flat)] = b2.PagedKv4Pool(pool.pages.clone(), cfg.block_size, cfg.head_dim)
    other = DecodeStep(cfg, ops, step.w, step.norms, step.embedding, flats, step.tables, batch, context + 1)
    step.ops.launches = 0
    got_next, got = step.step(inputs["tokens"], inputs["positions"], lens)
    want_next, want = other.step(inputs["tokens"], inputs["positions"], lens)
    torch.cuda.synchronize()
    assert int(step.status.item()) == 0 and int(other.status.item()) == 0 and step.ops.launches > 0
    assert rel_l2(got.cpu().numpy(), want.cpu().numpy()) <= 5e-3
    assert inputs["kv_bytes_per_step"] == 2 * batch * (context + 1) * 2 * 144


def test_captured_calls_replay_with_new_inputs():
    import riftco_transformer_b200 as b2
    first, second = (kv4_cases.Case(s, [2000, 700], 8, 2, 128, 16) for s in (41, 42))
    pool = b2.PagedKv4Pool(cuda(first.pages), 16, 128)
    q, tables, lens = cuda(first.q), cuda(first.tables), cuda(np.array(first.lens, np.uint32))
    ctx, status = torch.empty_like(q), status_word()
    need = b2.paged_decode_kv4_workspace_bytes(2, 8, 2, 128, 2000)
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call = lambda: b2.paged_decode_attention_kv4(q, pool, tables, lens, ctx, 2000, status=status,  # noqa: E731
                                                     workspace=workspace)
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for case in (first, second):
            pool.pages.copy_(cuda(case.pages))
            q.copy_(cuda(case.q))
            tables.copy_(cuda(case.tables))
            ctx.fill_(float("nan"))
            graph.replay()
            stream.synchronize()
            assert rel_l2(ctx.cpu().numpy(), case.decode()) <= F32_TOL
    assert int(status.item()) == 0


def test_two_calls_at_once_on_two_streams():
    import riftco_transformer_b200 as b2
    cases = [kv4_cases.Case(s, [3000, 900], 8, 2, 128, 16) for s in (51, 52)]
    need = b2.paged_decode_kv4_workspace_bytes(2, 8, 2, 128, 3000)
    todo = []
    for case in cases:
        todo.append((torch.cuda.Stream(), b2.PagedKv4Pool(cuda(case.pages), 16, 128), cuda(case.q), cuda(case.tables),
                     cuda(np.array(case.lens, np.uint32)), torch.empty(case.q.shape, device="cuda"),
                     torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, pool, q, tables, lens, ctx, workspace in todo:
            b2.paged_decode_attention_kv4(q, pool, tables, lens, ctx, 3000, workspace=workspace, stream=stream)
    torch.cuda.synchronize()
    for case, (_, _, _, _, _, ctx, _) in zip(cases, todo):
        assert rel_l2(ctx.cpu().numpy(), case.decode()) <= F32_TOL


@pytest.mark.parametrize("d,new,past", [(128, [20, 9], [3000, 5000]), (256, [150, 4], [900, 4000])])
def test_chunk_calls_captured_and_on_two_streams(d, new, past):
    """Split chunks: one call captured and replayed with new inputs, then two at once, a workspace each."""
    import riftco_transformer_b200 as b2
    lens = [p + m for p, m in zip(past, new)]
    cases = [kv4_cases.Case(s, lens, 16, 4, d, 16, rows=sum(new)) for s in (71, 72)]
    starts, max_len = cuda(np.array([0, new[0], sum(new)], np.uint32)), max(lens)
    need = b2.paged_chunk_kv4_workspace_bytes(2, sum(new), 16, 4, d, max(new), max_len)
    assert need > 0
    todo = []
    for case in cases:
        todo.append((torch.cuda.Stream(), b2.PagedKv4Pool(cuda(case.pages), 16, d), cuda(case.q), cuda(case.tables),
                     cuda(np.array(lens, np.uint32)), torch.empty(case.q.shape, dtype=torch.bfloat16, device="cuda"),
                     torch.empty(need, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()

    def call(stream, pool, q, tables, lens, ctx, workspace):
        b2.paged_chunk_attention_kv4(q, pool, tables, lens, starts, ctx, max(new), max_len, workspace=workspace, stream=stream)

    for _ in range(10):
        for one in todo:
            call(*one)
    torch.cuda.synchronize()
    assert b2.last_route() == "attention_kv4_tiles"
    want = [case.chunk(new) for case in cases]
    for w, one in zip(want, todo):
        assert rel_l2(one[5].float().cpu().numpy(), w) <= BF16_TOL
    stream, pool, q, tables, _, ctx, _ = todo[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(*todo[0])
    for case, w in zip(reversed(cases), reversed(want)):
        with torch.cuda.stream(stream):
            pool.pages.copy_(cuda(case.pages))
            q.copy_(cuda(case.q))
            tables.copy_(cuda(case.tables))
            ctx.fill_(float("nan"))
            graph.replay()
        stream.synchronize()
        assert rel_l2(ctx.float().cpu().numpy(), w) <= BF16_TOL


# ---- refusals -------------------------------------------------------------------------------------------

def test_refusals():
    import riftco_transformer_b200 as b2
    case = kv4_cases.Case(61, [40, 20], 8, 2, 128, 16)
    pool = b2.PagedKv4Pool(cuda(case.pages), 16, 128)
    q, tables, lens = cuda(case.q), cuda(case.tables), cuda(np.array(case.lens, np.uint32))
    ctx = torch.empty_like(q)

    def call(q=q, pool=pool, tables=tables, lens=lens, ctx=ctx, max_len=40, **rules):
        b2.paged_decode_attention_kv4(q, pool, tables, lens, ctx, max_len, **rules)

    call()
    bad = [
        dict(q=q.half()), dict(q=q[:, :7]), dict(q=q.transpose(0, 1)), dict(q=q[:1]), dict(ctx=None), dict(ctx=q),
        dict(ctx=ctx[:1]), dict(lens=lens.float()), dict(lens=lens[:1]), dict(tables=tables.long()),
        dict(max_len=0), dict(max_len=49), dict(max_len=-1), dict(softcap=-1.0), dict(softcap=float("nan")),
        dict(softcap=float("inf")), dict(softcap=1e-7), dict(softcap=2e18), dict(window=-1),
        dict(alibi_slopes=torch.ones(7, device="cuda")),
        dict(alibi_slopes=torch.ones(8)), dict(context_bf16=torch.empty_like(q)), dict(q=q.cpu()),
        dict(status=torch.zeros(1, device="cuda")), dict(workspace=torch.zeros(16, dtype=torch.uint8)),
        dict(ctx=pool.pages.view(-1)[:q.numel() * 4].view(torch.float32).view(q.shape)),
    ]
    for change in bad:
        with pytest.raises((ValueError, RuntimeError, OverflowError)):
            call(**change)
    torch.cuda.synchronize()
    # q heads that are no multiple of the K/V heads
    with pytest.raises(ValueError):
        call(q=torch.empty((2, 7, 128), device="cuda"), ctx=torch.empty((2, 7, 128), device="cuda"))
    # a workspace that is too small, or badly aligned
    long = kv4_cases.Case(62, [5000], 8, 2, 128, 16)
    args = (cuda(long.q), b2.PagedKv4Pool(cuda(long.pages), 16, 128), cuda(long.tables),
            cuda(np.array([5000], np.uint32)), torch.empty(long.q.shape, device="cuda"), 5000)
    need = b2.paged_decode_kv4_workspace_bytes(1, 8, 2, 128, 5000)
    assert need > 0
    raw = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    for ws in (raw[:need - 1], raw[4:need + 4]):
        with pytest.raises(ValueError):
            b2.paged_decode_attention_kv4(*args, workspace=ws)
    b2.paged_decode_attention_kv4(*args, workspace=raw[:need])

    # chunks
    qc = torch.randn((10, 8, 128), device="cuda")
    out = torch.empty((10, 8, 128), dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, 6, 10], dtype=torch.int32, device="cuda")

    def chunk_call(q=qc, starts=starts, out=out, max_chunk=6, max_len=40, **rules):
        b2.paged_chunk_attention_kv4(q, pool, tables, lens, starts, out, max_chunk, max_len, **rules)

    chunk_call()
    for change in (dict(starts=starts[:2]), dict(out=torch.empty((10, 8, 128), device="cuda")), dict(max_chunk=0),
                   dict(max_chunk=11), dict(max_chunk=41), dict(max_len=49), dict(q=qc[:, :3]),
                   dict(prefix_lens=lens[:1]), dict(softcap=-2.0)):
        with pytest.raises((ValueError, RuntimeError, OverflowError)):
            chunk_call(**change)

    # append
    k = torch.randn((2, 2, 128), device="cuda")
    pos = torch.tensor([3, 4], dtype=torch.int32, device="cuda")

    def put(q=q, k=k, v=k.clone(), pos=pos, theta=1e4, **more):
        b2.rope_append_kv4(q, k, v, pos, pool, tables, theta, **more)

    put(q=q.clone())
    for change in (dict(theta=0.0), dict(theta=-1.0), dict(theta=float("inf")), dict(theta=float("nan")),
                   dict(k=k[:, :1]), dict(k=k.half()), dict(pos=pos.long()), dict(pos=pos[:1]),
                   dict(token_seq=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(queries_out=q[:, :4]),
                   dict(queries_out=k)):
        with pytest.raises((ValueError, RuntimeError, OverflowError)):
            put(**change)
    buffer = torch.randn((3, 8, 128), device="cuda")
    with pytest.raises(ValueError):
        put(q=buffer[:2], queries_out=buffer[1:])   # overlapping, but not the same
    with pytest.raises(ValueError):
        b2.dequantize_kv4(pool, tables, pos, k, k)
    torch.cuda.synchronize()


def test_workspace_growth_is_refused_inside_a_capture():
    """The library's arena must not grow while a stream is captured; a caller's workspace is taken."""
    import riftco_transformer_b200 as b2
    n = 64
    lens = [6000] * n
    need = b2.paged_decode_kv4_workspace_bytes(n, 64, 1, 128, 6000)
    pool = b2.PagedKv4Pool(torch.zeros((400, 1, 1, 18 * 128), dtype=torch.uint8, device="cuda"), 16, 128)
    tables = torch.zeros((n, 375), dtype=torch.int32, device="cuda")
    q = torch.randn((n, 64, 128), device="cuda")
    ctx = torch.empty_like(q)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b2.paged_decode_attention_kv4(q, pool, tables, dl, ctx, 6000, workspace=workspace)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((ctx == 0).all())   # pages of zeros hold zeros
