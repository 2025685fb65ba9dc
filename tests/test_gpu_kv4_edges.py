"""The 4-bit paged K/V cache on the GPU at the edges of what its calls allow: rows and tokens that are nobody's,
groups whose stored scale is negative, weights far below the largest, queries and bounds of any size.

Tolerances. FP32 contexts and those of the tile kernel as in test_gpu_kv4.py (F32_TOL, BF16_TOL, derived there); a context
of the row-by-row form is the FP32 one rounded to bf16, half a step of which is 2^-8 of a value: ROW_TOL. Where a test has
another bound its derivation stands beside it."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv4_cases
from conftest import rel_l2
from test_gpu_kv4 import BF16_TOL, F32_TOL, chunk, cuda, decode, guarded_bf16, status_word

pytestmark = pytest.mark.gpu

ROW_TOL = 2.0 ** -8 + F32_TOL


class Held(kv4_cases.Case):
    """A cache that holds given keys and values, [kv_heads, tokens, d] of each sequence, on pages in order."""

    def __init__(self, q, k, v, bs=16):
        self.hq, (self.hkv, _, self.d), self.bs = q.shape[1], k[0].shape, bs
        self.q, self.lens = np.asarray(q, np.float32), [x.shape[1] for x in k]
        need = [-(-n // bs) for n in self.lens]
        self.tables = np.full((len(k), max(need)), 0xFFFFFFFF, np.uint32)
        self.k, self.v, pages, at = [], [], [], 0
        for i, n in enumerate(self.lens):
            held = []
            for x in (k[i], v[i]):
                x = np.concatenate((x, np.zeros((self.hkv, need[i] * bs - n, self.d))), 1).astype(np.float32)
                held.append(x.reshape(self.hkv, need[i], bs, self.d).swapaxes(0, 1))
            packed = kv4_cases.pack(*held)
            for to, x in zip((self.k, self.v), kv4_cases.unpack(packed, self.d)):
                to.append(x.swapaxes(0, 1).reshape(self.hkv, -1, self.d)[:, :n])
            pages.append(packed)
            self.tables[i, :need[i]] = np.arange(at, at + need[i])
            at += need[i]
        self.pages = np.concatenate(pages)
        self.slopes = None


# ---- rows behind the last sequence, row by row -------------------------------------------------

PADDED = [   # lengths, new tokens, rows of the call, max_seq_len, q heads, K/V heads
    ([1000], [1], 64, 1000, 4, 1),
    ([300] * 4, [1] * 4, 64, 300, 16, 4),
    ([60] * 10 + [0] * 6, [1] * 10 + [0] * 6, 32, 2048, 32, 8),
    ([1000] * 2 + [0] * 62, [1] * 2 + [0] * 62, 128, 4096, 32, 8),
    ([50], [1], 5, 400, 8, 8),
    ([700, 0, 37], [2, 0, 2], 8, 2500, 24, 2),
    ([0, 0], [0, 0], 16, 3000, 8, 2),
]


def padded_call(lens, new, rows, max_len, hq, hkv, d, seed=81):
    """A case, and a function that runs it in a call of `rows` rows and returns (contexts, status)."""
    import riftco_transformer_b200 as b2
    case = kv4_cases.Case(seed, lens, hq, hkv, d, 16, rows=sum(new))
    tables = np.full((len(lens), -(-max_len // 16)), 0xFFFFFFFF, np.uint32)
    tables[:, :case.tables.shape[1]] = case.tables
    q = np.concatenate((case.q, np.full((rows - sum(new), hq, d), np.nan, np.float32)))
    pool, q, tables = b2.PagedKv4Pool(cuda(case.pages), 16, d), cuda(q), cuda(tables)
    seq_lens, starts = cuda(np.array(lens, np.uint32)), cuda(np.concatenate(([0], np.cumsum(new))).astype(np.uint32))
    need = b2.paged_chunk_kv4_workspace_bytes(len(lens), rows, hq, hkv, d, max(1, max(new)), max_len)
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    ctx, check = guarded_bf16((rows, hq, d))
    status = status_word()

    def launch():
        b2.paged_chunk_attention_kv4(q, pool, tables, seq_lens, starts, ctx, max(1, max(new)), max_len, status=status,
                                     workspace=workspace)

    def run(how=launch):
        workspace.fill_(0xFF)   # NaN: nothing that the call has not written may be joined
        ctx.fill_(7.0)
        status.zero_()
        how()
        check()
        assert bool((ctx[sum(new):] == 7.0).all())
        return ctx[:sum(new)].float().cpu().numpy(), int(status.item())
    return case, run, launch, (pool, q, tables, seq_lens, starts)


@pytest.mark.parametrize("lens,new,rows,max_len,hq,hkv", PADDED)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_are_nobodys_take_no_part_in_the_join(lens, new, rows, max_len, hq, hkv, d):
    import riftco_transformer_b200 as b2
    case, run, _, _ = padded_call(lens, new, rows, max_len, hq, hkv, d)
    out, status = run()
    assert b2.last_route() == "attention_kv4" and status == 0
    if sum(new):
        assert rel_l2(out, case.chunk(new)) <= ROW_TOL


def test_padded_call_captured_once_and_replayed_with_other_batches():
    """16 slots and 32 rows, from one live token at length 40 to two in every slot at 900."""
    batches = [([40] + [0] * 15, [1] + [0] * 15), ([900] * 16, [2] * 16), ([7, 900, 0, 333] * 4, [1, 2, 0, 2] * 4),
               ([0] * 16, [0] * 16), ([1] * 3 + [0] * 13, [1] * 3 + [0] * 13)]
    cases = [padded_call(lens, new, 32, 2048, 16, 4, 128, seed=90 + i) for i, (lens, new) in enumerate(batches)]
    # the graph's own buffers, as many pages as the largest batch takes
    captured = padded_call(*batches[1], 32, 2048, 16, 4, 128, seed=91)
    _, run, launch, buffers = captured
    launch()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        launch()

    def replay():
        torch.cuda.synchronize()
        graph.replay()
    for i in (0, 2, 1, 3, 4):
        case, _, _, (pool, *rest) = cases[i]
        buffers[0].pages[:pool.pages.shape[0]].copy_(pool.pages)
        for to, x in zip(buffers[1:], rest):
            to.copy_(x)
        live = sum(batches[i][1])
        out, status = run(replay)
        assert status == 0 and (out[live:] == 7.0).all()
        if live:
            assert rel_l2(out[:live], case.chunk(batches[i][1])) <= ROW_TOL


# ---- groups whose fp16 base lies above their largest value -------------------------------------

def rounded_up(kind, d, tokens=300):
    """Values [1, tokens, d] with constant groups that fp16 rounds up (1.0005 to 1.000977, 1000.3 to 1000.5): their stored
    scale, (largest - base) / 15, is negative."""
    rng = np.random.default_rng(d)
    v = np.full((1, tokens, d), 1.0005)
    if kind == "large beside small":   # the small one's scale is 1.6e-6
        v[:] = 1000.3
        if d == 64:
            v[:, 1::2] = 0.1
        else:
            v[..., 64:128] = 0.1
    elif kind == "ordinary later":
        v[:, 200:] = rng.standard_normal((1, tokens - 200, d)) + 0.3
    elif kind == "ordinary before":
        v[:, :100] = rng.standard_normal((1, 100, d)) + 0.3
    return v


SCALES = ["constant", "large beside small", "ordinary later", "ordinary before"]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq", [4, 12])
@pytest.mark.parametrize("kind", SCALES)
def test_values_of_negative_scale(kind, d, hq):
    rng = np.random.default_rng(7)
    v = rounded_up(kind, d)
    assert (kv4_cases.quantize(v.astype(np.float32))[1] < 0).any()
    k = 0.5 * rng.standard_normal(v.shape)
    case = Held(rng.standard_normal((3, hq, d)), [k], [v])

    def check(out, want, tolerance):
        for group in range(d // 64):   # each by itself: they differ by orders of magnitude
            part = (..., slice(64 * group, 64 * group + 64))
            assert rel_l2(out[part], want[part]) <= tolerance
    want = case.chunk([3])
    for tiles, tolerance in ((False, ROW_TOL), (True, BF16_TOL)):
        out, status = chunk(case, [3], tiles=tiles)
        assert status == 0
        check(out, want, tolerance)
    case.q = case.q[2:]
    out, status = decode(case)
    assert status == 0
    check(out, want[2:], F32_TOL)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_stores_negative_scales_as_defined(d):
    """Code 0 and the rounded base: the bytes of the restatement, and read back the base alone."""
    import riftco_transformer_b200 as b2
    for kind in SCALES:
        v = np.ascontiguousarray(rounded_up(kind, d, 304).swapaxes(0, 1), np.float32)   # [tokens, 1, d]
        q = np.zeros((304, 1, d), np.float32)
        pool = b2.PagedKv4Pool(torch.zeros((19, 1, 1, 18 * d), dtype=torch.uint8, device="cuda"), 16, d)
        tables, positions = cuda(np.arange(19, dtype=np.uint32)[None]), cuda(np.arange(304, dtype=np.uint32))
        owner, status = cuda(np.zeros(304, np.uint32)), status_word()
        b2.rope_append_kv4(cuda(q), cuda(q), cuda(v), positions, pool, tables, 1e4, token_seq=owner, status=status)
        by_page = v[:, 0].reshape(19, 1, 16, d)
        want = kv4_cases.pack(np.zeros_like(by_page), by_page)
        assert (pool.pages.cpu().numpy()[..., 9 * d:] == want[..., 9 * d:]).all()
        k_out, v_out = torch.empty((304, 1, d), device="cuda"), torch.empty((304, 1, d), device="cuda")
        b2.dequantize_kv4(pool, tables, positions, k_out, v_out, token_seq=owner, status=status)
        codes, scale, base = kv4_cases.quantize(v)
        assert (v_out.cpu().numpy() == kv4_cases.values(codes, scale, base)).all() and int(status.item()) == 0


# ---- weights far below the largest -------------------------------------------------------------

def peaked(d, hq, new, tokens, period):
    """Every `period`-th token has a key that lifts its score 20 to 29 (log2 units, by head) above the others' of zero, and
    values of zero, so that the context is what the many small weights carry. Queries and keys are exact in fp16 and the
    product of both with 1 / sqrt(d) is the score: the tile kernel's operands round nothing of it."""
    rng = np.random.default_rng(d + period)
    k = np.zeros((1, tokens, d))
    k[:, ::period] = np.float16(25.5 * np.log(2.0) / np.sqrt(d))
    v = 1.0 + 0.25 * rng.standard_normal((1, tokens, d))
    v[:, ::period] = 0.0
    q = np.ones((new, hq, d)) * (0.8125 + 0.0625 * (np.arange(hq) % 6))[:, None]
    return Held(q, [k], [v], bs=64)


def small_weight_bound(case, want, period):
    """A weight is fp16 against at least 2^7 at the peak: half a step, 2^-11 of it or 2^-25 / 2^7 = 2^-32 of the largest,
    `period` of them under each peak; values round by 2^-11 and the context by 2^-8, the exponential and FP32 sums by
    less than 2^-18."""
    largest = max(np.abs(v).max() for v in case.v)
    return period * 2.0 ** -32 * largest + (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -18) * np.abs(want)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,new", [(4, 5), (4, 40)])   # one tile's rows, and two tiles'
def test_chunk_small_weights_under_a_peak(d, hq, new):
    case = peaked(d, hq, new, 5000, 512)
    out, status = chunk(case, [new])
    want = case.chunk([new])
    # (a value's group rounds to 4 bits before; what the cache holds is what `want` averages)
    assert status == 0
    assert (np.abs(out - want) <= small_weight_bound(case, want, 512)).all()


def test_chunk_peak_over_131071_flat_tokens():
    """One peak at the context's start, the rest of it read by the same CTA: 148 sequences over the same pages leave no
    SM to split them for."""
    import riftco_transformer_b200 as b2
    n, new, hq, d, seqs = 131072, 4, 4, 128, 148
    case = peaked(d, hq, new, n, n)
    pool = b2.PagedKv4Pool(cuda(case.pages), case.bs, d)
    ctx = torch.empty((seqs * new, hq, d), dtype=torch.bfloat16, device="cuda")
    status = status_word()
    assert b2.paged_chunk_kv4_workspace_bytes(seqs, seqs * new, hq, 1, d, new, n) == 0   # not split
    b2.paged_chunk_attention_kv4(cuda(np.tile(case.q, (seqs, 1, 1))), pool, cuda(np.tile(case.tables, (seqs, 1))),
                                 cuda(np.full(seqs, n, np.uint32)), cuda(np.arange(0, seqs * new + 1, new, dtype=np.uint32)),
                                 ctx, new, n, status=status)
    assert b2.last_route() == "attention_kv4_tiles" and int(status.item()) == 0
    out = ctx.view(seqs, new, hq, d)
    assert bool((out == out[:1]).all())
    want = case.chunk([new])
    assert (np.abs(out[0].float().cpu().numpy() - want) <= small_weight_bound(case, want, n)).all()


# ---- scores and queries of any finite magnitude ------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("power", [-120, 0, 20, 60, 112])
def test_chunk_scores_of_any_finite_magnitude(d, tiles, power):
    """Keys that are constant over a token, one of them the largest, queries 2^power times 1 or 2: large scores (up to 2^119,
    inside FP32) pick that token, tiny ones weigh all alike. Keys and queries are exact in fp16."""
    rng = np.random.default_rng(d)
    n, new, hq = 200, 6, 4
    k = np.broadcast_to((np.arange(n) % 64 / 64.0 + (np.arange(n) // 64) / 4.0)[None, :, None], (1, n, d))
    v = rng.standard_normal((1, n, d)) + 0.3
    q = np.exp2(power) * rng.integers(1, 3, (new, hq, 1)) * np.ones((1, 1, d))
    case = Held(q, [k], [v])
    out, status = chunk(case, [new], tiles=tiles)
    assert status == 0
    assert rel_l2(out, case.chunk([new])) <= (BF16_TOL if tiles else ROW_TOL)


def a_step_apart(d, hq, power):
    """Scores of about 1.5 * 2^power (log2 units) that rise by 4 every 128 tokens: at 2^25 by one step of FP32, which decides
    between tokens as it will, but a context is an average of values. Returns a case of 4 rows, and the values' extremes."""
    n = 3000
    rng = np.random.default_rng(power)
    k = np.ones((1, n, d))
    k[..., 64:] = np.arange(n)[None, :, None] // 128 / 4.0
    v = rng.standard_normal((1, n, d)) + 0.3
    unit = np.sqrt(d) / np.log2(np.e) / 64
    q = np.full((4, hq, d), 0.0)
    q[..., :64], q[..., 64:128] = 1.5 * 2.0 ** power * unit, 16.0 * unit
    case = Held(q, [k], [v])
    return case, case.v[0].min(1)[0], case.v[0].max(1)[0]


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("hq", [4, 8])
@pytest.mark.parametrize("power", range(18, 31))
def test_chunk_scores_a_rounding_step_apart(d, hq, power):
    case, low, high = a_step_apart(d, hq, power)
    out, status = chunk(case, [4])
    assert status == 0
    # 2^-7 covers the context's bf16 and the values' fp16
    assert (out >= low - 2.0 ** -7 * np.abs(low)).all() and (out <= high + 2.0 ** -7 * np.abs(high)).all()


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("hq", [4, 8])
@pytest.mark.parametrize("power", range(18, 31))
def test_decode_scores_a_rounding_step_apart(d, hq, power):
    case, low, high = a_step_apart(d, hq, power)
    out, status = chunk(case, [4], tiles=False)
    assert status == 0
    assert (out >= low - ROW_TOL * np.abs(low)).all() and (out <= high + ROW_TOL * np.abs(high)).all()
    case.q = case.q[-1:]
    out, status = decode(case)
    assert status == 0
    assert (out >= low - F32_TOL * np.abs(low)).all() and (out <= high + F32_TOL * np.abs(high)).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("power", [116, 118, 123])
def test_chunk_queries_near_the_end_of_fp32(d, tiles, power):
    """Queries of 2^power and twice that over keys of 2^-14 to 2^-13 (scores up to 2^118): the largest key's token is picked,
    the queries' size overflows nothing."""
    rng = np.random.default_rng(d)
    n, new, hq = 200, 6, 4
    k = np.broadcast_to(2.0 ** -14 * (1.0 + np.arange(n) % 191 / 256.0)[None, :, None], (1, n, d))
    v = rng.standard_normal((1, n, d)) + 0.3
    q = np.exp2(power) * rng.integers(1, 3, (new, hq, 1)) * np.ones((1, 1, d))
    case = Held(q, [k], [v])
    out, status = chunk(case, [new], tiles=tiles)
    assert status == 0
    assert rel_l2(out, case.chunk([new])) <= (BF16_TOL if tiles else ROW_TOL)


# ---- chunk starts past the call's rows ----------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,claimed,tiles", [([5, 4], 7, False), ([60, 70], 75, True), ([9, 0], 3, False), ([130, 0], 5, True)])
def test_chunk_starts_past_the_rows_are_flagged(d, new, claimed, tiles):
    """The last sequence says it has more new tokens than the call has rows: the rows there are get the contexts of their
    positions, in both forms, and the call is flagged."""
    import riftco_transformer_b200 as b2
    from riftco_transformer_b200 import _lib
    case = kv4_cases.Case(91, [max(40, new[0]), 150], 8, 8, d, 16, rows=sum(new))
    ctx, check = guarded_bf16(case.q.shape)
    status = status_word()
    b2.paged_chunk_attention_kv4(cuda(case.q), b2.PagedKv4Pool(cuda(case.pages), 16, d), cuda(case.tables),
                                 cuda(np.array(case.lens, np.uint32)), cuda(np.array([0, new[0], new[0] + claimed], np.uint32)),
                                 ctx, max(claimed, new[0]), 150, status=status)
    check()
    assert b2.last_route() == ("attention_kv4_tiles" if tiles else "attention_kv4")
    assert int(status.item()) == _lib.ATTN_STATUS_BAD_BLOCK
    want = [kv4_cases.attend(case.q[i], case.k[0], case.v[0], case.lens[0] - new[0] + i) for i in range(new[0])]
    want += [kv4_cases.attend(case.q[new[0] + i], case.k[1], case.v[1], 150 - claimed + i) for i in range(new[1])]
    assert rel_l2(ctx.float().cpu().numpy(), np.stack(want)) <= (BF16_TOL if tiles else ROW_TOL)


# ---- a window over a bound at which the sums of all lists pass 32 bits ------------------------

@pytest.mark.parametrize("given", [False, True])
def test_window_under_the_largest_bound(given):
    """64 sequences with a capacity of 2^31 - 1 tokens: the size query answers 0, with a window or without, and the call
    asks for no more."""
    import riftco_transformer_b200 as b2
    n, d, bs, max_len = 64, 64, 1 << 20, 0x7FFFFFFF
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((1, 64, d)) for _ in range(2))
    case = Held(rng.standard_normal((n, 1, d)), [k] * n, [v] * n)
    pages = torch.zeros((1, 1, bs // 16, 18 * d), dtype=torch.uint8, device="cuda")
    pages[0, 0, :4] = cuda(case.pages[:4, 0, 0])
    pool = b2.PagedKv4Pool(pages, bs, d)
    tables = torch.zeros((n, 2048), dtype=torch.int32, device="cuda")
    lens = np.arange(1, n + 1).astype(np.uint32)
    assert b2.paged_decode_kv4_workspace_bytes(n, 1, 1, d, max_len) == 0
    workspace = torch.empty(16, dtype=torch.uint8, device="cuda") if given else None
    out = torch.empty((n, 1, d), device="cuda")
    for window in (0, 1, 20, 1000, 1 << 30):
        out.fill_(float("nan"))
        status = status_word()
        b2.paged_decode_attention_kv4(cuda(case.q), pool, tables, cuda(lens), out, max_len, window=window, status=status,
                                      workspace=workspace)
        want = np.stack([kv4_cases.attend(case.q[i], case.k[i], case.v[i], i, window=window) for i in range(n)])
        assert int(status.item()) == 0 and rel_l2(out.cpu().numpy(), want) <= F32_TOL


# ---- forms that the other tests reach at one width only ----------------------------------------

RULES = [dict(softcap=5.0), dict(bias=True), dict(softcap=20.0, window=40, bias=True), dict(window=33)]


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("hq", [2, 8, 16])
@pytest.mark.parametrize("rules", RULES)
def test_decode_score_rules_at_other_widths(rules, hq, d):
    case = kv4_cases.Case(101, [1, 16, 33, 700, 3000], hq, 2, d, 16)
    out, status = decode(case, **rules)
    rules = dict(rules)
    if rules.pop("bias", False):
        rules["slopes"] = case.slopes
    assert status == 0
    assert rel_l2(out, case.decode(**rules)) <= F32_TOL


@pytest.mark.parametrize("new,past", [([5, 2], [90, 20]), ([150, 260], [33, 0]), ([4], [5000])])
@pytest.mark.parametrize("rules", RULES + [dict(prefix=[70, 10])])
def test_chunk_score_rules_with_heads_of_64(rules, new, past):
    rules = dict(rules)
    if "prefix" in rules:
        rules["prefix"] = rules["prefix"][:len(new)]
    case = kv4_cases.Case(102, [p + m for p, m in zip(past, new)], 4, 2, 64, 16, rows=sum(new))
    for tiles, tolerance in ((True, BF16_TOL), (False, ROW_TOL)):
        if not tiles and sum(new) > 16:
            continue
        out, status = chunk(case, new, tiles=tiles, **rules)
        plain = dict(rules)
        if plain.pop("bias", False):
            plain["slopes"] = case.slopes
        assert status == 0
        assert rel_l2(out, case.chunk(new, **plain)) <= tolerance


@pytest.mark.parametrize("hq", [4, 7])
def test_decode_of_more_rows_than_a_cta_looks_through(hq):
    lens = [1 + i % 37 for i in range(1100)]
    lens[7], lens[500], lens[1099] = 2000, 0, 901
    case = kv4_cases.Case(103, lens, hq, 1, 128, 16)
    out, status = decode(case)
    assert status == 0
    assert rel_l2(out, case.decode()) <= F32_TOL


@pytest.mark.parametrize("d,hq,hkv,new,past", [(128, 32, 8, [5, 3, 4], [2000, 1500, 900]), (128, 16, 8, [300], [1000]),
                                               (64, 8, 2, [40, 7], [3000, 100]), (256, 16, 4, [150], [2000])])
def test_a_call_repeats_itself_bit_for_bit(d, hq, hkv, new, past):
    """Partial results are joined in a fixed order, with no atomics on values."""
    case = kv4_cases.Case(104, [p + m for p, m in zip(past, new)], hq, hkv, d, 16, rows=sum(new))
    for rules in (dict(), dict(softcap=30.0, bias=True)):
        first, _ = chunk(case, new, **rules)
        for _ in range(3):
            assert (chunk(case, new, **rules)[0] == first).all()
    rows, case.q = case.q, case.q[:len(new)]
    first, _ = decode(case)
    for _ in range(3):
        assert (decode(case)[0] == first).all()
    case.q = rows


def test_arena_growth_is_refused_inside_a_capture():
    """Without a workspace a call that needs more than the library's arena holds is refused while its stream is captured;
    nothing of it is enqueued, and the capture goes on. (The bound below asks for 7 GB, which is never allocated.)"""
    import riftco_transformer_b200 as b2
    d, bs = 64, 1 << 20
    pool = b2.PagedKv4Pool(torch.zeros((1, 1, bs // 16, 18 * d), dtype=torch.uint8, device="cuda"), bs, d)
    tables = torch.zeros((8, 2048), dtype=torch.int32, device="cuda")
    q, lens = torch.randn((8, 4, d), device="cuda"), torch.full((8,), 30, dtype=torch.int32, device="cuda")
    ctx = torch.full_like(q, float("nan"))
    assert b2.paged_decode_kv4_workspace_bytes(8, 4, 1, d, 0x7FFFFFFF) > 1 << 32
    b2.paged_decode_attention_kv4(q, pool, tables, lens, ctx, 30)
    ctx.fill_(float("nan"))
    refused, graph = None, torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b2.paged_decode_attention_kv4(q, pool, tables, lens, ctx, 30)
        try:
            b2.paged_decode_attention_kv4(q, pool, tables, lens, ctx, 0x7FFFFFFF)
        except ValueError as e:
            refused = str(e)
    assert refused is not None and "stream capture" in refused
    graph.replay()
    torch.cuda.synchronize()
    assert bool((ctx == 0).all())   # pages of zeros hold zeros
