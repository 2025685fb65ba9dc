"""What is measured of the 4-bit paged K/V cache: appending to it, and the two attentions that read it.

The cache is one uint8 pool [physical_blocks, kv_heads, block_size / 16, 18 * d]. A tile holds 16
consecutive slots of one K/V head: 9d bytes of keys, then 9d bytes of values, each as codes
[d / 32][16 slots][16 bytes] (byte j: channels 2j in the low and 2j + 1 in the high nibble) followed by
[16 slots][d / 64] pairs of fp16 (scale, base). A value is base + scale * code, one pair for 64 channels.

`op` of a case:
  append  rotate q and k at their positions, store k and v in the cache, read the stored tokens back
  decode  one query token per sequence over the cache
  chunk   several new query tokens per sequence (a prompt, or a part of one), causal, over the cache
"""
import math
import random

import torch

own = False

# ---- cases ---------------------------------------------------------------------------------

def _append(name, tokens, seqs, hq, hkv, d, bs, far, theta=1e4):
    return {"name": name, "op": "append", "tokens": tokens, "seqs": seqs, "q_heads": hq, "kv_heads": hkv, "d": d,
            "block": bs, "far": far, "theta": theta}


def _decode(name, seqs, low, high, hq, hkv, d, bs, cap=0.0, window=0, bias=False):
    return {"name": name, "op": "decode", "seqs": seqs, "low": low, "high": high, "q_heads": hq, "kv_heads": hkv,
            "d": d, "block": bs, "cap": cap, "window": window, "bias": bias}


def _chunk(name, seqs, new_low, new_high, past, hq, hkv, d, bs, cap=0.0, window=0, bias=False, prefix=0):
    return {"name": name, "op": "chunk", "seqs": seqs, "new_low": new_low, "new_high": new_high, "past": past,
            "q_heads": hq, "kv_heads": hkv, "d": d, "block": bs, "cap": cap, "window": window, "bias": bias,
            "prefix": prefix}


def listed():
    return [
        # one user generating: a single token goes into the cache, latency is all that counts
        _append("append 1 token", 1, 1, 32, 8, 128, 16, 2048),
        # a serving batch's step, one token per sequence, far into long conversations
        _append("append batch 64", 64, 64, 32, 8, 128, 16, 120000, 5e5),
        # a batch of ragged prompts going in at once, large pages
        _append("append prompt 8191", 8191, 5, 32, 8, 128, 64, 4000),
        # the first words of one conversation: a context that fills two pages and a bit
        _decode("decode 1 x 37", 1, 37, 37, 32, 8, 128, 16),
        # the decode step's own workload: 32 sequences at 2049 tokens
        _decode("decode 32 x 2049", 32, 2049, 2049, 32, 8, 128, 16),
        # a mixed serving batch: 64 sequences of 512 to 8192 tokens
        _decode("decode 64 ragged", 64, 512, 8192, 32, 8, 128, 16),
        # one long document, so few heads that the context has to be cut to fill the card
        _decode("decode 1 x 131071", 1, 131071, 131071, 32, 8, 128, 32),
        # wide heads, capped scores, local layers that see the last 4096 tokens of a longer context
        _decode("decode capped window", 8, 3000, 20000, 16, 8, 256, 16, 50.0, 4096),
        # narrow heads, one K/V head per query head, a bias that falls with distance
        _decode("decode distance bias", 16, 700, 4100, 32, 32, 64, 16, 0.0, 0, True),
        # a few drafted tokens per sequence, verified in one pass
        _chunk("chunk 16 x 5", 16, 3, 5, 2000, 32, 8, 128, 16),
        # a middle part of long prompts, with a cap and a window
        _chunk("chunk 4 x 700 capped", 4, 300, 700, 2500, 16, 8, 128, 16, 30.0, 2000),
        # a whole prompt
        _chunk("chunk 1 x 4096", 1, 4096, 4096, 0, 32, 8, 128, 16),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    d = rng.choice([64, 128, 128, 128, 256])
    bs = rng.choice([16, 16, 32, 64])
    hkv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    hq = hkv * rng.choice([1, 2, 3, 4, 4, 5, 8, 12])
    cap = rng.choice([0.0, 0.0, 0.0, 20.0, 50.0])
    bias = rng.random() < 0.25
    op = rng.choice(["append", "decode", "decode", "chunk"])
    if op == "append":
        tokens = min(_log(rng, 1, 8191), (8191 * 48 * 128) // ((hq + 2 * hkv) * d))
        seqs = rng.randint(1, min(tokens, 70))
        if rng.random() < 0.4:
            tokens = seqs
        c = _append("", tokens, seqs, hq, hkv, d, bs, _log(rng, 64, 200000), rng.choice([1e4, 1e4, 5e5, 1e6]))
    elif op == "decode":
        room = 64 * 4352 * 8 * 128 // (hkv * d) // 2   # half the tokens of the largest listed case
        seqs = min(_log(rng, 1, 100), max(1, room // 64))
        high = min(_log(rng, 1, 60000), max(1, room // seqs))
        low = rng.randint(1, high)
        window = rng.choice([0, 0, 0, _log(rng, 1, 5000)])
        c = _decode("", seqs, low, high, hq, hkv, d, bs, cap, window, bias)
    else:
        room = 32 * 4096 * 4096 * 128 // (hq * d) // 2   # scores over all heads, half the largest listed case
        seqs = min(_log(rng, 1, 20), max(1, room // 4096))
        high = max(1, min(_log(rng, 1, 2500), int(math.sqrt(room / seqs))))
        past = rng.choice([0, max(0, min(_log(rng, 1, 6000), room // seqs // high - high))])
        low = rng.randint(1, high)
        window = rng.choice([0, 0, 0, _log(rng, 1, 3000)])
        prefix = rng.choice([0, 0, 0, rng.randint(1, high + past)])
        c = _chunk("", seqs, low, high, past, hq, hkv, d, bs, cap, window, bias, prefix)
    del c["name"]
    return c


def _lengths(case):
    """Host-side plan of a case, by the case alone: (lengths, new tokens) of its sequences."""
    r = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["seqs"]
    if case["op"] == "append":
        cuts = sorted(r.sample(range(1, case["tokens"]), n - 1)) if n > 1 else []
        new = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
        past = [r.randint(0, case["far"]) for _ in range(n)]
        return [p + k for p, k in zip(past, new)], new
    if case["op"] == "decode":
        lens = [r.randint(case["low"], case["high"]) for _ in range(n)]
        lens[r.randrange(n)] = case["high"]
        return lens, [1] * n
    new = [r.randint(case["new_low"], case["new_high"]) for _ in range(n)]
    new[r.randrange(n)] = case["new_high"]
    past = [r.randint(case["past"] // 2, case["past"]) for _ in range(n)]
    return [p + k for p, k in zip(past, new)], new


# ---- inputs ---------------------------------------------------------------------------------

def _quantise(x):
    """x [..., d] FP32 -> codes [..., d] (FP32 whole numbers), scale and base [..., d / 64] (fp16)."""
    g = x.float().unflatten(-1, (-1, 64))
    low, high = g.amin(-1), g.amax(-1)
    base = low.half()
    span = high - base.float()
    scale = (span / torch.full_like(span, 15.0)).half()   # by a tensor: a true division, not a product with 1/15
    step = scale.float()
    inverse = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    codes = ((g - base.float().unsqueeze(-1)) * inverse.unsqueeze(-1)).round().clamp(0, 15)
    return codes.flatten(-2), scale, base


def _tiles(x):
    """x [n, 16, d] FP32 -> the bytes [n, 9d] of n tiles' keys or values."""
    n, _, d = x.shape
    codes, scale, base = _quantise(x)
    c = codes.to(torch.uint8).view(n, 16, d // 32, 16, 2)
    packed = (c[..., 0] | (c[..., 1] << 4)).transpose(1, 2).reshape(n, 8 * d)
    pairs = torch.stack((scale, base), -1).contiguous().view(torch.uint8).reshape(n, d)
    return torch.cat((packed, pairs), 1)


def _half_of_tile(part):
    """The bytes [..., 9d] of keys or values of tiles -> codes [..., 16, d] and pairs [..., 16, d / 64, 2]."""
    d = part.shape[-1] // 9
    lead = part.shape[:-1]
    packed = part[..., :8 * d].reshape(*lead, d // 32, 16, 16)
    codes = torch.stack((packed & 15, packed >> 4), -1).transpose(-4, -3).reshape(*lead, 16, d)
    pairs = part[..., 8 * d:].contiguous().view(torch.float16).reshape(*lead, 16, d // 64, 2)
    return codes, pairs


def _pool(case, blocks, gen, real=True):
    """A pool whose pages hold keys with a few strong channels and values of one spread."""
    d, hkv, per = case["d"], case["kv_heads"], case["block"] // 16
    pages = torch.empty((blocks, hkv, per, 18 * d), dtype=torch.uint8, device="cuda")
    flat = pages.view(-1, 18 * d)
    if not real:
        return pages.zero_()
    strength = torch.exp(0.5 * torch.randn(d, device="cuda", generator=gen))
    centre = torch.randn(d, device="cuda", generator=gen) * (torch.rand(d, device="cuda", generator=gen) < 0.1)
    for at in range(0, flat.shape[0], 1 << 17):
        n = min(1 << 17, flat.shape[0] - at)
        flat[at:at + n, :9 * d] = _tiles(torch.randn((n, 16, d), device="cuda", generator=gen) * strength + centre)
        flat[at:at + n, 9 * d:] = _tiles(torch.randn((n, 16, d), device="cuda", generator=gen))
    return pages


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lens, new = _lengths(case)
    n, d, bs, hq, hkv = case["seqs"], case["d"], case["block"], case["q_heads"], case["kv_heads"]
    need = [-(-k // bs) for k in lens]
    s = {"case": case, "lens": lens, "new": new}
    if case["op"] == "append":   # only the pages that the new tokens touch are there; earlier ones belong to the past
        first = [(k - m) // bs for k, m in zip(lens, new)]
        need_new = [b - a for a, b in zip(first, need)]
        blocks = sum(need_new) + 3
        order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
        tables = torch.zeros((n, max(need)), dtype=torch.int32, device="cuda")
        at = 0
        for i in range(n):
            tables[i, first[i]:need[i]] = order[at:at + need_new[i]]
            at += need_new[i]
    else:
        blocks = sum(need) + 3
        order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
        tables = torch.zeros((n, max(need)), dtype=torch.int32, device="cuda")
        at = 0
        for i in range(n):
            tables[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
    s["tables"] = tables
    s["seq_lens"] = _ints(lens)
    total = sum(new)
    s["q"] = torch.randn((total, hq, d), device="cuda", generator=gen)
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    s["pages"] = _pool(case, blocks, gen, case["op"] != "append")
    if case["op"] == "append":
        s["k"] = torch.randn((total, hkv, d), device="cuda", generator=gen)
        s["v"] = torch.randn((total, hkv, d), device="cuda", generator=gen)
        s["token_seq"] = torch.repeat_interleave(_ints(list(range(n))), _ints(new).long())
        s["positions"] = torch.cat([torch.arange(k - m, k, device="cuda", dtype=torch.int32)
                                    for k, m in zip(lens, new)])
        s["q_out"] = torch.empty_like(s["q"])
        s["k_read"], s["v_read"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    else:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq) if case["bias"] else None
        starts = [0]
        for m in new:
            starts.append(starts[-1] + m)
        s["starts"] = _ints(starts)
        s["prefix"] = _ints([min(case["prefix"], k) for k in lens]) if case.get("prefix") else None
        s["max_new"], s["max_len"] = max(new), max(lens)
        s["ctx"] = torch.empty((total, hq, d), device="cuda",
                               dtype=torch.float32 if case["op"] == "decode" else torch.bfloat16)
    if own:
        import riftco_transformer_b200 as b2
        s["b2"] = b2
        s["pool"] = b2.PagedKv4Pool(s["pages"], bs, d)
        if case["op"] != "append":
            need_bytes = (b2.paged_decode_kv4_workspace_bytes(n, hq, hkv, d, s["max_len"]) if case["op"] == "decode"
                          else b2.paged_chunk_kv4_workspace_bytes(n, total, hq, hkv, d, s["max_new"], s["max_len"]))
            s["workspace"] = torch.empty(max(need_bytes, 16), dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "chunk": _own_chunk}[op](state)
    return {"append": _plain_append, "decode": _plain_decode, "chunk": _plain_chunk}[op](state)


def _own_append(s):
    b2, c = s["b2"], s["case"]
    one_each = c["tokens"] == c["seqs"]
    owner = None if one_each else s["token_seq"]
    b2.rope_append_kv4(s["q"], s["k"], s["v"], s["positions"], s["pool"], s["tables"], c["theta"], token_seq=owner,
                       queries_out=s["q_out"], status=s["status"])
    b2.dequantize_kv4(s["pool"], s["tables"], s["positions"], s["k_read"], s["v_read"], token_seq=owner,
                      status=s["status"])
    return {"q": s["q_out"], "k": s["k_read"], "v": s["v_read"]}


def _own_decode(s):
    b2, c = s["b2"], s["case"]
    b2.paged_decode_attention_kv4(s["q"], s["pool"], s["tables"], s["seq_lens"], s["ctx"], s["max_len"],
                                  softcap=c["cap"], window=c["window"], alibi_slopes=s["slopes"], status=s["status"],
                                  workspace=s["workspace"])
    return s["ctx"]


def _own_chunk(s):
    b2, c = s["b2"], s["case"]
    b2.paged_chunk_attention_kv4(s["q"], s["pool"], s["tables"], s["seq_lens"], s["starts"], s["ctx"], s["max_new"],
                                 s["max_len"], softcap=c["cap"], window=c["window"], alibi_slopes=s["slopes"],
                                 prefix_lens=s["prefix"], status=s["status"], workspace=s["workspace"])
    return s["ctx"]


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    c = s["case"]
    d, bs = c["d"], c["block"]
    position = s["positions"].long()
    turn = c["theta"] ** (torch.arange(d // 2, device="cuda", dtype=torch.float64) * -2.0 / d)
    angle = position.double()[:, None, None] * turn
    cos, sin = angle.cos().float(), angle.sin().float()
    k = _rotate(s["k"], cos, sin)
    page = s["tables"][s["token_seq"].long(), position // bs].long()
    tile, slot = (position % bs) // 16, position % 16
    tiles = s["pages"].unflatten(-1, (2, 9 * d))   # a view: keys and values of every tile
    read = []
    for which, x in ((0, k), (1, s["v"])):
        codes, scale, base = _quantise(x)
        heads = torch.arange(c["kv_heads"], device="cuda")
        b = codes.to(torch.uint8).unflatten(-1, (d // 32, 16, 2))
        rows = (b[..., 0] | (b[..., 1] << 4))                            # [tokens, heads, d/32, 16]
        at = (page[:, None], heads[None, :], tile[:, None], which)
        stored = tiles[..., :8 * d].unflatten(-1, (d // 32, 16, 16))
        stored[at[0][..., None], at[1][..., None], at[2][..., None], which,
               torch.arange(d // 32, device="cuda"), slot[:, None, None]] = rows
        pairs = torch.stack((scale, base), -1).contiguous().view(torch.uint8).flatten(-2)
        tiles[..., 8 * d:].unflatten(-1, (16, -1))[at[0], at[1], at[2], which, slot[:, None]] = pairs
        read.append((base.float().unsqueeze(-1) + scale.float().unsqueeze(-1) * codes.unflatten(-1, (-1, 64)))
                    .flatten(-2))
    return {"q": _rotate(s["q"], cos, sin), "k": read[0], "v": read[1]}


def _read_cache(s, kind):
    """Keys and values of every sequence, padded to whole pages of the longest: [n, heads, length, d]."""
    d = s["case"]["d"]
    got = s["pages"][s["tables"].long()]                                  # [n, blocks, heads, per, 18d]
    out = []
    for part in got.split(9 * d, -1):
        codes, pairs = _half_of_tile(part)
        value = codes.to(kind).unflatten(-1, (-1, 64)) * pairs[..., :1].to(kind) + pairs[..., 1:].to(kind)
        out.append(value.flatten(-2).permute(0, 2, 1, 3, 4, 5).flatten(2, 4))
    return out


def _softmax_over(scores, seen, values):
    """sum over t of softmax(scores)[t] * values[t] where `seen`; zeros where a row sees nothing."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    weight = (scores - top).exp()
    total = weight.sum(-1, keepdim=True)
    return (weight @ values) / torch.where(total > 0, total, torch.ones_like(total))


def _scores(q, k, case):
    s = (q @ k.transpose(-1, -2)) / math.sqrt(case["d"])
    return torch.tanh(s / case["cap"]) * case["cap"] if case["cap"] else s


def _plain_decode(s):
    c = s["case"]
    n, hq, hkv, d = c["seqs"], c["q_heads"], c["kv_heads"], c["d"]
    k, v = _read_cache(s, torch.float32)
    scores = _scores(s["q"].view(n, hkv, hq // hkv, d), k, c)            # [n, hkv, rep, length]
    at = torch.arange(k.shape[2], device="cuda")
    last = s["seq_lens"].view(n, 1, 1, 1) - 1
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(1, hkv, -1, 1) * (last - at).float()
    seen = at <= last
    if c["window"]:
        seen = seen & (at > last - c["window"])
    return _softmax_over(scores, seen, v).reshape(n, hq, d)


def _plain_chunk(s):
    c = s["case"]
    n, hq, hkv, d = c["seqs"], c["q_heads"], c["kv_heads"], c["d"]
    rep, m = hq // hkv, s["max_new"]
    k, v = _read_cache(s, torch.float32)
    new = s["starts"].diff().long()
    row = torch.arange(m, device="cuda")
    real = row < new[:, None]                                             # [n, m]
    q = torch.zeros((n, m, hq, d), device="cuda")
    q[real] = s["q"]
    q = q.view(n, m, hkv, rep, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, rep * m, d)
    scores = _scores(q, k, c).view(n, hkv, rep, m, -1)
    at = torch.arange(k.shape[2], device="cuda")
    where = (s["seq_lens"].long()[:, None] - new[:, None] + row).view(n, 1, 1, m, 1)
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(1, hkv, rep, 1, 1) * (where - at).abs().float()
    seen = at <= where
    if s["prefix"] is not None:
        seen = seen | (at < s["prefix"].view(n, 1, 1, 1, 1))
    seen = seen & (at < s["seq_lens"].view(n, 1, 1, 1, 1))
    if c["window"]:
        seen = seen & (at > where - c["window"])
    out = _softmax_over(scores.flatten(2, 3), seen.expand(-1, 1, rep, -1, -1).flatten(2, 3), v)
    out = out.view(n, hkv, rep, m, d).permute(0, 3, 1, 2, 4).reshape(n, m, hq, d)
    return out[real].to(torch.bfloat16)


# ---- what a pass cannot do without ------------------------------------------------------------

def _seen(case, lens, new):
    """Scores of one head, and cache tokens that any query of a sequence sees, summed over the sequences."""
    pairs = tokens = 0
    w, prefix = case["window"], case.get("prefix", 0)
    for length, m in zip(lens, new):
        first = length
        for p in range(length - m, length):
            end = min(length, max(p + 1, min(prefix, length)))
            begin = max(0, p - w + 1) if w else 0
            pairs += max(0, end - begin)
            first = min(first, begin)
        tokens += length - first
    return pairs, tokens


def work(case):
    lens, new = _lengths(case)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["d"]
    total = sum(new)
    stored = hkv * 2 * (d // 2 + d // 16)   # bytes of one token in the cache
    if case["op"] == "append":
        # q in and out, k and v in, the cache's bytes written and read, k and v out
        return {"bytes": total * (2 * hq * d * 4 + 4 * hkv * d * 4 + 2 * stored + 12),
                "flops": total * (hq + hkv) * d * 3 + total * hkv * d * 2 * 6}
    pairs, tokens = _seen(case, lens, new)
    out = 4 if case["op"] == "decode" else 2
    return {"bytes": tokens * stored + total * hq * d * (4 + out) + sum(-(-k // case["block"]) for k in lens) * 4,
            "flops": 4 * d * hq * pairs}


# ---- the definition in 64 bits -----------------------------------------------------------------

def _f32(x):
    return x.float().double()


def _exact_append(s):
    c = s["case"]
    d = c["d"]
    out = {}
    p = s["positions"].double().view(-1, 1)
    channel = torch.arange(0, d, 2, device="cuda", dtype=torch.float64)
    angle = p * torch.pow(torch.tensor(c["theta"], dtype=torch.float64, device="cuda"), -channel / d)
    cos, sin = _f32(torch.cos(angle)).unsqueeze(1), _f32(torch.sin(angle)).unsqueeze(1)
    turned = {}
    for name in ("q", "k"):
        x = s[name].double()
        a, b = x[..., :d // 2], x[..., d // 2:]
        # products and sums of FP32 numbers, each rounded to FP32 as the definition says
        turned[name] = torch.cat((_f32(_f32(a * cos) - _f32(b * sin)), _f32(_f32(b * cos) + _f32(a * sin))), -1)
    out["q"] = turned["q"]
    for name, x in (("k", turned["k"]), ("v", s["v"].double())):
        groups = x.reshape(*x.shape[:-1], d // 64, 64)
        base = groups.min(-1, keepdim=True).values.half().double()
        scale = _f32(_f32(groups.max(-1, keepdim=True).values - base) / 15.0).half().double()
        back = torch.where(scale > 0, _f32(1.0 / scale.clamp_min(1e-30)), torch.zeros_like(scale))
        code = torch.round(_f32(_f32(groups - base) * back)).clamp(0.0, 15.0)
        out[name] = (base + scale * code).reshape(x.shape)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    rows, d, hq, hkv = [], case["d"], case["q_heads"], case["kv_heads"]
    slopes = torch.zeros(hq, dtype=torch.float64, device="cuda") if s["slopes"] is None else s["slopes"].double()
    begin = 0
    for i, (length, m) in enumerate(zip(s["lens"], s["new"])):
        blocks = -(-length // case["block"])
        tile = s["pages"][s["tables"][i, :blocks].long()].transpose(0, 1).reshape(hkv, -1, 18 * d)
        kv = []
        for part in (tile[..., :9 * d], tile[..., 9 * d:]):
            codes, pairs = _half_of_tile(part)
            pairs = pairs.double().repeat_interleave(64, dim=-2)
            kv.append((codes.double() * pairs[..., 0] + pairs[..., 1]).reshape(hkv, -1, d)[:, :length])
        pos = torch.arange(length - m, length, device="cuda").view(-1, 1)
        t = torch.arange(length, device="cuda").view(1, -1)
        limit = pos + 1
        if s.get("prefix") is not None:
            limit = limit.clamp_min(int(s["prefix"][i]))
        hidden = t >= limit
        if case["window"]:
            hidden = hidden | (t <= pos - case["window"])
        q = s["q"][begin:begin + m].double()
        got = torch.empty((m, hq, d), dtype=torch.float64, device="cuda")
        for h in range(hq):
            g = h // (hq // hkv)
            x = q[:, h] @ kv[0][g].T / math.sqrt(d)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            x = x - slopes[h] * (pos - t).abs()
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            got[:, h] = x @ kv[1][g]
        rows.append(got)
        begin += m
    return torch.cat(rows)
