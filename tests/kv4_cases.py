"""The 4-bit paged K/V cache restated in numpy: its bytes (FP32 arithmetic, every operation rounded,
as the header defines them) and the attention over it in 64 bits."""
import numpy as np


def quantize(x):
    """x [..., d] float32 -> codes uint8 [..., d], scale, base float16 [..., d / 64]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 64)
    with np.errstate(all="ignore"):
        low, high = g.min(-1), g.max(-1)
        base = low.astype(np.float16)
        scale = ((high - base.astype(np.float32)) / np.float32(15)).astype(np.float16)
        step = scale.astype(np.float32)
        inverse = np.where(step > 0, np.float32(1) / step, np.float32(0))
        codes = np.rint((g - base.astype(np.float32)[..., None]) * inverse[..., None])
        codes = np.clip(codes, 0, 15)
    good = np.isfinite(g).all(-1) & (low >= -65000) & (high <= 65000)
    codes = np.where(good[..., None], codes, 0)
    nan = np.array(0x7FFF, np.uint16).view(np.float16)
    return (codes.astype(np.uint8).reshape(x.shape), np.where(good, scale, nan), np.where(good, base, nan))


def values(codes, scale, base):
    """FP32 values: one rounding of base + scale * code."""
    g = codes.reshape(*codes.shape[:-1], -1, 64).astype(np.float64)
    v = base.astype(np.float64)[..., None] + scale.astype(np.float64)[..., None] * g
    return v.astype(np.float32).reshape(codes.shape)


def pack(k, v):
    """k, v float32 [blocks, heads, block_size, d] -> pages uint8 [blocks, heads, block_size / 16, 18 d]."""
    blocks, heads, bs, d = k.shape
    out = np.empty((blocks, heads, bs // 16, 18 * d), np.uint8)
    for at, x in ((0, k), (9 * d, v)):
        codes, scale, base = quantize(x)
        c = codes.reshape(blocks, heads, bs // 16, 16, d // 32, 16, 2)
        rows = (c[..., 0] | (c[..., 1] << 4)).swapaxes(3, 4)
        out[..., at:at + 8 * d] = rows.reshape(blocks, heads, bs // 16, 8 * d)
        pairs = np.stack((scale, base), -1).reshape(blocks, heads, bs // 16, 16 * (d // 64) * 2)
        out[..., at + 8 * d:at + 9 * d] = np.ascontiguousarray(pairs).view(np.uint8)
    return out


def unpack(pages, d):
    """pages -> (k, v) float32 [blocks, heads, block_size, d]."""
    blocks, heads, per, _ = pages.shape
    out = []
    for at in (0, 9 * d):
        rows = pages[..., at:at + 8 * d].reshape(blocks, heads, per, d // 32, 16, 16).swapaxes(3, 4)
        codes = np.stack((rows & 15, rows >> 4), -1).reshape(blocks, heads, per * 16, d)
        pairs = np.ascontiguousarray(pages[..., at + 8 * d:at + 9 * d]).view(np.float16)
        pairs = pairs.reshape(blocks, heads, per * 16, d // 64, 2)
        out.append(values(codes, pairs[..., 0], pairs[..., 1]))
    return out


def attend(q, k, v, position, end=None, softcap=0.0, window=0, slopes=None):
    """One query row q [q_heads, d] at `position` over k, v [kv_heads, tokens, d] in 64 bits; it sees
    tokens below `end` (default position + 1). Returns ctx [q_heads, d]."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rep = q.shape[0] // k.shape[0]
    end = position + 1 if end is None else end
    begin = max(0, position - window + 1) if window else 0
    out = np.zeros_like(q)
    t = np.arange(begin, end)
    if t.size == 0:
        return out
    for h in range(q.shape[0]):
        s = k[h // rep, begin:end] @ q[h] / np.sqrt(q.shape[1])
        if softcap:
            s = softcap * np.tanh(s / softcap)
        if slopes is not None:
            s = s - np.float64(slopes[h]) * np.abs(position - t)
        w = np.exp(s - s.max())
        out[h] = w @ v[h // rep, begin:end] / w.sum()
    return out


class Case:
    """A pool with `lens` tokens per sequence on shuffled pages. Slots that hold no token are filled
    with `poison` bytes; `k`, `v` are what the cache holds, [kv_heads, tokens, d] per sequence."""

    def __init__(self, seed, lens, hq, hkv, d, bs, rows=None, poison=0xFF, strength=1.0, spare=2):
        rng = np.random.default_rng(seed)
        self.lens, self.hq, self.hkv, self.d, self.bs = list(lens), hq, hkv, d, bs
        need = [-(-n // bs) for n in lens]
        blocks = sum(need) + spare
        order = rng.permutation(blocks)[:sum(need)]
        self.tables = np.full((len(lens), max(max(need), 1)), 0xFFFFFFFF, np.uint32)   # unused entries are no block
        pages = np.full((blocks, hkv, bs // 16, 18 * d), poison, np.uint8)
        self.k, self.v, at = [], [], 0
        for i, n in enumerate(lens):
            mine = order[at:at + need[i]]
            at += need[i]
            self.tables[i, :need[i]] = mine
            if n == 0:
                self.k.append(np.zeros((hkv, 0, d)))
                self.v.append(np.zeros((hkv, 0, d)))
                continue
            shape = (need[i], hkv, bs, d)
            spread = np.exp(0.5 * rng.standard_normal(d)) * strength
            k = (rng.standard_normal(shape) * spread).astype(np.float32)
            v = (rng.standard_normal(shape) + 0.3).astype(np.float32)
            packed = pack(k, v)
            rk, rv = unpack(packed, d)
            # bytes of the slots behind the last token become poison
            flat = packed.transpose(0, 2, 1, 3).reshape(need[i] * (bs // 16), hkv, 18 * d)
            for tile in range(flat.shape[0]):
                first = max(0, n - tile * 16)
                if first < 16:
                    for half in (0, 9 * d):
                        flat[tile, :, half:half + 8 * d].reshape(hkv, d // 32, 16, 16)[:, :, first:] = poison
                        flat[tile, :, half + 8 * d:half + 9 * d].reshape(hkv, 16, -1)[:, first:] = poison
            pages[mine] = flat.reshape(need[i], bs // 16, hkv, 18 * d).transpose(0, 2, 1, 3)
            self.k.append(rk.transpose(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n])
            self.v.append(rv.transpose(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n])
        self.pages = pages
        n_rows = len(lens) if rows is None else rows
        self.q = rng.standard_normal((n_rows, hq, d)).astype(np.float32)
        self.slopes = (2.0 ** (-8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32)

    def decode(self, **rules):
        return np.stack([attend(self.q[i], self.k[i], self.v[i], n - 1, **rules) for i, n in enumerate(self.lens)])

    def chunk(self, new, prefix=None, **rules):
        out, at = [], 0
        for i, (n, m) in enumerate(zip(self.lens, new)):
            for p in range(n - m, n):
                end = p + 1 if prefix is None else max(p + 1, min(prefix[i], n))
                out.append(attend(self.q[at], self.k[i], self.v[i], p, end, **rules))
                at += 1
        return np.stack(out) if out else np.zeros((0, self.hq, self.d))
