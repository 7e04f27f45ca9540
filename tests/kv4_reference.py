"""Plain 64-bit (and, for the stored bits, IEEE 32-bit) restatement of the 4-bit key/value cache, on the CPU."""
import numpy as np

SHIFTS = (0, 8, 16, 24, 4, 12, 20, 28)


def quantise(x16):
    """fp16 rows [..., 128] -> (codes words uint32 [..., 16], scale fp16, zero fp16): the header's formula in IEEE fp32."""
    x = x16.astype(np.float32)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1), x.max(-1)
        scale = ((hi - lo) / np.float32(15)).astype(np.float16)
        s = scale.astype(np.float32)
        zero = (lo + np.float32(8) * s).astype(np.float16)
        z = zero.astype(np.float32)
        code = np.where(s[..., None] > 0, np.rint((x - z[..., None]) / np.where(s > 0, s, 1)[..., None]) + 8, 8)
    bad = ~np.isfinite(x).all(-1)
    code = np.where(bad[..., None], 8, code)
    scale, zero = np.where(bad, np.float16("nan"), scale), np.where(bad, np.float16("nan"), zero)
    code = np.clip(code, 0, 15).astype(np.uint64).reshape(*x.shape[:-1], 16, 8)
    words = sum(code[..., j] << np.uint64(SHIFTS[j]) for j in range(8)).astype(np.uint32)
    return words, scale, zero


def rotate(x64, positions, inv_freq):
    """Rows [tokens, heads, 128] in 64 bits, pairs (d, d + 64) turned by positions * inv_freq."""
    angle = positions.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x64[..., :64], x64[..., 64:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


class Pool:
    """A pool in host memory with the device layout."""

    def __init__(self, num_pages, kv_heads, page_size, fill=0):
        self.words = np.full((num_pages, kv_heads, 34 * page_size), fill, np.uint32)
        self.weight = np.zeros((num_pages, kv_heads, page_size), np.float32)
        self.kv, self.ps, self.num_pages = kv_heads, page_size, num_pages

    def put(self, page, head, slot, part, words, scale, zero):
        rec = self.words[page, head]
        rec[(part * self.ps + slot) * 16:][:16] = words
        rec[(32 + part) * self.ps + slot] = np.uint32(scale.view(np.uint16)) | (np.uint32(zero.view(np.uint16)) << np.uint32(16))

    def row(self, page, head, slot, part):
        rec = self.words[page, head]
        w = rec[(part * self.ps + slot) * 16:][:16]
        code = np.stack([(w >> np.uint32(s)) & np.uint32(15) for s in SHIFTS], -1).reshape(-1).astype(np.float64)
        p = int(rec[(32 + part) * self.ps + slot])
        scale, zero = (np.array([p & 0xFFFF, p >> 16], np.uint16).view(np.float16).astype(np.float64))
        return (code - 8) * scale + zero

    def rows(self, table_row, head, n, part):
        """Positions 0 .. n of a sequence, 64 bits; the pages' numbers that are no pages give None rows."""
        out, there = np.zeros((n, 128)), np.zeros(n, bool)
        for j in range(n):
            page = int(table_row[j // self.ps])
            if 0 <= page < self.num_pages:
                out[j], there[j] = self.row(page, head, j % self.ps, part), True
        return out, there

    def fill_random(self, rng, key_scale=1.0, value_scale=1.0):
        x = (rng.standard_normal((self.num_pages, self.kv, 2, self.ps, 128)) * np.array([key_scale, value_scale])[:, None, None]).astype(np.float16)
        w, s, z = quantise(x)
        ps = self.ps
        for part in range(2):
            self.words[..., part * 16 * ps:(part + 1) * 16 * ps] = w[:, :, part].reshape(self.num_pages, self.kv, -1)
            self.words[..., (32 + part) * ps:(33 + part) * ps] = (
                s[:, :, part].view(np.uint16).astype(np.uint32) | (z[:, :, part].view(np.uint16).astype(np.uint32) << np.uint32(16)))
        return self


def spans(lens, new):
    """(sequence, first row of the batch, length, new tokens) of every sequence."""
    first = 0
    for b, (L, n) in enumerate(zip(lens, new)):
        yield b, first, L, n
        first += n


def attention(pool, table, lens, new, q, scale, fp16_rows=False):
    """q [tokens, heads, 128] -> out, lse, and bounds of the 32-bit result's error: the tokens' outputs and lse.

    Score error: a sum of 128 exact products in 32 bits, whatever its order and with truncation, is off by at most 128 * 2^-23
    times the sum of the magnitudes; the zero's part and the scaling add four roundings.  With scores off by at most d, weights
    are off by a factor of at most 1 + 2 d, as is their sum, so the output by 4 d * max|v|; the weights' two fp16 parts, the
    exponential (2 ulp) and the sums of up to L terms in 32 bits add (2^-21 + 2^-21 + L * 2^-23 / 16) * max|v|, as the tensor
    core adds 16 terms at a time.  lse: d and the logarithm's rounding.  fp16_rows: values and weights are rounded to fp16 on the
    way, 2^-11 each."""
    tokens, heads, _ = q.shape
    group = heads // pool.kv
    out, lse = np.zeros((tokens, heads, 128)), np.full((tokens, heads), -np.inf)
    eout, else_ = np.zeros((tokens, heads, 1)), np.zeros((tokens, heads))
    for b, first, L, n in spans(lens, new):
        top = min(L, table.shape[1] * pool.ps)
        for h in range(pool.kv):
            k, there = pool.rows(table[b], h, top, 0)
            v, _ = pool.rows(table[b], h, top, 1)
            step = 2.0 ** -11 if fp16_rows else 0.0
            for i in range(n):
                see = there & (np.arange(top) <= L - n + i)
                if not see.any():
                    continue
                kk, vv = k[see], v[see]
                for g in range(group):
                    x = q[first + i, h * group + g].astype(np.float64)
                    s = kk @ x * scale
                    m = s.max()
                    p = np.exp(s - m)
                    out[first + i, h * group + g] = p @ vv / p.sum()
                    lse[first + i, h * group + g] = m + np.log(p.sum())
                    size = (np.abs(kk) @ np.abs(x) + 2 * np.abs(kk).max(1) * np.abs(x).sum()).max() * scale
                    d = (128 * 2.0 ** -23 + 4 * 2.0 ** -24) * size + 2.0 ** -22 * max(1, np.abs(s).max())
                    eout[first + i, h * group + g] = (4 * d + 2 * step + 2.0 ** -20 + see.sum() * 2.0 ** -27) * np.abs(vv).max() * 3
                    else_[first + i, h * group + g] = 2 * d + 2.0 ** -21 + 2.0 ** -22 * abs(lse[first + i, h * group + g])
    return out, lse, eout, else_


def key_weights(pool, table, lens, new, q, lse, scale):
    """What the batch adds to every position: [pages, kv, page_size], and how far 32 bits may be off, relative to the sum."""
    add, rel = np.zeros_like(pool.weight, dtype=np.float64), 0.0
    group = q.shape[1] // pool.kv
    for b, first, L, n in spans(lens, new):
        top = min(L, table.shape[1] * pool.ps)
        for h in range(pool.kv):
            k, there = pool.rows(table[b], h, top, 0)
            for i in range(n):
                see = np.flatnonzero(there & (np.arange(top) <= L - n + i))
                for g in range(group):
                    x = q[first + i, h * group + g].astype(np.float64)
                    s = k[see] @ x * scale
                    for j, p in zip(see, np.exp(s - lse[first + i, h * group + g])):
                        add[table[b, j // pool.ps], h, j % pool.ps] += p
                    if len(see):
                        size = (np.abs(k[see]) @ np.abs(x) + 2 * np.abs(k[see]).max(1) * np.abs(x).sum()).max() * scale
                        rel = max(rel, (128 * 2.0 ** -23 + 4 * 2.0 ** -24) * size + 2.0 ** -21 * max(1, np.abs(s).max(), abs(lse[first + i, h * group + g])))
    return add, 2 * rel + n_terms(new, group) * 2.0 ** -23


def n_terms(new, group):
    return max(new) * group


def evict(weight, table, L, head, ps, num_pages, budget, sink, recent):
    """Old positions that one sequence and head keeps, in order."""
    if L <= budget:
        return list(range(L))
    middle = []
    for j in range(sink, L - recent):
        page = int(table[j // ps])
        w = float(weight[page, head, j % ps]) if 0 <= page < num_pages else float("nan")
        middle.append((-w if w == w else float("inf"), w != w, j))
    middle.sort()
    best = [j for *_, j in middle[:budget - sink - recent]]
    return sorted([*range(sink), *best, *range(L - recent, L)])
