"""The paged 8-bit KV cache (include/aihost_hip.h) in plain numpy, 64 bits:
bookkeeping request by request, blocks as lists of tokens, attention row by
row.  Nothing here is shared with the library."""
import math

import numpy as np
import torch

INT8, E4M3 = 0, 1
MOST = {INT8: 127.0, E4M3: 448.0}


# ---- bookkeeping ---------------------------------------------------------------
def plan(lens, n_new, tables, block, n_blocks, free, n_free, rows):
    """aih_kv_plan as a loop over the requests; tables is changed in place."""
    width = tables.shape[1]
    starts, new_lens, slots, positions, refused = [0], [], [], [], 0
    wanted = asked = taken = 0
    for s, (l, n) in enumerate(zip(map(int, lens), map(int, n_new))):
        ok = l >= 0 and n >= 0 and l + n <= width * block
        if ok:
            had, need = -(-l // block), -(-(l + n) // block) - -(-l // block)
            wanted += need
            asked += n
            ok = n == 0 or ((need == 0 or wanted <= n_free) and asked <= rows)
        if not ok:
            refused += 1
            n = 0
        else:
            for j in range(need):
                tables[s, had + j] = free[n_free - 1 - taken - j]
            taken += need
        for p in range(l, l + n):
            b = int(tables[s, p // block])
            slots.append(b * block + p % block if 0 <= b < n_blocks else -1)
            positions.append(p)
        starts.append(starts[-1] + n)
        new_lens.append(l + n)
    pad = [-1] * (rows - len(slots))
    return dict(starts=starts, new_lens=new_lens, slots=slots + pad, positions=positions + pad,
                n_free=n_free - taken, refused=refused)


# ---- the formats -----------------------------------------------------------------
def to_code(x, fmt):
    """Numbers (64 bits, within the range) to codes as numbers, ties to even."""
    if fmt == INT8:
        return np.clip(np.rint(x), -127, 127)
    # 448 / 2^-9 and below: fp32 holds x / scale of fp32 values over a power of two exactly
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
    return t.to(torch.float8_e4m3fn).to(torch.float64).numpy()


def first_scale(top, fmt):
    if top == 0:
        return 0.0
    if fmt == INT8:
        return max(float(np.float32(np.float64(top) / 127)), 2.0 ** -126)
    k = -126
    while 448.0 * 2.0 ** k < top:
        k += 1
    return 2.0 ** k


class Cache:
    """Blocks of code numbers and scales, keys and values alike: codes
    [2][block, head, token, dim], scales [2][block, head]."""

    def __init__(self, fmt, heads, dim, block, n_blocks):
        self.fmt, self.heads, self.dim, self.block, self.n_blocks = fmt, heads, dim, block, n_blocks
        self.codes = np.zeros((2, n_blocks, heads, block, dim))
        self.scales = np.zeros((2, n_blocks, heads))

    def append(self, k, v, slots):
        """k, v: (rows, heads, dim)."""
        rows = len(slots)
        valid = [0 <= s < self.n_blocks * self.block for s in slots]
        r = 0
        while r < rows:
            if not valid[r]:
                r += 1
                continue
            b, end = slots[r] // self.block, r
            while end < rows and valid[end] and slots[end] // self.block == b:
                end += 1
            at = [s % self.block for s in slots[r:end]]
            for which, x in ((0, k), (1, v)):
                for h in range(self.heads):
                    self._run(which, b, h, x[r:end, h].astype(np.float64), at)
            r = end

    def _run(self, which, b, h, x, at):
        c, fmt = self.codes[which, b, h], self.fmt
        s = self.scales[which, b, h]
        if 0 in at:
            c[:] = 0
            s = 0.0
        if not np.all(np.isfinite(x)) or math.isnan(s):
            self.scales[which, b, h] = np.nan
            c[at] = 0
            return
        top = float(np.max(np.abs(x)))
        if s == 0.0:
            s = first_scale(top, fmt)
        else:
            d = 0
            while MOST[fmt] * s * 2.0 ** d < top:
                d += 1
            if d:
                c[:] = to_code(c * 2.0 ** -d, fmt)
                s *= 2.0 ** d
        for o, row in zip(at, x):
            c[o] = to_code(row / s, fmt) if s else 0.0
        self.scales[which, b, h] = s

    def values(self):
        """(keys, values), each (slots, heads, dim)."""
        out = self.codes * self.scales[..., None, None]
        return out.transpose(0, 1, 3, 2, 4).reshape(2, -1, self.heads, self.dim)

    # -- the library's bytes
    def packed(self):
        """Key bytes and value bytes in the library's layout."""
        if self.fmt == INT8:
            c = self.codes.astype(np.int8).view(np.uint8)
        else:
            c = torch.from_numpy(self.codes.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        n, h, bt, d = c.shape[1:]
        k = c[0].reshape(n, h, bt // 16, 4, 4, d // 64, 4, 16).transpose(0, 1, 2, 3, 5, 4, 6, 7)
        v = c[1].reshape(n, h, bt // 16, 16, d).transpose(0, 1, 2, 4, 3)
        return np.ascontiguousarray(k).reshape(-1), np.ascontiguousarray(v).reshape(-1)

    def fill_random(self, rng, spread=1.0):
        """Every block full: normal values, scales a factor of `spread` apart at most."""
        x = rng.standard_normal(self.codes.shape)
        top = np.abs(x).max((3, 4))
        s = top / MOST[self.fmt]
        self.codes = to_code(x / s[..., None, None] if self.fmt == INT8 else np.clip(x / s[..., None, None], -448, 448),
                             self.fmt)
        self.scales = (s * spread ** rng.uniform(0, 1, s.shape)).astype(np.float32).astype(np.float64)


# ---- attention ---------------------------------------------------------------------
def attention(cache, q, starts, lens, tables, scale, cap=0.0, window=0, slopes=None, prefix=None,
              rows=None):
    """q: (rows, n_heads, dim); rows: the ones wanted, None for all.  Returns (o, bound): the result and, for every
    row and head, what an fp32 evaluation may be off by (see `bound` below);
    rows of no request are NaN in both."""
    n_rows, n_heads, dim = q.shape
    wanted = set(range(n_rows) if rows is None else map(int, rows))
    kv, group = cache.heads, n_heads // cache.heads
    keys, vals = cache.values()
    o = np.full((n_rows, n_heads, dim), np.nan)
    bound = np.full((n_rows, n_heads), np.nan)
    q = q.astype(np.float64)
    for s in range(len(lens)):
        n, length = starts[s + 1] - starts[s], int(lens[s])
        j = np.arange(length)
        ids = np.array([tables[s, x // cache.block] for x in j], dtype=np.int64)
        there = (ids >= 0) & (ids < cache.n_blocks)
        slot = np.where(there, ids * cache.block + j % cache.block, 0)
        for i in range(n):
            p, r = length - n + i, starts[s] + i
            if r not in wanted:
                continue
            end = p + 1 if prefix is None else max(p + 1, int(prefix[s]))
            seen = there & (j < end)
            if window:
                seen &= j > p - window
            for h in range(n_heads):
                if not seen.any():
                    o[r, h], bound[r, h] = 0.0, 0.0
                    continue
                k, v = keys[slot[seen], h // group], vals[slot[seen], h // group]
                t = k @ q[r, h] * scale
                with np.errstate(all="ignore"):
                    part = np.max(np.abs(k) @ np.abs(q[r, h])) * scale     # sum of the products' magnitudes
                if cap:
                    t = cap * np.tanh(t / cap)
                far = np.zeros(1)
                if slopes is not None:
                    far = slopes[h] * np.abs(p - j[seen])
                    t = t - far
                w = np.exp(t - t.max())
                o[r, h] = w @ v / w.sum()
                # A score: 2 dim products summed in fp32 (half a step, 2^-24, of the partial sum at each), q cut at 22
                # bits (2^-22), and 8 roundings of the score itself (scales, cap, tanh within 4 steps) and of its bias.
                # A weight: twice the score's error (its own and the sum's), exp within 2 steps, cut at 22 bits.  The sums
                # over n keys: n / 32 chained adds and 48 within a tile and over the parts, in the products and in the sum
                # of the probabilities.  Each is relative to the largest value seen.
                dt = part * (2 * dim * 2.0 ** -24 + 2.0 ** -22) + 8 * 2.0 ** -24 * (np.abs(t).max() + np.max(far))
                bound[r, h] = np.max(np.abs(v)) * (2 * dt + 2.0 ** -20 + 2 * (seen.sum() / 32 + 48) * 2.0 ** -24)
    return o, bound
