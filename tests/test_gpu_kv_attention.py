"""aih_kv_attention against the plain implementation (kv_ref.py, 64 bits).

Two bars.  Every row and head stays within the worst case of its own
arithmetic (kv_ref.attention's `bound`).  The 2-norm over all rows is within
BAR: rounding errors of random sign add like the root of their number, so that
a score of 2 D <= 512 products with partial sums of a few units (unit normal
rows, scale 1 / sqrt(D): |partial sum| <= 8, half a step 2^-22) is off by about
sqrt(512 / 3) 2^-22 = 3e-6 at the very most and 5e-7 typically, and a weighted mean of
values by that share of the values' spread: 4e-6 with the weights' 2^-21.
Capped scores start from queries four times as large (four times the bar).
"""
import ctypes

import numpy as np
import pytest

import kv_ref as R
from aihost_amd import _native as nat
from gpu_util import upload

pytestmark = pytest.mark.gpu

I32 = np.int32
BAR = 4e-6


class Batch:
    """A full random cache, tables over it and queries, on the device."""

    def __init__(self, device, fmt, heads, kv, dim, block, lens, new, width=None, pad=0, behind=0, seed=0, spread=4.0,
                 q_size=1.0):
        rng = self.rng = np.random.default_rng(seed + dim + block + len(lens))
        self.dev, self.heads, self.dim, self.pad = device, heads, dim, pad
        need = [-(-l // block) for l in lens]
        self.width = width or max(1, max(need))
        self.ref = R.Cache(fmt, kv, dim, block, max(1, sum(need)) + 2)
        self.ref.fill_random(rng, spread)
        ids = rng.permutation(self.ref.n_blocks)
        self.tables, at = np.full((len(lens), self.width), -1), 0
        for s, b in enumerate(need):
            self.tables[s, :b] = ids[at:at + b]
            at += b
        self.lens = list(lens)
        self.starts = np.concatenate([[0], np.cumsum(new)])
        self.rows = int(self.starts[-1]) + behind
        self.q = (q_size * rng.standard_normal((self.rows, heads, dim))).astype(np.float32)
        self.scale = float(np.float32(1 / np.sqrt(dim)))

    def run(self, cap=0.0, window=0, slopes=None, prefix=None, times=1):
        L, h = nat.lib(), self.dev.handle
        k, v = self.ref.packed()
        bufs = [upload(self.dev, k), upload(self.dev, v)] + [upload(self.dev, s.astype(np.float32)) for s in self.ref.scales]
        c = nat.KvCache(format=self.ref.fmt, n_kv_heads=self.ref.heads, head_dim=self.dim, block_tokens=self.ref.block,
                        n_blocks=self.ref.n_blocks, k=bufs[0].get_pointer(), v=bufs[1].get_pointer(),
                        k_scale=bufs[2].get_pointer(), v_scale=bufs[3].get_pointer())
        wide = self.heads * self.dim
        ld = wide + self.pad
        q = np.full((self.rows, ld), np.nan, np.float32)
        q[:, :wide] = self.q.reshape(self.rows, wide)
        o = np.full((self.rows, ld), -7, np.float32)
        up = [upload(self.dev, x) for x in (q, o, self.starts.astype(I32), np.asarray(self.lens, I32),
                                            self.tables.astype(I32))]
        opt = [upload(self.dev, np.asarray(slopes, np.float32)) if slopes is not None else None,
               upload(self.dev, np.asarray(prefix, I32)) if prefix is not None else None]
        sc = nat.KvScores(cap=cap, window=window, slopes=opt[0] and opt[0].get_pointer(),
                          prefix=opt[1] and opt[1].get_pointer())
        floats = nat.check_size(L.aih_kv_attention_scratch_floats(h, ctypes.byref(c), self.heads, self.rows,
                                                                  len(self.lens), self.width), "scratch")
        sb = self.dev.create_buffer(max(16, 4 * floats))
        sb.write(np.full(max(4, floats), np.nan, np.float32))     # nothing in it has to be set
        for _ in range(times):
            nat.check(L.aih_kv_attention(h, ctypes.byref(c), up[0].get_pointer(), ld, up[1].get_pointer(), ld, self.rows,
                                         self.heads, len(self.lens), up[2].get_pointer(), up[3].get_pointer(),
                                         up[4].get_pointer(), self.width, self.scale, ctypes.byref(sc),
                                         sb.get_pointer(), floats), "aih_kv_attention")
        self.dev.synchronize()
        got = up[1].read_range(0, self.rows * ld, np.float32).reshape(self.rows, ld)
        for b in bufs + up + [sb] + [x for x in opt if x]:
            b.dispose()
        assert np.all(got[:, wide:] == -7)
        return got[:, :wide].reshape(self.rows, self.heads, self.dim)

    def tile_rows(self):
        """Rows per tile of the kernel that a call takes (aih_kv_attention_tile_rows)."""
        c = nat.KvCache(format=self.ref.fmt, n_kv_heads=self.ref.heads, head_dim=self.dim, block_tokens=self.ref.block,
                        n_blocks=self.ref.n_blocks)
        return nat.lib().aih_kv_attention_tile_rows(self.dev.handle, ctypes.byref(c), self.heads, self.rows,
                                                    len(self.lens), self.width)

    def check(self, bar=BAR, **kw):
        got = self.run(**kw)
        want, bound = R.attention(self.ref, self.q, self.starts, self.lens, self.tables, self.scale, **kw)
        n = int(self.starts[-1])
        assert np.all(got[n:] == -7)            # rows behind the last request stay as they were
        got, want, bound = got[:n], want[:n], bound[:n]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        ok = ~np.isnan(want)
        err = np.where(ok, np.abs(got - want), 0).max(-1)
        assert np.all((err <= bound) | ~ok.all(-1)), "row, head %s: %.3g over %.3g" % (
            np.unravel_index(np.argmax(err - bound), err.shape), err.max(), bound.max())
        nrm = np.linalg.norm((got - want)[ok]) / max(np.linalg.norm(want[ok]), 1e-30)
        assert nrm <= bar, nrm
        return got


FORMATS = [R.INT8, R.E4M3]


def within(got, want, bound):
    return bool(np.all(np.abs(got - want).max(-1) <= bound))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,block", [(8, 2, 16), (3, 3, 32), (5, 1, 64), (20, 1, 16), (6, 2, 256)])
def test_single_tokens(device, fmt, dim, heads, kv, block):
    """One token each, lengths from one to several parts, an empty request and padding between them."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 255, 257, 700, 1030]
    new = [1, 1, 1, 1, 1, 1, 1, 1, 0, 1, 1, 1, 1]
    Batch(device, fmt, heads, kv, dim, block, lens, new, pad=4, behind=3).check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,block,lens,new", [
    (32, 8, 128, 16, [513], [1]), (32, 8, 128, 32, [5000], [1]), (8, 8, 64, 16, [2100, 33], [1, 1]),
    (16, 8, 256, 64, [1500], [1]), (4, 4, 128, 16, [4096, 64, 1], [1, 1, 1])])
def test_long_single_tokens(device, fmt, heads, kv, dim, block, lens, new):
    Batch(device, fmt, heads, kv, dim, block, lens, new).check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,block,lens,new", [
    (8, 2, 128, 16, [4, 20, 300], [4, 4, 4]), (4, 4, 64, 32, [7, 130, 1025], [7, 2, 5]),
    (10, 2, 128, 16, [40, 90], [3, 12]), (2, 1, 256, 16, [33, 90], [9, 1])])
def test_a_few_tokens(device, fmt, heads, kv, dim, block, lens, new):
    Batch(device, fmt, heads, kv, dim, block, lens, new).check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,block,lens,new", [
    (8, 2, 128, 16, [200], [200]), (4, 1, 128, 32, [1, 33, 65, 190, 0, 300], [1, 33, 65, 190, 0, 130]),
    (3, 3, 64, 16, [257, 129], [257, 100]), (5, 1, 64, 64, [140], [140]), (4, 2, 256, 16, [150, 70], [150, 20]),
    (8, 8, 128, 16, [130], [130]), (4, 1, 128, 64, [2500], [70]), (32, 1, 64, 16, [60], [60])])
def test_prompts(device, fmt, heads, kv, dim, block, lens, new):
    Batch(device, fmt, heads, kv, dim, block, lens, new, pad=8, behind=2).check()


@pytest.mark.parametrize("fmt,heads,kv,dim,lens,new,scores", [
    (R.INT8, 32, 8, 128, [1500, 900], [1500, 900], dict()), (R.E4M3, 24, 8, 64, [2100, 40], [2000, 40], dict()),
    (R.E4M3, 48, 8, 128, [1700], [1600], dict(cap=20.0, prefix=[500], window=1000)),
    (R.INT8, 8, 1, 64, [9000], [1500], dict(slopes=[0.01] * 8))])
def test_large_prompts(device, fmt, heads, kv, dim, lens, new, scores):
    """Enough work for tiles of 128 rows.  The oracle takes every 37th row."""
    b = Batch(device, fmt, heads, kv, dim, 32, lens, new, q_size=4.0 if "cap" in scores else 1.0)
    assert b.tile_rows() == 128
    got = b.run(**scores)
    rows = np.arange(0, int(b.starts[-1]), 37)
    want, bound = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale, rows=rows, **scores)
    assert within(got[rows], want[rows], bound[rows])
    nrm = np.linalg.norm(got[rows] - want[rows]) / np.linalg.norm(want[rows])
    assert nrm <= (4 * BAR if "cap" in scores else BAR), nrm


SCORES = [dict(cap=30.0), dict(cap=2.0), dict(window=1), dict(window=17), dict(window=64, cap=50.0), dict(slopes=True),
          dict(slopes=True, cap=20.0, window=90), dict(prefix=[0, 20, 150]), dict(prefix=[300, 500, 5], window=40),
          dict(prefix=[64, 1, 33], slopes=True, cap=10.0)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 3, 30], [200, 25, 160]])
@pytest.mark.parametrize("scores", SCORES, ids=[str(i) for i in range(len(SCORES))])
def test_scores(device, fmt, dim, new, scores):
    scores = dict(scores)
    if scores.get("slopes"):
        scores["slopes"] = [2.0 ** -(1 + h) for h in range(4)]
    cap = "cap" in scores
    Batch(device, fmt, 4, 2, dim, 16, [300, 25, 160], new, q_size=4.0 if cap else 1.0).check(
        bar=4 * BAR if cap else BAR, **scores)


@pytest.mark.parametrize("new", [[1, 1], [6, 2], [100, 90]])
@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_outside_the_cache(device, fmt, new):
    """A table entry outside the pool hides its tokens; a row that sees none gives zeros."""
    b = Batch(device, fmt, 4, 2, 128, 16, [330, 100], new)
    b.tables[0, [0, 3, 20]] = [-1, b.ref.n_blocks, 2 ** 31 - 1]
    b.tables[1, :] = -2 ** 31
    got = b.check()
    assert np.all(got[b.starts[1]:b.starts[2]] == 0)


@pytest.mark.parametrize("new", [[1, 1], [6, 2], [100, 90]])
@pytest.mark.parametrize("fmt", FORMATS)
def test_lengths_that_do_not_fit(device, fmt, new):
    """More rows than tokens (rows before the first token see nothing), a negative length, a length past the table."""
    b = Batch(device, fmt, 4, 2, 128, 16, [200, 96], new)
    b.lens[0] = 0 if new[0] == 1 else new[0] - 3
    want_zero = 1 if new[0] == 1 else 3
    if new[0] == 1:
        b.lens[0] = -5
    got = b.run()
    assert np.all(got[:want_zero] == 0)
    b.lens[0] = max(b.lens[0], 0)
    want, bound = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale)
    assert within(got, want, bound)
    b.lens = [200, 10 ** 9]
    got = b.run()
    b.lens = [200, b.width * 16]
    want, bound = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale)
    assert within(got, want, bound)


@pytest.mark.parametrize("new", [[1, 1], [6, 2], [100, 90]])
@pytest.mark.parametrize("fmt", FORMATS)
def test_what_hidden_tokens_hold_has_no_effect(device, fmt, new):
    """Past the length, before the window, in another request's rows: NaN scales and values of 1e30."""
    b = Batch(device, fmt, 4, 2, 128, 16, [200, 100], new)
    plain = b.run(window=50)
    seen = set()
    for s in (0, 1):
        low = max(0, b.lens[s] - new[s] - 49)
        seen |= {int(b.tables[s, x // 16]) for x in range(low, b.lens[s])}
    hidden = [x for x in range(b.ref.n_blocks) if x not in seen]
    assert len(hidden) > 2
    before_all = b.ref.scales.copy()
    b.ref.scales[:, hidden[::2]] = np.nan
    b.ref.scales[:, hidden[1::2]] = 1e30
    np.testing.assert_array_equal(b.run(window=50), plain)
    b.ref.scales = before_all
    # a later token's block: rows before it are as exact as without it
    n = new[0]
    if n >= 100:
        for bad in (np.nan, 1e30, 1e-30):
            last = int(b.tables[0, 199 // 16])
            b.ref.scales[:, last] = bad
            got, (want, bound) = b.run(), R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale)
            before = 192 - (200 - n)
            fine = np.abs(got - want)[:before].max(-1) <= bound[:before]
            assert fine.all(), (bad, fine.sum())
            assert np.isnan(got[before:n]).all() == np.isnan(bad)


@pytest.mark.parametrize("new", [[1], [5], [120]])
@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_far_apart(device, fmt, new):
    """Blocks of zeros (no scale), value scales from 2^-120 to 2^100, key scales from tiny to large."""
    b = Batch(device, fmt, 4, 2, 128, 16, [400], new)
    t = b.tables[0]
    for values in ([0.0] * 5, [2.0 ** -120, 1.0, 0.0, 2.0 ** -60, 2.0 ** -10], [2.0 ** 100, 1.0, 0.0, 2.0 ** 60, 2.0 ** -20]):
        for i, f in enumerate(values):
            b.ref.scales[1, t[i::5]] = np.float32(f)
            if f == 0:
                b.ref.codes[1, t[i::5]] = 0
        b.ref.scales[0, t[3]] = 0
        b.ref.codes[0, t[3]] = 0
        got = b.run()
        want, bound = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale)
        assert within(got, want, bound)
    b.ref.scales[1, t[:25]] = np.float32(2.0 ** -126)     # all of them at the floor
    b.ref.codes[1, t[:25]] = b.ref.codes[1, t[1]]
    got = b.run()
    want, bound = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale)
    # values of 2^-119: an output is a multiple of 2^-149
    assert within(got, want, bound + 2.0 ** -148)


@pytest.mark.parametrize("new", [[1, 1], [4, 3], [64, 70]])
def test_queries_that_are_not_finite(device, new):
    """A query with NaN or an infinity makes its own row NaN and no other."""
    b = Batch(device, R.INT8, 4, 2, 64, 16, [90, 100], new)
    plain = b.run()
    b.q[0, 1, 5], b.q[b.starts[1], 2, 63] = np.nan, np.inf
    got = b.run()
    bad = np.zeros(got.shape[:2], bool)
    bad[0, 1] = bad[b.starts[1], 2] = True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], plain[~bad])
    b.q[0, 1] = 0                                      # a zero query weighs all alike
    b.q[b.starts[1], 2] = 1e30 * np.sign(b.q[b.starts[1], 2])      # a huge one picks one key
    b.q[b.starts[1], 2, 63] = 1e30
    got = b.run()
    assert np.isfinite(got).all()


def test_same_twice_and_over_many_requests(device):
    """The same bits again; 900 requests of one token (several scan steps of 64)."""
    lens = [1 + (7 * s) % 150 for s in range(900)]
    b = Batch(device, R.INT8, 4, 2, 64, 16, lens, [1] * 900)
    one = b.check()
    np.testing.assert_array_equal(b.run(times=3), one)


def test_shape_of_the_batch_does_not_change_a_short_row(device):
    """Requests that are not split give the same bits alone and in a batch."""
    b = Batch(device, R.E4M3, 8, 2, 128, 16, [100, 250, 3], [1, 1, 1])
    both = b.run()
    for s in range(3):
        one = Batch.__new__(Batch)
        one.__dict__.update(b.__dict__)
        one.lens, one.tables, one.starts, one.rows, one.q = [b.lens[s]], b.tables[s:s + 1], np.array([0, 1]), 1, b.q[s:s + 1]
        np.testing.assert_array_equal(one.run()[0], both[s])


@pytest.mark.parametrize("new", [[1, 1], [6, 2], [100, 70]])
@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_that_were_never_started(device, fmt, new):
    """The pool as it comes: every block that no request holds full of bytes that are no number (0x7F, 0xFF), its scales
    NaN.  The last tiles of these requests end inside such ground."""
    b = Batch(device, fmt, 4, 2, 128, 16, [210, 75], new)
    held = set(b.tables[b.tables >= 0].tolist())
    assert len(held) < b.ref.n_blocks
    # block 0, which hidden keys would be read from, is one that nobody holds
    if 0 in held:
        spare = next(x for x in range(b.ref.n_blocks) if x not in held)
        b.ref.codes[:, [0, spare]] = b.ref.codes[:, [spare, 0]]
        b.ref.scales[:, [0, spare]] = b.ref.scales[:, [spare, 0]]
        b.tables[b.tables == 0] = spare
        held = set(b.tables[b.tables >= 0].tolist())
    plain = b.run()
    empty = [x for x in range(b.ref.n_blocks) if x not in held]
    b.ref.scales[:, empty] = np.nan
    packed = b.ref.packed()
    for a, byte in zip(packed, (0x7F, 0xFF)):
        a.reshape(b.ref.n_blocks, -1)[empty] = byte
    b.ref.packed = lambda: packed
    np.testing.assert_array_equal(b.run(), plain)


@pytest.mark.parametrize("fmt,n,rows", [(R.INT8, 4096, 16), (R.E4M3, 4095, 16), (R.INT8, 65, 16), (R.E4M3, 256, 16), (R.INT8, 257, 16),
                                        (R.INT8, 300, 64), (R.E4M3, 190, 64)])
def test_many_requests(device, fmt, n, rows):
    """As many requests as a call takes, most of a few tokens, some without rows, the first, one inside and the last long
    enough to be split; prompts of a few rows beside them."""
    lens = [1 + (5 * s) % 23 for s in range(n)]
    new = [0 if s % 9 == 4 else 1 if rows == 16 or s % 2 else min(lens[s], 20) for s in range(n)]
    for s, (length, k) in {0: (2100, 1), n // 2: (3000, 2), n - 1: (1500, 3)}.items():
        lens[s], new[s] = length, k
    b = Batch(device, fmt, 4, 1, 64, 32, lens, new, behind=1, seed=n)
    b.check()


def test_many_requests_in_parts_and_prompts(device):
    """More requests than the lanes of a wave: one of them long, so that it is split; prompts in tiles of 64 rows."""
    lens = [5000 if s == 66 else 40 + s for s in range(80)]
    b = Batch(device, R.INT8, 4, 1, 64, 32, lens, [1] * 80, seed=1)
    assert b.tile_rows() == 16
    b.check()
    lens = [30 + s % 50 for s in range(130)]
    b = Batch(device, R.E4M3, 8, 2, 64, 16, lens, lens, seed=2)
    assert b.tile_rows() == 64
    b.check()


@pytest.mark.parametrize("new", [[1, 3], [50, 70]])
def test_extreme_arguments(device, new):
    """A window as large as an int, prefixes outside the request, more rows than tokens beside a prefix."""
    b = Batch(device, R.INT8, 4, 2, 64, 16, [200, 100], new)
    plain = b.run()
    np.testing.assert_array_equal(b.run(window=2 ** 31 - 1, prefix=[-2 ** 31, -5]), plain)
    b.check(window=2 ** 31 - 1, prefix=[2 ** 31 - 1, 2 ** 31 - 1])
    b.lens[1] = new[1] - 2          # its first two rows lie before the first token; they see the prefix
    b.check(window=2 ** 31 - 1, prefix=[0, 1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,lens,new", [
    (600, 600, 64, [70, 1, 1100], [1, 1, 1]), (71, 1, 64, [300, 20], [1, 3]), (130, 1, 128, [90], [40]),
    (258, 86, 64, [1100], [2]), (300, 100, 64, [80], [80]), (7, 7, 256, [1040], [30])])
def test_odd_and_many_heads(device, fmt, heads, kv, dim, lens, new):
    """More KV heads than workgroups that a call aims at, groups of more rows than a tile has, primes."""
    Batch(device, fmt, heads, kv, dim, 16, lens, new, pad=4).check()


def test_starts_that_overlap(device):
    """Rows claimed by several requests: nothing outside O and the scratch is touched, and the other rows are right."""
    b = Batch(device, R.INT8, 4, 2, 64, 16, [3000, 500], [64, 64], behind=64)
    b.lens, b.tables = b.lens * 40, np.tile(b.tables, (40, 1))
    good = b.starts.copy()
    b.starts = np.array([0, 64, 0] * 26 + [0, 0, -5])
    got = b.run()
    assert got.shape == (192, 4, 64)
    assert np.all(got[128:] == -7) or np.isfinite(got).all()
    b.starts = good


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,lens,new,tile,zeros", [
    (4, 2, 128, [400], [1], 16, 64), (4, 2, 256, [400], [5], 16, 128), (4, 2, 64, [1500], [1], 16, 512),
    (16, 8, 64, [700], [700], 64, 128), (8, 1, 64, [4000], [1500], 64, 2600), (8, 1, 64, [9000], [1500], 128, 8000)])
def test_small_values_after_zeros(device, fmt, heads, kv, dim, lens, new, tile, zeros):
    """Whole key tiles, and a whole part, of blocks without a value scale before values of any size."""
    b = Batch(device, fmt, heads, kv, dim, 32, lens, new)
    assert b.tile_rows() == tile
    t, scales = b.tables[0], b.ref.scales.copy()
    b.ref.scales[1, t[:zeros // 32]] = 0
    b.ref.codes[1, t[:zeros // 32]] = 0
    rows = np.arange(0, new[0], 1 if new[0] < 10 else 83)
    for f in (1.0, 1e-6, 1e-8, 1e-10, 2.0 ** -60, 2.0 ** -90):
        b.ref.scales[1, t[zeros // 32:]] = (scales[1, t[zeros // 32:]] * f).astype(np.float32)
        got = b.run()
        want, bound = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale, rows=rows)
        assert within(got[rows], want[rows], bound[rows]), f
        nrm = np.linalg.norm((got[rows] - want[rows]) / f) / np.linalg.norm(want[rows] / f)
        assert nrm <= BAR, (f, nrm)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,lens,new,tile", [
    (4, 2, 128, [400], [1], 16), (4, 2, 64, [1500], [1], 16), (16, 8, 64, [700], [700], 64),
    (8, 1, 64, [9000], [1500], 128)])
@pytest.mark.parametrize("small", [2.0 ** -50, 2.0 ** -75, 2.0 ** -100])
def test_large_values_that_hardly_count(device, fmt, heads, kv, dim, lens, new, tile, small):
    """The first tokens have values near 1 and scores 130 below the others', whose values are tiny and make the result."""
    b = Batch(device, fmt, heads, kv, dim, 32, lens, new)
    assert b.tile_rows() == tile
    t, n0 = b.tables[0], 128 // 32
    u = np.where(b.rng.random(dim) < 0.5, -1.0, 1.0)
    # every score is scale * dim * 16 * key scale * (-1 or 1)
    b.q[:] = u
    b.ref.codes[0, t] = 16 * u
    b.ref.codes[0, t[:n0]] *= -1
    b.ref.scales[0] = np.float32(65 / (16 * dim * b.scale))
    b.ref.scales[1, t[:n0]] = np.float32(1.0)
    b.ref.scales[1, t[n0:]] = (b.ref.scales[1, t[n0:]] * small).astype(np.float32)
    rows = np.arange(0, new[0], 83)
    rows = rows[rows + lens[0] - new[0] >= 128]          # those that see a token that counts
    got = b.run()[rows].astype(np.float64) / small
    want = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale, rows=rows)[0][rows] / small
    most = np.abs(b.ref.codes[1, t[n0:]] * b.ref.scales[1, t[n0:], :, None, None]).max() / small
    # the scores of the tokens that count are equal: sums of n values with 22 bits of a weight, and the weights' sum
    np.testing.assert_allclose(got, want, rtol=0, atol=most * (2.0 ** -20 + (lens[0] / 32 + 48) * 2.0 ** -23))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,lens,new,tile", [
    (4, 2, 128, [512], [1], 16), (16, 8, 64, [704], [704], 64), (8, 1, 64, [9024], [1500], 128)])
@pytest.mark.parametrize("size", [1e3, 1e6, 1.3e7, 2.4e7, 3e8, -1e3, -1e6, -1.3e7, -2.4e7, -3e8])
@pytest.mark.parametrize("biased", [False, True])
def test_scores_of_any_size(device, fmt, heads, kv, dim, lens, new, tile, size, biased):
    """Equal scores, large of either sign, weigh all tokens alike, whatever the values' scale is."""
    b = Batch(device, fmt, heads, kv, dim, 32, lens, new)
    assert b.tile_rows() == tile
    u = np.where(b.rng.random(dim) < 0.5, -1.0, 1.0)
    b.q[:] = np.sign(size) * u
    b.ref.codes[0] = 13 * u
    b.ref.scales[0] = np.float32(abs(size) / (13 * dim * b.scale))
    rows = np.arange(0, new[0], 83)
    most = np.abs(b.ref.codes[1]).max()
    # Every chained sum rounds, relative to the largest value.  Up to 2^20 in base 2 a score is rounded (half a step, to
    # either side) in tiles of which a row sees a part, and not in others.
    t = abs(size) / np.log(2)
    bar = most * (2.0 ** -20 + (lens[0] / 32 + 48) * 2.0 ** -23 + (t * 2.0 ** -23 if t < 2.0 ** 20 else 0))
    want = None
    for e in range(4):
        b.ref.scales[1] = np.float32(0.75 * 2.0 ** -e)     # one for all: see the comment on scores beyond 2^20
        if want is None:
            want = R.attention(b.ref, b.q, b.starts, b.lens, b.tables, b.scale, rows=rows)[0][rows] / 0.75
        got = b.run(slopes=[0.0] * heads if biased else None)[rows] / (0.75 * 2.0 ** -e)
        np.testing.assert_allclose(got, want, rtol=0, atol=bar)


@pytest.mark.parametrize("new", [[1], [30], [200]])
@pytest.mark.parametrize("cap", [3.4028234663852886e38, 1e35, 1e30, 1e-30, 2.0 ** -126, 1e-44])
def test_caps_of_any_size(device, cap, new):
    """A cap that no score comes near changes nothing; one below all of them leaves weights that are alike."""
    b = Batch(device, R.INT8, 4, 2, 128, 16, [300], new)
    b.ref.codes[0, b.tables[0, 2]] = 0          # scores of 0 among them
    b.check(cap=cap)


@pytest.mark.parametrize("tokens,fmt", [(2200000, R.INT8), (2111111, R.E4M3)])
def test_more_work_than_fp32_counts(device, tokens, fmt):
    """Row tiles times key tiles beyond 2^24, where the sums that split the work are rounded: the join takes the parts that
    were written.  The table names a few blocks again and again."""
    heads, dim, block, blocks, n = 8, 64, 32, 40, 8192
    b = Batch(device, fmt, heads, 1, dim, block, [block * (blocks - 2)], [n], width=-(-tokens // block))
    b.tables = b.rng.integers(0, blocks, (1, b.width))
    b.lens = [tokens]
    assert b.tile_rows() == 128 and -(-n * heads // 128) * -(-tokens // 64) > 2 ** 24
    got = b.run()
    keys, vals = (x[:, 0] for x in b.ref.values())
    slots = (b.tables[0][:, None] * block + np.arange(block)).reshape(-1)
    for r in (0, 4097, n - 1):
        seen = np.bincount(slots[:tokens - n + r + 1], minlength=len(keys))
        t = b.q[r].astype(np.float64) @ keys.T * b.scale                     # (head, slot)
        w = np.exp(t - t.max(1, keepdims=True)) * seen
        want = w @ vals / w.sum(1, keepdims=True)
        # the sums are chains of an add for 32 keys; all else is far below that
        np.testing.assert_allclose(got[r], want, rtol=0, atol=np.abs(vals).max() * (tokens / 32) * 2.0 ** -23)


def test_starts_that_overlap_stay_inside(device):
    """A request with rows of its own before many that claim the same rows again and again: its rows are right, the rows of
    no request stay, and nothing beside O and the scratch is written."""
    lens, new = [3000, 500], [64, 64]
    b = Batch(device, R.INT8, 4, 2, 64, 16, lens, new, behind=64)
    b.lens, b.tables = lens * 41, np.tile(b.tables, (41, 1))
    n = len(b.lens)
    starts = np.array([128, 192] + [0, 64] * 40 + [0])[:n + 1]
    L, h, guard = nat.lib(), device.handle, 64
    k, v = b.ref.packed()
    bufs = [upload(device, x) for x in (k, v, b.ref.scales[0].astype(np.float32), b.ref.scales[1].astype(np.float32))]
    c = nat.KvCache(format=b.ref.fmt, n_kv_heads=2, head_dim=64, block_tokens=16, n_blocks=b.ref.n_blocks,
                    k=bufs[0].get_pointer(), v=bufs[1].get_pointer(), k_scale=bufs[2].get_pointer(),
                    v_scale=bufs[3].get_pointer())
    wide, rows = 4 * 64, b.rows
    floats = nat.check_size(L.aih_kv_attention_scratch_floats(h, ctypes.byref(c), 4, rows, n, b.width), "scratch")
    assert floats > 0
    up = [upload(device, x) for x in (b.q, np.full(rows * wide + 2 * guard, -7, np.float32),
                                      np.full(floats + 2 * guard, -9, np.float32), starts.astype(I32),
                                      np.asarray(b.lens, I32), b.tables.astype(I32))]
    nat.check(L.aih_kv_attention(h, ctypes.byref(c), up[0].get_pointer(), wide, up[1].get_pointer() + 4 * guard, wide, rows, 4, n,
                                 up[3].get_pointer(), up[4].get_pointer(), up[5].get_pointer(), b.width, b.scale, None,
                                 up[2].get_pointer() + 4 * guard, floats), "aih_kv_attention")
    device.synchronize()
    o = up[1].read_range(0, rows * wide + 2 * guard, np.float32)
    scratch = up[2].read_range(0, floats + 2 * guard, np.float32)
    for x in bufs + up:
        x.dispose()
    for x, value in ((o, -7), (scratch, -9)):
        assert np.all(x[:guard] == value) and np.all(x[-guard:] == value)
    got = o[guard:-guard].reshape(rows, 4, 64)
    assert np.all(got[64:128] == -7)                       # no request has them
    assert np.isfinite(got).all()
    want, bound = R.attention(b.ref, b.q, [128, 192], b.lens[:1], b.tables[:1], b.scale)
    assert within(got[128:192], want[128:192], bound[128:192])


@pytest.mark.parametrize("window", [0, 2 ** 30 + 77, 5])
def test_as_many_tokens_as_a_length_counts(device, window):
    """A request of nearly 2^31 tokens; its table names three blocks, one for each part of it, whose values differ."""
    b = Batch(device, R.E4M3, 2, 1, 64, 256, [100], [1], width=2 ** 23 - 1)
    tokens = b.lens[0] = (2 ** 23 - 1) * 256 - 3
    b.tables = np.zeros((1, b.width), np.int32)
    b.tables[0, 2 ** 22:] = 1
    b.tables[0, -1] = 2
    values = (-1.0, 1.0, 3.0)
    for i, v in enumerate(values):
        b.ref.codes[1, i], b.ref.scales[1, i] = v, 1.0
    b.q[:] = 0                                         # all tokens weigh alike
    low = max(0, tokens - window) if window else 0
    ends = np.clip([2 ** 30, tokens // 256 * 256, tokens], low, None)
    counts = np.diff(np.concatenate([[low], ends]))
    want = (counts * values).sum() / counts.sum()
    # 2048 waves take 16384 tiles each, an add for each of four products to a tile
    np.testing.assert_allclose(b.run(window=window), want, rtol=0, atol=3 * 5 * 16384 * 2.0 ** -24)


@pytest.mark.parametrize("seed", range(48))
def test_mixed_batches_over_wide_tables(device, seed):
    """What a server sends: requests that wait, single tokens, drafts and prompts in one call, over tables of a fixed
    capacity (which the tile is chosen by), with any scores."""
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *a: a[rng.integers(len(a))]
    fmt, dim, block, kv = pick(*FORMATS), pick(64, 128, 128, 256), pick(16, 32, 64, 256), pick(1, 2, 3)
    heads = kv * pick(1, 2, 4, 5)
    lens, new = [], []
    for _ in range(rng.integers(1, 10)):
        n = int(pick(0, 1, 1, rng.integers(2, 9), rng.integers(9, 150)))
        lens.append(n + int(pick(0, rng.integers(0, 40), rng.integers(0, 600))))
        new.append(n)
    if seed % 4 == 0:
        lens.append(int(rng.integers(1100, 2000)))
        new.append(1)
    scores = {}
    if rng.random() < 0.3:
        scores["cap"] = float(pick(2.0, 30.0))
    if rng.random() < 0.3:
        scores["window"] = int(rng.integers(1, 300))
    if rng.random() < 0.3:
        scores["slopes"] = [2.0 ** -(1 + h) for h in range(heads)]
    if rng.random() < 0.3:
        scores["prefix"] = [int(rng.integers(0, l + 5)) for l in lens]
    need = max(1, max(-(-l // block) for l in lens))
    cap = "cap" in scores
    b = Batch(device, fmt, heads, kv, dim, block, lens, new, width=need + int(pick(0, 3, 8192 // block, 65536 // block)),
              pad=int(pick(0, 4)), behind=int(pick(0, 1, 200)) + (sum(new) == 0), seed=seed, q_size=4.0 if cap else 1.0)
    b.check(bar=4 * BAR if cap else BAR, **scores)
