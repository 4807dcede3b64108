"""aih_kv_plan, aih_kv_release, aih_kv_append, aih_kv_append_rope and
aih_kv_read against the plain implementation (kv_ref.py): bookkeeping, codes
and scales have to be equal."""
import ctypes

import numpy as np
import pytest

import kv_ref as R
from aihost_amd import _native as nat
from gpu_util import upload

pytestmark = pytest.mark.gpu

I32 = np.int32


class Pool:
    """A cache on the device, beside its oracle."""

    def __init__(self, device, ref, init=None):
        self.dev, self.ref = device, ref
        k, v = ref.packed() if init is None else init
        self.kb, self.vb = upload(device, k), upload(device, v)
        self.ks, self.vs = (upload(device, ref.scales[i].astype(np.float32)) for i in (0, 1))
        self.c = nat.KvCache(format=ref.fmt, n_kv_heads=ref.heads, head_dim=ref.dim, block_tokens=ref.block,
                             n_blocks=ref.n_blocks, k=self.kb.get_pointer(), v=self.vb.get_pointer(),
                             k_scale=self.ks.get_pointer(), v_scale=self.vs.get_pointer())
        self.p = ctypes.byref(self.c)

    def append(self, k, v, slots, pad=0):
        """Rows with `pad` floats behind each one."""
        rows, wide = len(slots), self.ref.heads * self.ref.dim
        a = np.full((2, rows, wide + pad), np.nan, np.float32)
        a[0, :, :wide], a[1, :, :wide] = k.reshape(rows, wide), v.reshape(rows, wide)
        kb, vb, sb = upload(self.dev, a[0]), upload(self.dev, a[1]), upload(self.dev, np.asarray(slots, I32))
        nat.check(nat.lib().aih_kv_append(self.dev.handle, self.p, kb.get_pointer(), wide + pad, vb.get_pointer(),
                                          wide + pad, sb.get_pointer(), rows), "aih_kv_append")
        self.dev.synchronize()
        for b in (kb, vb, sb):
            b.dispose()

    def state(self):
        n = self.ref.codes[0].size
        m = self.ref.scales[0].size
        return (self.kb.read_range(0, n, np.uint8), self.vb.read_range(0, n, np.uint8),
                self.ks.read_range(0, m, np.float32).reshape(self.ref.scales[0].shape),
                self.vs.read_range(0, m, np.float32).reshape(self.ref.scales[0].shape))

    def check(self):
        """Codes and scales equal the oracle's (a negative zero is a zero)."""
        k, v, ks, vs = self.state()
        want = self.ref.packed()
        for which, got, w in (("keys", k, want[0]), ("values", v, want[1])):
            if self.ref.fmt == R.E4M3:
                got, w = np.where(got == 0x80, 0, got), np.where(w == 0x80, 0, w)
            bad = np.flatnonzero(got != w)
            assert bad.size == 0, "%s: %d codes differ, first at byte %d: %d for %d" % (
                which, bad.size, bad[0], got[bad[0]], w[bad[0]])
        np.testing.assert_array_equal(ks, self.ref.scales[0].astype(np.float32))
        np.testing.assert_array_equal(vs, self.ref.scales[1].astype(np.float32))

    def dispose(self):
        for b in (self.kb, self.vb, self.ks, self.vs):
            b.dispose()


@pytest.fixture
def pool(device):
    made = []

    def make(fmt, heads, dim, block, n_blocks, ref=None, init=None):
        made.append(Pool(device, ref or R.Cache(fmt, heads, dim, block, n_blocks), init))
        return made[-1]

    yield make
    for p in made:
        p.dispose()


# ---- bookkeeping ------------------------------------------------------------------
def run_plan(device, lens, n_new, tables, block, n_blocks, free, n_free, rows, in_place=False):
    S, W = tables.shape
    bufs = dict(lens=upload(device, np.asarray(lens, I32)), new=upload(device, np.asarray(n_new, I32)),
                tables=upload(device, tables.astype(I32)), free=upload(device, np.asarray(free, I32)),
                n_free=upload(device, np.array([n_free], I32)), new_lens=upload(device, np.full(S, -7, I32)),
                new_n_free=upload(device, np.array([-7], I32)), starts=upload(device, np.full(S + 1, -7, I32)),
                slots=upload(device, np.full(rows + 2, -7, I32)), positions=upload(device, np.full(rows + 2, -7, I32)),
                refused=upload(device, np.array([-7], I32)))
    p = {k: b.get_pointer() for k, b in bufs.items()}
    to_lens, to_free = (p["lens"], p["n_free"]) if in_place else (p["new_lens"], p["new_n_free"])
    nat.check(nat.lib().aih_kv_plan(device.handle, p["lens"], p["new"], S, p["tables"], W, block, n_blocks, p["free"],
                                    p["n_free"], to_lens, to_free, p["starts"], p["slots"], p["positions"], rows,
                                    p["refused"]), "aih_kv_plan")
    device.synchronize()
    src = ("lens", "n_free") if in_place else ("new_lens", "new_n_free")
    out = dict(tables=bufs["tables"].read_range(0, S * W, I32).reshape(S, W), starts=bufs["starts"].read_range(0, S + 1, I32),
               slots=bufs["slots"].read_range(0, rows + 2, I32), positions=bufs["positions"].read_range(0, rows + 2, I32),
               new_lens=bufs[src[0]].read_range(0, S, I32), n_free=int(bufs[src[1]].read_range(0, 1, I32)[0]),
               refused=int(bufs["refused"].read_range(0, 1, I32)[0]))
    for b in bufs.values():
        b.dispose()
    return out


def make_tables(rng, lens, n_new, block, spare, width=None):
    after = [max(l, 0) + max(n, 0) for l, n in zip(lens, n_new)]
    width = width or max(1, max(-(-a // block) for a in after))
    used = [-(-max(l, 0) // block) for l in lens]
    n_blocks = sum(used) + spare
    ids = rng.permutation(n_blocks)
    tables, at = np.full((len(lens), width), -1), 0
    for s, u in enumerate(used):
        tables[s, :min(u, width)] = ids[at:at + min(u, width)]
        at += u
    free = np.concatenate([ids[at:], np.full(at, -1, ids.dtype)])
    return tables, free, len(ids) - at, n_blocks


PLANS = {   # lengths, new tokens, block, blocks to spare, rows
    "one token": ([0], [1], 16, 1, 1),
    "one token inside a block": ([5], [1], 16, 0, 1),
    "one token behind a full block": ([32], [1], 16, 1, 3),
    "nothing new": ([7, 0], [0, 0], 16, 2, 4),
    "no rows": ([7, 0], [0, 0], 16, 2, 0),
    "ragged": ([0, 15, 16, 17, 100, 31], [40, 1, 1, 15, 0, 33], 16, 9, 100),
    "out of blocks": ([0, 15, 16, 17, 100, 30], [40, 1, 1, 15, 0, 2], 16, 3, 100),
    "out of rows": ([0, 15, 16, 17, 100, 31], [20, 1, 9, 15, 0, 3], 32, 9, 30),
    "bad lengths": ([-1, 15, 16, 4], [4, -2, 3, 2 ** 31 - 1], 16, 9, 40),
    "300 requests": ([(37 * s) % 200 for s in range(300)], [(s * s) % 41 for s in range(300)], 64, 400, 7000),
    "1500 requests": ([s % 50 for s in range(1500)], [1 + (s % 3 == 0) for s in range(1500)], 16, 900, 2500),
    "4096 requests": ([s % 33 for s in range(4096)], [1] * 4096, 16, 5000, 4096),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", list(PLANS))
def test_plan(device, name, in_place):
    lens, n_new, block, spare, rows = PLANS[name]
    rng = np.random.default_rng(3)
    width = 8 if name == "bad lengths" else None
    tables, free, n_free, n_blocks = make_tables(rng, lens, n_new, block, spare, width)
    want_tables = tables.copy()
    want = R.plan(lens, n_new, want_tables, block, n_blocks, free, n_free, rows)
    got = run_plan(device, lens, n_new, tables, block, n_blocks, free, n_free, rows, in_place)
    np.testing.assert_array_equal(got["starts"], want["starts"])
    np.testing.assert_array_equal(got["new_lens"], want["new_lens"])
    np.testing.assert_array_equal(got["tables"], want_tables)
    np.testing.assert_array_equal(got["slots"], want["slots"] + [-7, -7])
    np.testing.assert_array_equal(got["positions"], want["positions"] + [-7, -7])
    assert (got["n_free"], got["refused"]) == (want["n_free"], want["refused"])


def test_plan_with_bad_entries(device):
    """A table or free entry outside the pool gives slots of -1, no access outside it."""
    tables = np.array([[99, -1], [-5, 1]])
    free = np.array([2, 77, 0, 3, 1])
    want_tables = tables.copy()
    want = R.plan([10, 3], [10, 20], want_tables, 16, 4, free, 2, 40)
    got = run_plan(device, [10, 3], [10, 20], tables, 16, 4, free, 2, 40)
    np.testing.assert_array_equal(got["slots"][:40], want["slots"])
    np.testing.assert_array_equal(got["tables"], want_tables)
    assert got["slots"][6:10].tolist() == [-1] * 4      # the new block of the first request is block 77


@pytest.mark.parametrize("n_seqs", [1, 5, 70, 1100])
@pytest.mark.parametrize("some", [False, True])
def test_release(device, n_seqs, some):
    rng = np.random.default_rng(n_seqs)
    lens = rng.integers(0, 90, n_seqs)
    lens[0] = 200
    tables, free, n_free, n_blocks = make_tables(rng, lens, [0] * n_seqs, 16, 3, 14)
    done = rng.integers(0, 2, n_seqs) if some else np.ones(n_seqs, int)
    if n_seqs == 5:
        tables[0, 3] = n_blocks      # not a block: dropped
    want_free, want_tables, want_lens = list(free[:n_free]), tables.copy(), lens.copy()
    for s in range(n_seqs):
        if done[s]:
            for j in range(-(-lens[s] // 16)):
                if 0 <= tables[s, j] < n_blocks:
                    want_free.append(tables[s, j])
                want_tables[s, j] = -1
            want_lens[s] = 0
    b = [upload(device, np.asarray(x, I32)) for x in (lens, tables, done, free, [n_free])]
    nat.check(nat.lib().aih_kv_release(device.handle, b[0].get_pointer(), n_seqs, b[1].get_pointer(), 14, 16, n_blocks,
                                       b[2].get_pointer() if some else None, b[3].get_pointer(), b[4].get_pointer()),
              "aih_kv_release")
    device.synchronize()
    assert int(b[4].read_range(0, 1, I32)[0]) == len(want_free)
    np.testing.assert_array_equal(b[3].read_range(0, len(want_free), I32), want_free)
    np.testing.assert_array_equal(b[1].read_range(0, n_seqs * 14, I32).reshape(n_seqs, 14), want_tables)
    np.testing.assert_array_equal(b[0].read_range(0, n_seqs, I32), want_lens)
    # a second time there is nothing to give back
    nat.check(nat.lib().aih_kv_release(device.handle, b[0].get_pointer(), n_seqs, b[1].get_pointer(), 14, 16, n_blocks,
                                       b[2].get_pointer() if some else None, b[3].get_pointer(), b[4].get_pointer()),
              "aih_kv_release")
    device.synchronize()
    assert int(b[4].read_range(0, 1, I32)[0]) == len(want_free)
    for x in b:
        x.dispose()


# ---- append ------------------------------------------------------------------------
FORMATS = [R.INT8, R.E4M3]


def rows_of(rng, n, heads, dim, size=1.0):
    return ((rng.standard_normal((n, heads, dim)) * size).astype(np.float32),
            (rng.standard_normal((n, heads, dim)) * size).astype(np.float32))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,dim,block", [(1, 64, 16), (2, 128, 16), (3, 128, 32), (8, 128, 64), (2, 256, 16),
                                             (1, 256, 128), (1, 64, 256)])
def test_append_token_by_token(device, pool, fmt, heads, dim, block):
    """A block filled one token at a time, its scale growing on the way, then the next one; garbage before."""
    rng = np.random.default_rng(dim + block)
    ref = R.Cache(fmt, heads, dim, block, 5)
    size = ref.codes[0].size
    p = pool(fmt, heads, dim, block, 5, ref, (rng.integers(0, 256, size, np.uint8), rng.integers(0, 256, size, np.uint8)))
    p.ks.write(np.full(ref.scales[0].size, np.nan, np.float32))
    order = [3, 1]
    # the oracle's untouched blocks hold the same bytes: compared block by block below
    for i in range(block + 3):
        k, v = rows_of(rng, 1, heads, dim, 0.5 * 1.5 ** (i % 9))
        slot = order[i // block] * block + i % block
        ref.append(k, v, [slot])
        p.append(k, v, [slot])
    k, v, ks, vs = p.state()
    wk, wv = ref.packed()
    for b in order:
        at = slice(b * heads * block * dim, (b + 1) * heads * block * dim)
        for got, want in ((k[at], wk[at]), (v[at], wv[at])):
            if fmt == R.E4M3:
                got, want = np.where(got == 0x80, 0, got), np.where(want == 0x80, 0, want)
            np.testing.assert_array_equal(got, want)
        np.testing.assert_array_equal(ks[b], ref.scales[0, b].astype(np.float32))
        np.testing.assert_array_equal(vs[b], ref.scales[1, b].astype(np.float32))
    assert np.isnan(ks[0]).all()     # other blocks are left alone


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,dim,block,lens,pad", [
    (2, 128, 16, [(0, 40), (7, 20), (16, 1), (31, 1), (15, 18)], 0), (8, 128, 32, [(0, 300), (5, 90)], 12),
    (1, 64, 64, [(0, 1), (63, 2), (64, 200)], 4), (4, 256, 16, [(3, 70), (0, 33)], 0),
    (1, 128, 16, [(0, 2500)], 0), (1, 64, 256, [(100, 700), (0, 2000)], 0)])
def test_append_prompts(device, pool, fmt, heads, dim, block, lens, pad):
    """Several requests' rows in one call, starting and ending inside blocks; above 2048 rows too."""
    rng = np.random.default_rng(11)
    need = [-(-(o + n) // block) for o, n in lens]
    ids, at, slots, held = rng.permutation(sum(need) + 2), 0, [], []
    for (o, n), b in zip(lens, need):
        t = ids[at:at + b]
        at += b
        held += [t[x // block] * block + x % block for x in range(o // block * block, o)]
        slots += [t[x // block] * block + x % block for x in range(o, o + n)]
    ref = R.Cache(fmt, heads, dim, block, len(ids))
    if held:
        ref.append(*rows_of(rng, len(held), heads, dim, 0.3), held)     # smaller, so that some scales grow
    p = pool(fmt, heads, dim, block, len(ids), ref)
    cut = lens[0][1]       # rows to skip, between two requests (a block's rows follow one another)
    slots = slots[:cut] + [-1, len(ids) * block, 2 ** 31 - 1] + slots[cut:]
    k, v = rows_of(rng, len(slots), heads, dim)
    bad = [i for i, s in enumerate(slots) if not 0 <= s < len(ids) * block]
    k[bad], v[bad] = np.nan, np.inf
    ref.append(k, v, slots)
    p.append(k, v, slots, pad)
    p.check()


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_special_values(device, pool, fmt):
    """Zeros, the smallest and largest numbers, exact ties, infinities and NaN, a slot given twice, any order of offsets."""
    ref = R.Cache(fmt, 1, 64, 16, 12)
    p = pool(fmt, 1, 64, 16, 12, ref)
    rng = np.random.default_rng(2)

    def put(block, rows, offsets):
        k = np.asarray(rows, np.float32).reshape(len(offsets), 1, 64)
        v = (k * np.float32(0.5))[:, :, ::-1].copy()
        slots = [block * 16 + o for o in offsets]
        ref.append(k, v, slots)
        p.append(k, v, slots)

    x = rng.standard_normal((16, 64)).astype(np.float32)
    put(0, np.zeros((2, 64)), [0, 1])                       # no scale yet
    put(0, x[:1], [2])                                      # the first value sets it
    put(0, np.zeros((1, 64)), [3])
    put(1, np.full((1, 64), 1e-45), [0])                    # the scale's floor
    put(1, x[:2], [1, 2])                                   # grows by far: the old codes become 0
    put(2, np.full((1, 64), np.finfo(np.float32).max), [0])
    put(2, x[:2], [1, 2])
    ties = np.arange(64) - 31.5                             # halves between codes
    put(3, np.concatenate([[127.0], ties[1:]])[None], [0])
    put(3, np.concatenate([[254.0], 2 * ties[1:]])[None], [1])     # grows by 2: halves again
    put(4, (np.arange(64) - 32) / 16.0 * 1.0625 * 100, [0])
    put(5, x[:3], [0, 1, 2])
    put(5, np.where(np.arange(64) == 9, np.nan, x[3:4]), [3])       # NaN in one token
    put(5, x[4:5], [4])
    put(6, np.where(np.arange(64) == 9, -np.inf, x[3:4]), [0])
    put(7, np.where(np.arange(64) == 9, np.inf, x[3:4]), [0])
    put(7, x[:1], [0])                                      # started anew
    put(8, x[:4], [3, 0, 2, 1])
    put(9, np.stack([x[0], 100 * x[1], x[2]]), [0, 1, 1])   # twice the same: the later stays, both count
    put(10, x[:16], range(16))
    put(10, 3 * x[5:6], [5])                                # a token written again
    p.check()
    assert np.isnan(ref.scales[0, 5, 0]) and ref.scales[0, 0, 0] > 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [127, 128, 700, 2100])
@pytest.mark.parametrize("heads,dim,block", [(2, 128, 16), (1, 64, 32), (1, 256, 16)])
def test_append_mixed_runs(device, pool, fmt, heads, dim, block, rows):
    """Single tokens, runs of a few, whole blocks and skipped rows side by side, into blocks with and without tokens."""
    rng = np.random.default_rng(rows + dim)
    n_blocks = rows + 3
    ref = R.Cache(fmt, heads, dim, block, n_blocks)
    p = pool(fmt, heads, dim, block, n_blocks, ref)
    ids = list(rng.permutation(n_blocks))
    started = ids[::3]
    k, v = rows_of(rng, len(started), heads, dim)
    ref.append(k, v, [b * block for b in started])
    p.append(k, v, [b * block for b in started])
    slots = []
    while len(slots) < rows:
        n = int(rng.choice([1, 1, 1, 2, 5, block, 0]))
        if n == 0:
            slots.append(-1)
            continue
        b = ids.pop()
        first = 1 + int(rng.integers(0, block - n)) if n < block else 0
        slots += [int(b) * block + first + i for i in range(n)]
    slots = slots[:rows]
    k, v = rows_of(rng, rows, heads, dim, 3.0)
    skipped = np.array(slots) < 0
    k[skipped], v[skipped] = np.nan, np.inf
    ref.append(k, v, slots)
    p.append(k, v, slots)
    p.check()


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_quotients_beside_ties(device, pool, fmt):
    """Values whose quotient by the scale lies within an ulp of a tie, for many scales."""
    rng = np.random.default_rng(8)
    n = 200
    ref = R.Cache(fmt, 2, 128, 16, n)
    p = pool(fmt, 2, 128, 16, n, ref)
    top = np.float32(2.0) ** rng.integers(-40, 40, n) * rng.uniform(1, 2, n).astype(np.float32)
    k = np.zeros((n, 2, 128), np.float32)
    for b in range(n):
        s = R.first_scale(float(top[b]), fmt)
        if fmt == R.INT8:
            at = (rng.integers(-126, 126, (2, 128)) + 0.5) * s
        else:
            at = np.ldexp(rng.integers(16, 32, (2, 128)) + 0.5, rng.integers(-12, 3, (2, 128))) * s
        near = at.astype(np.float32)
        step = rng.integers(-1, 2, (2, 128))
        near = np.where(step < 0, np.nextafter(near, np.float32(-np.inf)), np.where(step > 0, np.nextafter(near, np.float32(np.inf)), near))
        k[b] = np.clip(near, -top[b], top[b])
        k[b, :, 0] = top[b]
    slots = [b * 16 for b in range(n)]
    ref.append(k, -k, slots)
    p.append(k, -k, slots)
    p.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,dim,block,rows", [(2, 128, 16, 50), (1, 64, 32, 1), (3, 128, 16, 333), (2, 256, 64, 2200)])
def test_append_rope(device, pool, fmt, heads, dim, block, rows):
    """Bit for bit aih_rope of queries and keys, then aih_kv_append; parts of one projection's rows."""
    L, h, n_heads = nat.lib(), device.handle, 2 * heads
    rng = np.random.default_rng(rows)
    n_blocks, past = -(-(rows + 5) // block) + 1, 5
    a, b = (pool(fmt, heads, dim, block, n_blocks) for _ in range(2))
    ids = rng.permutation(n_blocks)
    slots = [ids[x // block] * block + x % block for x in range(past, past + rows)]
    first = rows_of(rng, past, heads, dim)
    for p in (a, b):
        p.append(first[0], first[1], [ids[0] * block + x for x in range(past)])
    qd, kd = n_heads * dim, heads * dim
    ld = qd + 2 * kd
    qkv = rng.standard_normal((rows, ld)).astype(np.float32)
    table = device.create_buffer((past + rows) * dim * 4)
    nat.check(L.aih_rope_table(h, table.get_pointer(), past + rows, dim, 10000.0), "table")
    x, y = upload(device, qkv), upload(device, qkv)
    sb, pb = upload(device, np.asarray(slots, I32)), upload(device, np.arange(past, past + rows, dtype=I32))
    nat.check(L.aih_kv_append_rope(h, a.p, x.get_pointer(), ld, n_heads, x.get_pointer() + 4 * qd, ld,
                                   x.get_pointer() + 4 * (qd + kd), ld, sb.get_pointer(), pb.get_pointer(), rows,
                                   table.get_pointer(), past + rows), "aih_kv_append_rope")
    for off, nh in ((0, n_heads), (qd, heads)):
        nat.check(L.aih_rope(h, y.get_pointer() + 4 * off, ld, y.get_pointer() + 4 * off, ld, rows, nh, dim, past, None,
                             table.get_pointer(), past + rows, 0, rows), "aih_rope")
    nat.check(L.aih_kv_append(h, b.p, y.get_pointer() + 4 * qd, ld, y.get_pointer() + 4 * (qd + kd), ld,
                              sb.get_pointer(), rows), "aih_kv_append")
    device.synchronize()
    gx, gy = (t.read_range(0, rows * ld, np.float32).reshape(rows, ld) for t in (x, y))
    np.testing.assert_array_equal(gx[:, :qd], gy[:, :qd])
    np.testing.assert_array_equal(gx[:, qd:], qkv[:, qd:])      # keys and values are only read
    for u, w in zip(a.state(), b.state()):
        np.testing.assert_array_equal(u, w)
    # positions outside the table: neither rotated nor stored
    before = a.state()
    x.write(qkv)
    pb.write(np.where(np.arange(rows) % 2, -1, past + rows).astype(I32))
    nat.check(L.aih_kv_append_rope(h, a.p, x.get_pointer(), ld, n_heads, x.get_pointer() + 4 * qd, ld,
                                   x.get_pointer() + 4 * (qd + kd), ld, sb.get_pointer(), pb.get_pointer(), rows,
                                   table.get_pointer(), past + rows), "aih_kv_append_rope")
    device.synchronize()
    np.testing.assert_array_equal(x.read_range(0, rows * ld, np.float32).reshape(rows, ld), qkv)
    for u, w in zip(before, a.state()):
        np.testing.assert_array_equal(u, w)
    for t in (table, x, y, sb, pb):
        t.dispose()


# ---- read ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,dim,block", [(1, 64, 16), (3, 128, 32), (2, 256, 64)])
def test_read(device, pool, fmt, heads, dim, block):
    rng = np.random.default_rng(4)
    ref = R.Cache(fmt, heads, dim, block, 6)
    ref.fill_random(rng, 100.0)
    ref.scales[0, 2] = np.nan
    p = pool(fmt, heads, dim, block, 6, ref)
    slots = np.concatenate([rng.integers(0, 6 * block, 75), [-1, 6 * block, 2 ** 31 - 1, -2 ** 31, 0]]).astype(I32)
    wide, ld = heads * dim, heads * dim + 4
    sb = upload(device, slots)
    out = [upload(device, np.full(len(slots) * ld, -3, np.float32)) for _ in range(2)]
    nat.check(nat.lib().aih_kv_read(device.handle, p.p, sb.get_pointer(), len(slots), out[0].get_pointer(), ld,
                                    out[1].get_pointer(), ld), "aih_kv_read")
    device.synchronize()
    vals = ref.values()
    inside = (slots >= 0) & (slots < 6 * block)
    for o, v in zip(out, vals):
        got = o.read_range(0, len(slots) * ld, np.float32).reshape(-1, ld)
        want = np.where(inside[:, None], v.reshape(-1, wide)[np.where(inside, slots, 0)], 0).astype(np.float32)
        np.testing.assert_array_equal(got[:, :wide], want)
        assert np.all(got[:, wide:] == -3)
        o.dispose()
    sb.dispose()
