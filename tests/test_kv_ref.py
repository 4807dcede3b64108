"""The paged cache's oracle, its layout and the refusals of its entry points,
on the CPU (a refused call returns before it looks at a device)."""
import ctypes

import numpy as np
import pytest

import kv_ref as R
from aihost_amd import _native as nat

INV, UNS, LIM = nat.AIH_E_INVALID, nat.AIH_E_UNSUPPORTED, nat.AIH_E_LIMIT


def test_layout_units():
    """Byte i of a key unit is dimension 64c + 16g + i of token 4t + r; byte i of value unit d is token i."""
    c = R.Cache(R.INT8, 2, 128, 32, 3)
    c.codes[0, 2, 1, 16 + 4 * 3 + 2, 64 * 1 + 16 * 2 + 5] = 7
    c.codes[1, 2, 1, 16 + 9, 77] = 9
    k, v = c.packed()
    base = (2 * 2 + 1) * 32 * 128 + 16 * 128
    assert k.nonzero()[0].tolist() == [base + (((3 * 2 + 1) * 4 + 2) * 4 + 2) * 16 + 5]
    assert v.nonzero()[0].tolist() == [base + 77 * 16 + 9]


@pytest.mark.parametrize("fmt", [R.INT8, R.E4M3])
def test_oracle_blocks(fmt):
    """A code ends within one step of its value however often the scale grows."""
    rng = np.random.default_rng(5)
    c = R.Cache(fmt, 1, 64, 16, 1)
    x = rng.standard_normal((16, 1, 64)) * 2.0 ** np.arange(16)[:, None, None] / 64
    for i in range(16):
        c.append(x[i:i + 1], x[i:i + 1], [i])
    err = np.abs(c.values()[0] - x)[:, 0]
    if fmt == R.INT8:
        assert np.all(err <= c.scales[0, 0, 0] * (1 + 1e-12))
    else:   # a step is 2^-3 of a normal value, 2^-9 scales of a smaller one; one rounding of half, then exact shifts
        assert np.all(err <= np.maximum(np.abs(x)[:, 0] * 2.0 ** -4, c.scales[0, 0, 0] * 2.0 ** -9) * (1 + 1e-12))
    assert c.scales[0, 0, 0] > 0
    assert R.first_scale(448.0, R.E4M3) == 1.0 and R.first_scale(449.0, R.E4M3) == 2.0
    assert R.first_scale(1e-45, R.INT8) == R.first_scale(1e-45, R.E4M3) == 2.0 ** -126


def cache(**kw):
    a = dict(format=nat.KV_INT8, n_kv_heads=2, head_dim=128, block_tokens=16, n_blocks=8, k=4096, v=8192, k_scale=16,
             v_scale=32)
    a.update(kw)
    return nat.KvCache(**a)


SHAPES = [(dict(format=2), UNS), (dict(format=-1), UNS), (dict(head_dim=96), UNS), (dict(head_dim=0), UNS),
          (dict(block_tokens=8), UNS), (dict(block_tokens=24), UNS), (dict(block_tokens=512), UNS),
          (dict(n_kv_heads=0), INV), (dict(n_blocks=0), INV), (dict(n_blocks=-1), INV), (dict(reserved=1), INV),
          (dict(n_blocks=1 << 27), LIM), (dict(n_blocks=(1 << 27) - 1, n_kv_heads=32), LIM)]
POINTERS = [(dict(k=None), INV), (dict(v=None), INV), (dict(k_scale=None), INV), (dict(v_scale=None), INV),
            (dict(k=8), INV), (dict(v=4104), INV), (dict(k_scale=18), INV)]


def test_cache_bytes():
    L = nat.lib()
    assert L.aih_kv_cache_bytes(ctypes.byref(cache(k=None))) == 8 * 16 * 2 * 128
    assert L.aih_kv_cache_bytes(ctypes.byref(cache(n_blocks=1 << 20, block_tokens=64, n_kv_heads=8))) == 1 << 36
    assert L.aih_kv_cache_bytes(None) == INV
    for kw, want in SHAPES:
        assert L.aih_kv_cache_bytes(ctypes.byref(cache(**kw))) == want, kw


# a context whose fields are all zero: refused calls read no more of it than its CU count
_fake = ctypes.create_string_buffer(1 << 14)
CTX = ctypes.addressof(_fake)


def plan(ctx=CTX, lens=16, n_new=16, n_seqs=2, tables=16, width=4, bt=16, nb=8, free=16, n_free=16, new_lens=16,
         new_n_free=16, starts=16, slots=16, positions=16, rows=0, refused=16):
    return nat.lib().aih_kv_plan(ctx, lens, n_new, n_seqs, tables, width, bt, nb, free, n_free, new_lens, new_n_free,
                                 starts, slots, positions, rows, refused)


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=None), INV), (dict(lens=None), INV), (dict(n_new=None), INV), (dict(tables=None), INV),
    (dict(free=None), INV), (dict(n_free=None), INV), (dict(new_lens=None), INV), (dict(new_n_free=None), INV),
    (dict(starts=None), INV), (dict(slots=None), INV), (dict(positions=None), INV), (dict(refused=None), INV),
    (dict(n_seqs=0), INV), (dict(n_seqs=-1), INV), (dict(width=0), INV), (dict(nb=0), INV), (dict(rows=-1), INV),
    (dict(bt=0), UNS), (dict(bt=17), UNS), (dict(n_seqs=4097), LIM), (dict(rows=1 << 31), LIM),
    (dict(nb=1 << 27), LIM), (dict(width=1 << 27), LIM)])
def test_plan_refuses(kw, want):
    assert plan(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=None), INV), (dict(lens=None), INV), (dict(tables=None), INV), (dict(free=None), INV),
    (dict(n_free=None), INV), (dict(n_seqs=0), INV), (dict(width=0), INV), (dict(nb=0), INV), (dict(bt=31), UNS),
    (dict(n_seqs=4097), LIM), (dict(nb=1 << 27), LIM), (dict(width=1 << 27), LIM)])
def test_release_refuses(kw, want):
    a = dict(ctx=CTX, lens=16, n_seqs=2, tables=16, width=4, bt=16, nb=8, free=16, n_free=16)
    a.update(kw)
    assert nat.lib().aih_kv_release(a["ctx"], a["lens"], a["n_seqs"], a["tables"], a["width"], a["bt"], a["nb"], None,
                                    a["free"], a["n_free"]) == want


ROWS = [(dict(ctx=None), INV), (dict(K=None), INV), (dict(V=None), INV), (dict(slots=None), INV), (dict(rows=-1), INV),
        (dict(ldk=252), INV), (dict(ldv=255), INV), (dict(ldk=257), INV), (dict(ldv=258), INV), (dict(K=4), INV),
        (dict(V=24), INV), (dict(rows=1 << 31), LIM), (dict(rows=0), nat.AIH_OK)]


@pytest.mark.parametrize("name", ["aih_kv_append", "aih_kv_read", "aih_kv_append_rope"])
def test_row_operators_refuse(name):
    def call(kv=None, ctx=CTX, K=16, ldk=256, V=16, ldv=256, slots=16, rows=0):
        c = None if kv == "null" else ctypes.byref(kv or cache())
        f = getattr(nat.lib(), name)
        if name == "aih_kv_read":
            return f(ctx, c, slots, rows, K, ldk, V, ldv)
        if name == "aih_kv_append":
            return f(ctx, c, K, ldk, V, ldv, slots, rows)
        return f(ctx, c, 16, 512, 4, K, ldk, V, ldv, slots, 16, rows, 16, 100)

    for kw, want in ROWS:
        assert call(**kw) == want, kw
    for kw, want in SHAPES + POINTERS:
        assert call(kv=cache(**kw)) == want, kw
    assert call(kv="null") == INV


def test_rope_refuses():
    def call(Q=16, ldq=512, n_heads=4, positions=16, table=16, table_rows=100):
        return nat.lib().aih_kv_append_rope(CTX, ctypes.byref(cache()), Q, ldq, n_heads, 16, 256, 16, 256, 16, positions,
                                            0, table, table_rows)

    assert call() == nat.AIH_OK
    for kw in (dict(Q=None), dict(ldq=508), dict(ldq=514), dict(n_heads=0), dict(positions=None), dict(table=None),
               dict(table_rows=0), dict(Q=8), dict(table=8)):
        assert call(**kw) == INV, kw


@pytest.mark.parametrize("kw,want", [
    (dict(), nat.AIH_OK), (dict(ctx=None), INV), (dict(Q=None), INV), (dict(O=None), INV), (dict(starts=None), INV),
    (dict(lens=None), INV), (dict(tables=None), INV), (dict(rows=-1), INV), (dict(n_heads=0), INV),
    (dict(n_heads=3), INV), (dict(n_seqs=0), INV), (dict(width=0), INV), (dict(ldq=508), INV), (dict(ldo=510), INV),
    (dict(ldo=508), INV), (dict(Q=8), INV), (dict(O=20), INV), (dict(scale=0.0), INV), (dict(scale=-1.0), INV),
    (dict(scale=float("nan")), INV), (dict(scale=float("inf")), INV), (dict(cap=-1.0), INV),
    (dict(cap=float("nan")), INV), (dict(cap=float("inf")), INV), (dict(window=-1), INV), (dict(n_seqs=4097), LIM),
    (dict(width=1 << 27), LIM), (dict(rows=1 << 31), LIM), (dict(rows=4, scratch=None, width=4096), INV),
    (dict(rows=4, scratch=8, width=4096), INV), (dict(rows=4, floats=0, width=4096), INV)])
def test_attention_refuses(kw, want):
    a = dict(ctx=CTX, Q=16, ldq=512, O=16, ldo=512, rows=0, n_heads=4, n_seqs=2, starts=16, lens=16, tables=16, width=4,
             scale=0.1, cap=0.0, window=0, scratch=16, floats=1 << 40)
    a.update(kw)
    sc = nat.KvScores(cap=a["cap"], window=a["window"])
    assert nat.lib().aih_kv_attention(a["ctx"], ctypes.byref(cache()), a["Q"], a["ldq"], a["O"], a["ldo"], a["rows"],
                                      a["n_heads"], a["n_seqs"], a["starts"], a["lens"], a["tables"], a["width"],
                                      a["scale"], ctypes.byref(sc), a["scratch"], a["floats"]) == want


def test_attention_refuses_caches():
    L = nat.lib()
    for kw, want in SHAPES + POINTERS:
        assert L.aih_kv_attention(CTX, ctypes.byref(cache(**kw)), 16, 512, 16, 512, 1, 4, 2, 16, 16, 16, 4, 0.1, None, 16,
                                  1 << 40) == want, kw
    for kw, want in SHAPES:
        assert L.aih_kv_attention_scratch_floats(CTX, ctypes.byref(cache(**kw)), 4, 8, 2, 4) == want, kw
        assert L.aih_kv_attention_tile_rows(CTX, ctypes.byref(cache(**kw)), 4, 8, 2, 4) == want, kw
    ok = ctypes.byref(cache())
    assert L.aih_kv_attention_scratch_floats(None, ok, 4, 8, 2, 4) == INV
    assert L.aih_kv_attention_scratch_floats(CTX, None, 4, 8, 2, 4) == INV
    for bad in ((3, 8, 2, 4), (4, -1, 2, 4), (4, 8, 0, 4), (4, 8, 2, 0)):
        assert L.aih_kv_attention_scratch_floats(CTX, ok, *bad) == INV
        assert L.aih_kv_attention_tile_rows(CTX, ok, *bad) == INV
    assert L.aih_kv_attention_tile_rows(None, ok, 4, 8, 2, 4) == INV
    assert L.aih_kv_attention_scratch_floats(CTX, ok, 4, 8, 4097, 4) == LIM
    # tables too short to be split need no scratch; longer ones do
    assert L.aih_kv_attention_scratch_floats(CTX, ok, 4, 8, 2, 4) == 0
    assert L.aih_kv_attention_scratch_floats(CTX, ok, 4, 8, 2, 4096) > 0


def test_sizes_past_a_launch_refused():
    """More heads than an index of a row's values holds, or more threads than one launch counts."""
    L, c = nat.lib(), ctypes.byref(cache())
    assert L.aih_kv_cache_bytes(ctypes.byref(cache(n_kv_heads=65535))) == 8 * 16 * 65535 * 128
    assert L.aih_kv_cache_bytes(ctypes.byref(cache(n_kv_heads=65536))) == LIM
    assert L.aih_kv_append(CTX, c, 16, 256, 16, 256, 16, 1 << 30) == LIM
    assert L.aih_kv_read(CTX, c, 16, 1 << 30, 16, 256, 16, 256) == LIM
    assert L.aih_kv_append_rope(CTX, c, 16, 1 << 24, 65536, 16, 256, 16, 256, 16, 16, 1, 16, 100) == LIM
    assert L.aih_kv_append_rope(CTX, c, 16, 1 << 20, 8192, 16, 256, 16, 256, 16, 16, 1 << 17, 16, 100) == LIM
    assert L.aih_kv_attention(CTX, c, 16, 1 << 24, 16, 1 << 24, 1, 65536, 2, 16, 16, 16, 4, 0.1, None, 16, 1 << 40) == LIM
    assert L.aih_kv_attention(CTX, c, 16, 512, 16, 512, 1 << 29, 4, 2, 16, 16, 16, 4, 0.1, None, 16, 1 << 40) == LIM


def test_plan_rows_below_the_sums_limit():
    """Sums of rows stop at 2^31 - 1, which has to be more than `rows`: a batch of more rows would be taken for one that fits."""
    assert plan(rows=(1 << 31) - 1) == LIM
