"""PagedKvCache's own checks and bookkeeping, on the CPU: a cache without a
device, whose buffers are recorded and whose library calls are counted."""
import ctypes

import numpy as np
import pytest

from aihost_amd import _native as nat
from aihost_amd.kvcache import PagedKvCache


class Buffer:
    def __init__(self, nbytes):
        self.nbytes, self.live = nbytes, True

    def get_pointer(self):
        return 1 << 20

    def dispose(self):
        self.live = False


class Device:
    def __init__(self):
        self.buffers = []

    def create_buffer(self, nbytes):
        self.buffers.append(Buffer(nbytes))
        return self.buffers[-1]


class Library:
    """What is called, and a scratch size that depends on the rows alone."""

    def __init__(self):
        self.calls = []

    def aih_kv_attention_scratch_floats(self, h, kv, n_heads, rows, n_seqs, width):
        return 1000 * rows

    def __getattr__(self, name):
        def f(*a):
            self.calls.append(name)
            return nat.AIH_OK
        return f


@pytest.fixture
def cache():
    c = PagedKvCache.__new__(PagedKvCache)
    c.dev, c.h, c.L = Device(), None, Library()
    c.n_layers, c.max_seqs, c.max_len, c.max_rows, c.n_blocks, c.block_tokens, c.width = 1, 4, 100, 512, 16, 32, 4
    c._bufs, c.caches = [], [nat.KvCache(n_kv_heads=2, head_dim=64)]
    c.scratch, c.scratch_floats, c.rows = None, 0, 0
    for name in ("lens", "n_new", "done", "tables", "free_blocks", "n_free", "refused", "starts", "slots", "positions"):
        setattr(c, name, c._buf(4096))
    c.dev.buffers.clear()
    return c


@pytest.mark.parametrize("request_", [-1, -4, 4, 1 << 30])
def test_read_of_a_request_that_is_not_there(cache, request_):
    """Before the table is read: a request below 0 would be a row before it."""
    cache.lengths = lambda: np.zeros(4, np.int32)
    with pytest.raises(IndexError):
        cache.read(0, request_)
    assert not cache.L.calls


def test_scratch_grows_by_doubling(cache):
    """Steps whose sizes creep up: what is kept for captured graphs stays within four times what is needed."""
    for rows in range(1, 513):
        cache.reserve(8, rows)
        assert cache.scratch_floats >= 1000 * rows
    held = sum(b.nbytes for b in cache.dev.buffers if b.live)
    assert held <= 4 * (4 * 1000 * 512) and len(cache.dev.buffers) <= 11
    cache.reserve(8, 7)                          # a smaller step takes nothing
    assert len(cache.dev.buffers) <= 11


def test_exact_scratch_at_first(cache):
    cache.reserve(8, 3)
    assert cache.scratch_floats == 3000 and [b.nbytes for b in cache.dev.buffers] == [12000]


def test_nothing_is_reachable_after_dispose(cache):
    """The library refuses the pointers that are left, as it does those of a disposed buffer."""
    ctx = ctypes.create_string_buffer(1 << 14)          # refused calls read nothing of it
    cache.dispose()
    cache.L, cache.h, cache.rows = nat.lib(), ctypes.addressof(ctx), 1
    assert not cache.dev.buffers or not any(b.live for b in cache.dev.buffers)
    for call in (lambda: cache.plan(rows=1), lambda: cache.release(), lambda: cache.release([1]), lambda: cache.reset(),
                 lambda: cache.lengths()):
        with pytest.raises(nat.AihError) as e:
            call()
        assert e.value.status == nat.AIH_E_INVALID
    for call in (lambda: cache.append(0, 16, 128, 16, 128), lambda: cache.attention(0, 16, 128, 16, 128, 2, 1.0)):
        with pytest.raises(IndexError):
            call()
