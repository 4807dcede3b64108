"""Paged 8-bit KV cache of many requests over the HIP library (aih_kv_*).

One pool of blocks serves every request; the block tables, the stack of free
blocks and the requests' lengths live in device memory, so that a step --
plan, append, attention -- can be captured into a graph and replayed while
the requests grow.  Every layer has its own codes and scales under the same
tables.

    cache = PagedKvCache(device, n_layers, n_kv_heads, head_dim, n_blocks=..., max_seqs=..., max_len=..., max_rows=...)
    cache.plan([n_0, n_1, ...])              # new tokens of each request: blocks, slots, row starts
    for l in layers:
        cache.append(l, k, ldk, v, ldv)      # or append_rope
        cache.attention(l, q, ldq, o, ldo, n_heads, scale)
    cache.release([1, 0, ...])               # give the blocks of finished requests back

The reference keeps one fp32 cache per conversation and concatenates to it
(AIHost/AIHost/Inference/InferenceEngine.cs:585-622).
"""
import ctypes

import numpy as np

from . import _native as nat

FORMATS = {"int8": nat.KV_INT8, "e4m3": nat.KV_E4M3}


class PagedKvCache:
    """Requests 0 .. max_seqs-1 of up to max_len tokens each (rounded up to
    whole blocks: only past that does plan() refuse) over n_blocks blocks of
    block_tokens tokens; a step has up to max_rows rows.  fmt: "int8" or
    "e4m3".  One device, one stream: its steps share the scratch of attention()
    and run one after the other."""

    def __init__(self, device, n_layers, n_kv_heads, head_dim, n_blocks, max_seqs, max_len, max_rows, fmt="int8",
                 block_tokens=32):
        if fmt not in FORMATS:
            raise ValueError("KV cache format %r (one of %s)" % (fmt, ", ".join(sorted(FORMATS))))
        self.dev, self.h, self.L = device, device.handle, nat.lib()
        self.n_layers, self.max_seqs, self.max_len, self.max_rows = n_layers, int(max_seqs), int(max_len), int(max_rows)
        self.n_blocks, self.block_tokens = int(n_blocks), int(block_tokens)
        self.width = -(-self.max_len // self.block_tokens)
        self._bufs = []
        self.caches = []
        shape = nat.KvCache(format=FORMATS[fmt], n_kv_heads=n_kv_heads, head_dim=head_dim,
                            block_tokens=self.block_tokens, n_blocks=self.n_blocks)
        nbytes = nat.check_size(self.L.aih_kv_cache_bytes(ctypes.byref(shape)), "aih_kv_cache_bytes")
        try:
            for _ in range(n_layers):
                c = nat.KvCache()
                ctypes.pointer(c)[0] = shape
                c.k, c.v = self._buf(nbytes), self._buf(nbytes)
                c.k_scale, c.v_scale = (self._buf(4 * self.n_blocks * n_kv_heads) for _ in range(2))
                self.caches.append(c)
            S, R = self.max_seqs, self.max_rows
            self.lens, self.n_new, self.done = self._buf(4 * S), self._buf(4 * S), self._buf(4 * S)
            self.tables, self.free_blocks = self._buf(4 * S * self.width), self._buf(4 * self.n_blocks)
            self.n_free, self.refused = self._buf(4), self._buf(4)
            self.starts, self.slots, self.positions = self._buf(4 * (S + 1)), self._buf(4 * R), self._buf(4 * R)
            self.scratch, self.scratch_floats = None, 0
            self.reset()
        except Exception:
            self.dispose()
            raise

    def _buf(self, nbytes):
        b = self.dev.create_buffer(max(16, int(nbytes)))
        self._bufs.append(b)
        return b.get_pointer()

    def _put(self, ptr, values):
        a = np.ascontiguousarray(values, dtype=np.int32)
        nat.check(self.L.aih_memcpy_h2d(self.h, ptr, a.ctypes.data, a.nbytes), "aih_memcpy_h2d")

    def _get(self, ptr, count):
        a = np.empty(count, dtype=np.int32)
        nat.check(self.L.aih_memcpy_d2h(self.h, a.ctypes.data, ptr, a.nbytes), "aih_memcpy_d2h")
        return a

    def reset(self):
        """Empty every request and free every block (the blocks' contents go with them)."""
        self._put(self.free_blocks, np.arange(self.n_blocks)[::-1])
        self._put(self.n_free, [self.n_blocks])
        self._put(self.lens, np.zeros(self.max_seqs))
        self._put(self.tables, np.full(self.max_seqs * self.width, -1))
        self._put(self.n_new, np.zeros(self.max_seqs))
        self._put(self.starts, np.zeros(self.max_seqs + 1))
        self._put(self.refused, [0])
        self.rows = 0

    def reserve(self, n_heads, rows):
        """Scratch for attention() of `n_heads` query heads over `rows` rows
        (at least twice as much as before when it grows).
        It cannot grow while the stream is being captured: reserve what the
        captured calls need before."""
        floats = nat.check_size(self.L.aih_kv_attention_scratch_floats(
            self.h, ctypes.byref(self.caches[0]), n_heads, int(rows), self.max_seqs, self.width),
            "aih_kv_attention_scratch_floats")
        if floats > self.scratch_floats:
            # the smaller one stays, since captured graphs may still point at it: with at least twice the room each time
            # all of them together are below four times what is needed
            floats = max(floats, 2 * self.scratch_floats)
            self.scratch, self.scratch_floats = self._buf(4 * floats), floats

    # -- a step
    def set_new(self, n_new):
        """The tokens each request adds in the steps that follow (kept on the device)."""
        n = np.zeros(self.max_seqs, dtype=np.int32)
        n[:len(n_new)] = n_new
        self._put(self.n_new, n)

    def plan(self, n_new=None, rows=None):
        """aih_kv_plan of the next step, in place; n_new: new tokens of each
        request (None: as set_new left them); rows: the rows that slots,
        positions and the calls below cover (default: max_rows; queries of
        all of them are read, and attention() chooses its tile by their
        number, so a step of few rows is faster with its own number)."""
        if n_new is not None:
            self.set_new(n_new)
        rows = self.max_rows if rows is None else int(rows)
        if not 0 <= rows <= self.max_rows:
            raise ValueError("%d rows (max %d)" % (rows, self.max_rows))
        nat.check(self.L.aih_kv_plan(self.h, self.lens, self.n_new, self.max_seqs, self.tables, self.width,
                                     self.block_tokens, self.n_blocks, self.free_blocks, self.n_free, self.lens,
                                     self.n_free, self.starts, self.slots, self.positions, rows, self.refused),
                  "aih_kv_plan")
        self.rows = rows

    def append(self, layer, k, ldk, v, ldv):
        """The step's key and value rows into a layer's cache (aih_kv_append)."""
        nat.check(self.L.aih_kv_append(self.h, ctypes.byref(self.caches[layer]), k, ldk, v, ldv, self.slots, self.rows),
                  "aih_kv_append")

    def append_rope(self, layer, q, ldq, n_heads, k, ldk, v, ldv, table, table_rows):
        """append() with the rotation of queries and keys (aih_kv_append_rope)."""
        nat.check(self.L.aih_kv_append_rope(self.h, ctypes.byref(self.caches[layer]), q, ldq, n_heads, k, ldk, v, ldv,
                                            self.slots, self.positions, self.rows, table, table_rows),
                  "aih_kv_append_rope")

    def attention(self, layer, q, ldq, o, ldo, n_heads, scale, scores=None):
        """Attention of the step's query rows over a layer's cache (aih_kv_attention)."""
        self.reserve(n_heads, self.rows)
        nat.check(self.L.aih_kv_attention(self.h, ctypes.byref(self.caches[layer]), q, ldq, o, ldo, self.rows, n_heads,
                                          self.max_seqs, self.starts, self.lens, self.tables, self.width, scale,
                                          ctypes.byref(scores) if scores is not None else None, self.scratch,
                                          self.scratch_floats), "aih_kv_attention")

    # -- requests
    def release(self, done=None):
        """Give the blocks of the requests with a non-zero entry in `done`
        (None: of all) back to the pool."""
        flags = None
        if done is not None:
            d = np.zeros(self.max_seqs, dtype=np.int32)
            d[:len(done)] = done
            self._put(self.done, d)
            flags = self.done
        nat.check(self.L.aih_kv_release(self.h, self.lens, self.max_seqs, self.tables, self.width, self.block_tokens,
                                        self.n_blocks, flags, self.free_blocks, self.n_free), "aih_kv_release")

    def lengths(self):
        """Tokens held of each request (waits for the device)."""
        return self._get(self.lens, self.max_seqs)

    def free(self):
        """Free blocks (waits for the device)."""
        return int(self._get(self.n_free, 1)[0])

    def last_refused(self):
        """Requests that the last plan refused (waits for the device)."""
        return int(self._get(self.refused, 1)[0])

    def read(self, layer, request):
        """(keys, values) that a layer holds of a request, as fp32 arrays of
        (tokens, n_kv_heads * head_dim) (aih_kv_read; waits for the device)."""
        if not 0 <= request < self.max_seqs:
            raise IndexError("request %d (of %d)" % (request, self.max_seqs))
        c = self.caches[layer]
        n, wide = int(self.lengths()[request]), c.n_kv_heads * c.head_dim
        t = self._get(self.tables + 4 * request * self.width, self.width)
        j = np.arange(n)
        slots = np.ascontiguousarray(t[j // self.block_tokens] * self.block_tokens + j % self.block_tokens, np.int32)
        sb = self.dev.create_buffer(max(16, 4 * n))
        out = [self.dev.create_buffer(max(16, 4 * n * wide)) for _ in range(2)]
        try:
            if n:
                sb.write(slots)
                nat.check(self.L.aih_kv_read(self.h, ctypes.byref(c), sb.get_pointer(), n, out[0].get_pointer(), wide,
                                             out[1].get_pointer(), wide), "aih_kv_read")
            return tuple(b.read_range(0, n * wide, np.float32).reshape(n, wide) for b in out)
        finally:
            for b in [sb] + out:
                b.dispose()

    def dispose(self):
        for b in self._bufs:
            b.dispose()
        self._bufs, self.caches = [], []
        # the library refuses NULL, so that no later call reaches what is freed
        self.lens = self.n_new = self.done = self.tables = self.free_blocks = self.n_free = self.refused = None
        self.starts = self.slots = self.positions = self.scratch = None
