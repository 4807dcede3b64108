"""The paged 8-bit KV cache as it is used: a server's requests that come, grow
and go (PagedKvCache), and the decoder on it (LlamaDecoder(kv_format=...)).

Bars.  Attention: those of test_gpu_kv_attention.  Decoder logits against
the oracle decoder whose keys and values go through the oracle's cache
(kv_ref.Cache): 1e-2 normwise.  Without the cache the bar is 3e-3
(test_gpu_decoder).  With it, a key or value off by d lands on another code
for a share d / step of the values, which are then off by a whole step: the
root mean square becomes sqrt(d step).  With d = 3e-4 of a unit-normal value
(fp16 GEMM operands) and a step of 2^-5 (int8: 4 / 127; e4m3: 2^-4 to 2^-3
of the value) that is 3e-3 to 6e-3 of each value, averaged over keys by the
attention, once per layer, beside a residual that does not change."""
import ctypes

import numpy as np
import pytest

import kv_ref as R
from aihost_amd import _native as nat
from aihost_amd import llama
from aihost_amd.kvcache import PagedKvCache
from gpu_util import upload
from oracle import llama as ol
from test_gpu_kv_attention import BAR

pytestmark = pytest.mark.gpu

CFG = llama.LlamaConfig(n_layers=2, dim=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
TOL = 1e-2
FORMATS = {"int8": R.INT8, "e4m3": R.E4M3}


@pytest.fixture(scope="module")
def model(device):
    w = llama.synth_weights(CFG, seed=5)
    dw = llama.DeviceWeights(device, w)
    yield w, dw
    dw.dispose()


class Rows:
    """Keys or values of the oracle decoder, kept in the oracle's cache."""

    def __init__(self, cache, which):
        self.cache, self.which, self.wait = cache, which, None

    def __setitem__(self, at, x):
        self.pending = (at, np.asarray(x, np.float32))
        if self.other.wait is None:
            self.wait = True
            return
        a, b = (self, self.other) if self.which == 0 else (self.other, self)
        c = self.cache
        n = at.stop - at.start
        c.append(a.pending[1].reshape(n, c.heads, c.dim), b.pending[1].reshape(n, c.heads, c.dim),
                 list(range(at.start, at.stop)))
        self.wait = self.other.wait = None

    def __array__(self, dtype=None, copy=None):
        v = self.cache.values()[self.which]
        return v.reshape(v.shape[0], -1).astype(dtype or np.float64)


def oracle_setup(w, max_len, fmt):
    kv = []
    for _ in range(CFG.n_layers):
        c = R.Cache(fmt, CFG.n_kv_heads, CFG.head_dim, 32, -(-max_len // 32))
        k, v = Rows(c, 0), Rows(c, 1)
        k.other, v.other = v, k
        kv.append((k, v))
    return ol.Model(CFG, w), kv, ol.rope_table(max_len, CFG.head_dim, CFG.theta)


def rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("n", [40, 5, 1, 100])
def test_decoder_matches_oracle(device, model, fmt, n):
    """Prompts through the fused layer, through the separate operators (up to 8 rows) and of one token; then decode."""
    w, dw = model
    ids = np.random.default_rng(n).integers(0, CFG.vocab, n).astype(np.int32)
    dec = llama.LlamaDecoder(device, CFG, dw, 130, 100, kv_format=fmt)
    try:
        token = dec.prefill(ids)
        m, kv, table = oracle_setup(w, 130, FORMATS[fmt])
        ref = m.forward(list(ids), 0, kv, table)[0]
        assert rel(dec.read_logits(), ref) < TOL
        for step in range(5):
            dec.decode_step()
            ref = m.forward([token], n + step, kv, table)[0]
            got = dec.read_logits()
            assert rel(got, ref) < TOL, step
            token = int(np.argmax(got))
        assert dec.paged.lengths()[0] == n + 5
        # The caches against the oracle's: sqrt(d step), as above.  Layer 0: d = 3e-4, at most 6e-3.  Layer 1 is
        # computed from layer 0's output, whose own bar is 3e-3 (test_gpu_decoder): d = 3e-3 and a step of at most
        # 2^-3 of a value give sqrt(3e-3 / 8) = 1.94e-2.
        for layer, bar in ((0, TOL), (1, 2e-2)):
            keys, values = dec.paged.read(layer, 0)
            assert rel(keys, np.asarray(kv[layer][0])[:n + 5]) < bar
            assert rel(values, np.asarray(kv[layer][1])[:n + 5]) < bar
    finally:
        dec.dispose()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_decoder_graph_equals_eager(device, model, fmt):
    """Replays of the captured step (its plan among them) over block borders, two prompts, work in between."""
    _, dw = model
    ids = [np.random.default_rng(s).integers(0, CFG.vocab, k).astype(np.int32) for s, k in ((1, 29), (2, 60))]
    runs = []
    for use_graph in (False, True):
        dec = llama.LlamaDecoder(device, CFG, dw, 160, 64, kv_format=fmt)
        try:
            out = []
            for prompt in ids:
                dec.prefill(prompt)
                for k in (3, 40, 1):
                    dec.decode(k, use_graph=use_graph)
                    device.synchronize()
                    out.append((dec.tokens(dec.position - len(prompt) + 1).copy(), dec.read_logits().copy(),
                                dec.paged.lengths().copy(), dec.paged.free()))
            runs.append(out)
        finally:
            dec.dispose()
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)


def test_decoder_refuses_formats(device, model):
    with pytest.raises(ValueError):
        llama.LlamaDecoder(device, CFG, model[1], 64, 16, kv_format="int4")


# ---- a server's requests ------------------------------------------------------------
class Server:
    """PagedKvCache beside the oracle's bookkeeping and cache, one layer."""

    def __init__(self, device, fmt, heads, kv, dim, n_blocks, seqs, max_len, max_rows, block=16):
        self.dev, self.heads, self.kv, self.dim = device, heads, kv, dim
        self.c = PagedKvCache(device, 1, kv, dim, n_blocks, seqs, max_len, max_rows, fmt, block)
        self.ref = R.Cache(FORMATS[fmt], kv, dim, block, n_blocks)
        self.tables = np.full((seqs, self.c.width), -1)
        self.free = list(range(n_blocks))[::-1]
        self.lens = np.zeros(seqs, int)
        self.rng = np.random.default_rng(seqs)
        wide = heads * dim
        self.q, self.o = device.create_buffer(max_rows * wide * 4), device.create_buffer(max_rows * wide * 4)
        self.k, self.v = (device.create_buffer(max_rows * kv * dim * 4) for _ in range(2))
        self.scale = float(np.float32(1 / np.sqrt(dim)))

    def inputs(self, rows):
        """New rows in the buffers, and as the oracle's."""
        x = [self.rng.standard_normal((rows, n, self.dim)).astype(np.float32) for n in (self.heads, self.kv, self.kv)]
        for b, a in zip((self.q, self.k, self.v), x):
            b.write(a)
        self.o.write(np.full(rows * self.heads * self.dim, -7, np.float32))
        return x

    def launch(self, rows):
        """The step's calls (recorded, when the stream is being captured)."""
        w, kw = self.heads * self.dim, self.kv * self.dim
        self.c.plan(rows=rows)
        self.c.append(0, self.k.get_pointer(), kw, self.v.get_pointer(), kw)
        self.c.attention(0, self.q.get_pointer(), w, self.o.get_pointer(), w, self.heads, self.scale)

    def follow(self, n_new, rows, x):
        """The oracle's step, and the device's results against it."""
        p = R.plan(self.lens, n_new, self.tables, self.c.block_tokens, self.c.n_blocks, self.free, len(self.free), rows)
        del self.free[p["n_free"]:]
        self.lens = np.array(p["new_lens"])
        self.ref.append(x[1], x[2], p["slots"])
        got = self.o.read_range(0, rows * self.heads * self.dim, np.float32).reshape(rows, self.heads, self.dim)
        want, bound = R.attention(self.ref, x[0], p["starts"], self.lens, self.tables, self.scale)
        n = p["starts"][-1]
        assert np.all(got[n:] == -7)
        assert np.all(np.abs(got - want)[:n].max(-1, initial=0) <= bound[:n])
        if n:
            assert np.linalg.norm((got - want)[:n]) <= BAR * np.linalg.norm(want[:n])
        np.testing.assert_array_equal(self.c.lengths(), self.lens)
        assert (self.c.free(), self.c.last_refused()) == (len(self.free), p["refused"])
        return p

    def step(self, n_new, rows):
        x = self.inputs(rows)
        self.c.set_new(n_new)
        self.launch(rows)
        return self.follow(n_new, rows, x)

    def release(self, done):
        self.c.release(done)
        for s, d in enumerate(done):
            if d:
                n = -(-self.lens[s] // self.c.block_tokens)
                self.free += [int(b) for b in self.tables[s, :n]]
                self.tables[s, :n] = -1
                self.lens[s] = 0

    def dispose(self):
        for b in (self.q, self.o, self.k, self.v):
            b.dispose()
        self.c.dispose()


@pytest.mark.parametrize("fmt,heads,kv,dim", [("int8", 8, 2, 128), ("e4m3", 6, 2, 64), ("int8", 2, 1, 256)])
def test_requests_come_grow_and_go(device, fmt, heads, kv, dim):
    """Prompts beside decoding requests, chunks, a pool that runs out, released blocks used again."""
    s = Server(device, fmt, heads, kv, dim, 30, 5, 300, 200)
    try:
        s.step([40, 0, 0, 0, 0], 64)
        s.step([1, 100, 0, 7, 0], 128)
        for _ in range(18):
            s.step([1, 1, 0, 1, 0], 8)
        p = s.step([1, 1, 150, 1, 0], 200)          # ten blocks: all that is left, or more
        s.step([1, 60, 1, 1, 1], 200)
        while not p["refused"]:
            p = s.step([16, 16, 0, 16, 16], 64)
        s.release([1, 0, 0, 1, 0])
        s.step([90, 1, 1, 0, 1], 200)
        s.step([0, 0, 0, 0, 0], 3)
        s.release([1, 1, 1, 1, 1])
        s.step([200, 0, 0, 0, 0], 200)
        s.step([17, 33, 1, 15, 64], 150)
    finally:
        s.dispose()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_captured_steps_replay_over_growing_requests(device, fmt):
    """One captured decode step, replayed with other inputs, eager steps, synchronizations and a release in between."""
    L, h = nat.lib(), device.handle
    s = Server(device, fmt, 8, 2, 128, 200, 4, 900, 256)
    g = ctypes.c_void_p()
    try:
        s.step([60, 200, 0, 5], 256)
        s.c.reserve(8, 6)
        s.c.reserve(8, 4)
        one = [1, 1, 0, 1]
        s.c.set_new(one)
        nat.check(L.aih_capture_begin(h), "aih_capture_begin")
        s.launch(6)
        nat.check(L.aih_capture_end(h, ctypes.byref(g)), "aih_capture_end")
        for i in range(24):
            x = s.inputs(6)
            nat.check(L.aih_graph_launch(h, g), "aih_graph_launch")
            if i % 5 == 4:
                device.synchronize()
            s.follow(one, 6, x)
            if i == 9:                              # an eager chunk, then the requests go on by replays
                s.step([0, 37, 0, 0], 64)
                s.c.set_new(one)
            if i == 15:
                s.release([0, 0, 0, 1])
                s.step([0, 0, 70, 0], 80)
                one = [1, 1, 1, 1]
                s.c.set_new(one)
    finally:
        if g:
            L.aih_graph_destroy(g)
        s.dispose()


def test_two_contexts_at_once(device):
    """Two contexts (two streams) with a pool each run side by side and give what each gives alone."""
    from aihost_amd.compute import HipComputeDevice
    other = HipComputeDevice(0)
    servers = []
    try:
        for dev, fmt in ((device, "int8"), (other, "e4m3")):
            servers.append(Server(dev, fmt, 8, 4, 128, 60, 3, 400, 300))
        plans = [([100, 30, 170], 300), ([1, 1, 1], 3), ([9, 1, 1], 12)]
        for n_new, rows in plans:
            x = []
            for s in servers:
                x.append(s.inputs(rows))
                s.c.set_new(n_new)
            for s in servers:
                s.launch(rows)
            for s, y in zip(servers, x):
                s.follow(n_new, rows, y)
    finally:
        for s in servers:
            s.dispose()
        other.dispose()


def test_cache_past_4_gib(device):
    """Blocks that lie beyond 32-bit byte offsets (9 GiB of keys and of values)."""
    kv, dim, block, n = 8, 128, 64, 147456
    c = PagedKvCache(device, 1, kv, dim, n, 2, 4096, 4096, "int8", block)
    try:
        rng = np.random.default_rng(3)
        # the stack's end: the pool's highest blocks first for request 0, its lowest for request 1
        order = np.arange(n)
        order[-3:], order[-6:-3] = [0, 1, 2], [n - 1, n - 2, n - 3]
        c._put(c.free_blocks, order[np.r_[0:n - 6, n - 3:n, n - 6:n - 3]])
        rows = 300
        x = [rng.standard_normal((rows, h, dim)).astype(np.float32) for h in (8, kv, kv)]
        bufs = [upload(device, a) for a in x] + [device.create_buffer(rows * 8 * dim * 4)]
        p = [b.get_pointer() for b in bufs]
        c.plan([150, 150], rows)
        c.append(0, p[1], kv * dim, p[2], kv * dim)
        c.attention(0, p[0], 8 * dim, p[3], 8 * dim, 8, 0.1)
        got = bufs[3].read_range(0, rows * 8 * dim, np.float32).reshape(rows, 8, dim)
        assert c._get(c.tables, 2)[0] > n - 10
        ref = R.Cache(R.INT8, kv, dim, block, 6)
        tables = np.array([[0, 1, 2], [3, 4, 5]])
        ref.append(x[1], x[2], [i if i < 150 else 3 * block + i - 150 for i in range(rows)])
        want, bound = R.attention(ref, x[0], [0, 150, 300], [150, 150], tables, 0.1)
        assert np.all(np.abs(got - want).max(-1) <= bound)
        keys, values = c.read(0, 0)
        np.testing.assert_array_equal(keys, ref.values()[0][:150].reshape(150, -1).astype(np.float32))
        np.testing.assert_array_equal(values, ref.values()[1][:150].reshape(150, -1).astype(np.float32))
        for b in bufs:
            b.dispose()
    finally:
        c.dispose()
