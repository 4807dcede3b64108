"""The operators of the paged 8-bit key/value cache, as cases to be measured.

A server of several requests keeps their keys and values in blocks of tokens
that a pool hands out, one byte per value and one fp32 scale per block and KV
head.  Kinds of case:

  plan     aih_kv_plan: block tables, slot maps, row starts and positions of
           the next step's rows, from the requests' lengths
  append   aih_kv_append of a step's key and value rows, and aih_kv_read of
           what their blocks then hold
  attend   aih_kv_attention over the cache: single tokens, prompts, chunks of
           a long prompt, with capped scores, a distance bias, a prefix mask
           or a sliding window

listed() names the ones that are always looked at, draw() gives others of the
same ranges.  With `own` false, run() computes the operators with elementary
torch operations in 32 bits (the codes' quotients, which decide a rounding, in
64); with `own` true it makes the library's calls.  exact() follows the
definitions in 64 bits.

The cache's layout is the one of include/aihost_hip.h.  A block of one head
holds its tokens in groups of 16.  Keys: byte i of 16-byte unit ((t C + c) 4 +
r) 4 + g of a group is the code of token 4 t + r at dimension 64 c + 16 g + i,
C = head_dim / 64.  Values: byte i of unit d is the code of token i at
dimension d.
"""
import math
import random

import torch

own = False

MOST = {"int8": 127.0, "e4m3": 448.0}   # the largest code
TINY = 2.0 ** -126                       # the smallest scale


# ---- the cases ---------------------------------------------------------------
def listed():
    return [
        # the step of a full decode batch: one token each, most requests inside a block
        {"name": "plan_decode_64", "kind": "plan", "seqs": 64, "new": 1, "past": 4000, "block": 16, "pick": 1},
        # many prompts admitted at once, some requests idle
        {"name": "plan_prompts_256", "kind": "plan", "seqs": 256, "new": 512, "past": 2000, "block": 32, "pick": 2},
        # the keys and values of one decode step of 32 requests
        {"name": "append_decode_32_int8", "kind": "append", "format": "int8", "seqs": 32, "new": 1, "past": 1000,
         "kv": 8, "dim": 128, "block": 16, "pick": 3},
        # one layer's rows of several prompts, odd lengths, the last blocks part filled
        {"name": "append_prompts_e4m3", "kind": "append", "format": "e4m3", "seqs": 12, "new": 1500, "past": 0,
         "kv": 8, "dim": 128, "block": 32, "pick": 4},
        # one conversation's next token: latency
        {"name": "decode_1_at_513_int8", "kind": "attend", "format": "int8", "seqs": 1, "new": 1, "past": 512,
         "heads": 32, "kv": 8, "dim": 128, "block": 16, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0,
         "pick": 0},
        # a full decode batch, requests of very different lengths
        {"name": "decode_64_ragged_int8", "kind": "attend", "format": "int8", "seqs": 64, "new": 1, "past": 8192,
         "heads": 32, "kv": 8, "dim": 128, "block": 16, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0,
         "pick": 5},
        # wide heads with capped scores that look at a window of 4096 tokens
        {"name": "decode_16_capped_d256_e4m3", "kind": "attend", "format": "e4m3", "seqs": 16, "new": 1,
         "past": 8000, "heads": 16, "kv": 8, "dim": 256, "block": 32, "cap": 50.0, "slopes": False, "window": 4096,
         "prefix": 0, "pick": 6},
        # narrow heads, no grouping, positions by a distance bias; the last drafted tokens of each request at once
        {"name": "draft_16x4_bias_d64_int8", "kind": "attend", "format": "int8", "seqs": 16, "new": 4, "past": 3000,
         "heads": 16, "kv": 16, "dim": 64, "block": 16, "cap": 0.0, "slopes": True, "window": 0, "prefix": 0,
         "pick": 7},
        # the benchmark's prompt
        {"name": "prompt_512_int8", "kind": "attend", "format": "int8", "seqs": 1, "new": 512, "past": 0,
         "heads": 32, "kv": 8, "dim": 128, "block": 32, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0,
         "pick": 0},
        # several long prompts, odd lengths
        {"name": "prompts_ragged_e4m3", "kind": "attend", "format": "e4m3", "seqs": 4, "new": 4096, "past": 0,
         "heads": 32, "kv": 8, "dim": 128, "block": 32, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0,
         "pick": 8},
        # prompts whose first part (an image, an instruction) is seen whole, scores capped
        {"name": "prompts_prefix_capped_int8", "kind": "attend", "format": "int8", "seqs": 3, "new": 1100, "past": 0,
         "heads": 16, "kv": 4, "dim": 128, "block": 16, "cap": 30.0, "slopes": False, "window": 0, "prefix": 300,
         "pick": 9},
        # a piece of a long document behind 16000 tokens already read
        {"name": "chunk_200_at_16000_int8", "kind": "attend", "format": "int8", "seqs": 1, "new": 200, "past": 16000,
         "heads": 32, "kv": 8, "dim": 128, "block": 64, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0,
         "pick": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["plan", "append", "attend", "attend"], [1, 1, 2, 2])[0]
    block, pick = rng.choice([16, 32, 64]), rng.randint(1, 10 ** 6)
    if kind == "plan":
        new = rng.choice([1, _log(rng, 2, 512)])
        return {"kind": kind, "seqs": _log(rng, 1, 256), "new": new, "past": _log(rng, 1, 8000), "block": block,
                "pick": pick}
    fmt, dim = rng.choice(["int8", "e4m3"]), rng.choice([64, 128, 128, 256])
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 1500)])
        seqs = _log(rng, 1, 128) if new == 1 else _log(rng, 1, max(2, 12000 // new))
        return {"kind": kind, "format": fmt, "seqs": min(seqs, 128), "new": new,
                "past": rng.choice([0, _log(rng, 1, 500)]), "kv": rng.choice([1, 2, 4, 8]), "dim": dim,
                "block": block, "pick": pick}
    group, kv = rng.choice([1, 2, 4, 4, 5, 8]), rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "format": fmt, "heads": kv * group, "kv": kv, "dim": dim, "block": block,
            "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "slopes": rng.random() < 0.25,
            "window": rng.choice([0, 0, _log(rng, 64, 4096)]), "prefix": 0, "pick": pick}
    how = rng.choice(["token", "token", "few", "prompt", "prompt", "chunk"])
    if how == "token":
        past = _log(rng, 1, 8000)
        return dict(case, seqs=min(64, _log(rng, 1, max(2, 200000 // past))), new=1, past=past)
    if how == "few":
        return dict(case, seqs=_log(rng, 1, 32), new=rng.randint(2, 12), past=_log(rng, 1, 5000))
    if how == "prompt":
        new = _log(rng, 9, 2500)
        return dict(case, seqs=min(8, _log(rng, 1, max(2, 5000 // new))), new=new, past=0,
                    prefix=rng.choice([0, 0, rng.randint(1, new)]))
    return dict(case, seqs=1, new=_log(rng, 16, 400), past=_log(rng, 500, 16000))


def _lengths(case):
    """Cached tokens before the step and new ones, for each request: as given
    where pick is 0, spread below that by it otherwise."""
    n, past, new = case["seqs"], case["past"], case["new"]
    if case["pick"] == 0:
        return [past] * n, [new] * n
    rng = random.Random(case["pick"])
    old = [min(past, _log(rng, max(1, past // 16), past + 1)) if past else 0 for _ in range(n)]
    if new == 1:
        return old, [1] * n
    if case["kind"] == "attend" and past:
        return old, [new] * n
    fresh = [min(new, _log(rng, max(1, new // 16), new + 1)) for _ in range(n)]
    if case["kind"] == "plan":      # every eighth request has nothing to add
        fresh = [0 if s % 8 == 5 else f for s, f in enumerate(fresh)]
    return old, fresh


def _blocks(tokens, block):
    return -(-tokens // block)


# ---- the cache in plain torch ---------------------------------------------------
def _values(codes, fmt):
    """Codes (uint8) as the numbers they stand for, before the scale."""
    return codes.view(torch.int8).float() if fmt == "int8" else codes.view(torch.float8_e4m3fn).float()


def _codes(x, fmt):
    """Numbers within the format's range to codes, to nearest, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.float().to(torch.float8_e4m3fn).view(torch.uint8)


def _keys_out(k, dim):
    """Stored key blocks (n, kv, block * dim) -> (n, block, kv, dim)."""
    n, kv = k.shape[:2]
    t = k.reshape(n, kv, -1, 4, dim // 64, 4, 4, 16)         # group, t, c, r, g, i
    return t.permute(0, 2, 3, 5, 1, 4, 6, 7).reshape(n, -1, kv, dim)


def _keys_in(x):
    n, block, kv, dim = x.shape
    t = x.reshape(n, block // 16, 4, 4, kv, dim // 64, 4, 16)  # group, t, r, head, c, g, i
    return t.permute(0, 4, 1, 2, 5, 3, 6, 7).reshape(n, kv, block * dim)


def _vals_out(v, dim):
    """Stored value blocks (n, kv, block * dim) -> (n, block, kv, dim)."""
    n, kv = v.shape[:2]
    return v.reshape(n, kv, -1, dim, 16).permute(0, 2, 4, 1, 3).reshape(n, -1, kv, dim)


def _vals_in(x):
    n, block, kv, dim = x.shape
    return x.reshape(n, block // 16, 16, kv, dim).permute(0, 3, 1, 4, 2).reshape(n, kv, block * dim)


def _first_scale(top, fmt):
    """The scale of a block whose largest magnitude is `top` (0 for none)."""
    if fmt == "int8":
        s = (top.double() / 127).float().clamp_min(TINY)
    else:
        m, e = torch.frexp(top.double())                      # top = m 2^e, 448 = 0.875 * 2^9
        k = (e - torch.where(m <= 0.875, 9, 8)).clamp_min(-126)
        s = torch.ldexp(torch.ones_like(top.double()), k).float()
    return torch.where(top == 0, torch.zeros_like(top), s)


def _grown(top, old, fmt):
    """How many times a block's scale `old` is doubled to hold `top`."""
    m, e = torch.frexp(top.double() / (MOST[fmt] * old.double()).clamp_min(1e-300))
    return torch.where(old > 0, torch.where(m > 0.5, e, e - 1).clamp_min(0), 0)


class _State:
    """What a program holds."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


# ---- inputs ----------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(old, after, block, spare, gen):
    """Block tables of requests that hold `old` tokens, and the pool's free
    blocks (their ids in `free`, the last one first to go): blocks for `after`
    tokens and `spare` more, in random order."""
    width = max(1, max(_blocks(a, block) for a in after))
    pool = sum(_blocks(a, block) for a in after) + spare
    ids = torch.randperm(pool, generator=gen).tolist()
    tables, at = [], 0
    for o in old:
        b = _blocks(o, block)
        tables.append(ids[at:at + b] + [-1] * (width - b))
        at += b
    return _ints(tables), ids[at:], pool, width


def _inputs(case, seed):
    """Every input of a case; prepare() and exact() both start here."""
    host = torch.Generator().manual_seed(int(seed) * 7919 + 17)
    make = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 18)
    old, new = _lengths(case)
    after = [o + n for o, n in zip(old, new)]
    block = case["block"]
    if case["kind"] == "plan":
        tables, free, pool, width = _tables(old, after, block, 7, host)
        d = _State(lens=_ints(old), new=_ints(new), tables=tables, pool=pool, width=width, n_free=_ints([len(free)]),
                   free=_ints(free + [-1] * (pool - len(free))), rows=sum(new) + 3)
        return d

    # as a plan leaves them: every request's blocks handed out
    tables, _, pool, width = _tables(after, after, block, 3, host)
    rows, kv, dim, fmt = sum(new), case["kv"], case["dim"], case["format"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    d = _State(lens=_ints(after), starts=_ints(starts), tables=tables, pool=pool, width=width, rows=rows)

    def normal(*shape):
        return torch.randn(*shape, generator=make, device="cuda", dtype=torch.float32)

    if case["kind"] == "append":
        seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
        pos = torch.arange(rows) - torch.tensor(starts)[seq] + torch.tensor(old)[seq]
        t = tables.cpu().long()
        slots = t[seq, pos // block] * block + pos % block
        d.slots = slots.to(torch.int32).cuda()
        # what the touched blocks hold in the end, in token order
        first = [o // block * block for o in old]
        seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor([a - f for a, f in zip(after, first)]))
        pos = torch.cat([torch.arange(f, a) for f, a in zip(first, after)])
        d.held = (t[seq, pos // block] * block + pos % block).to(torch.int32).cuda()
        # the blocks' earlier tokens; rows of keys and values, one channel of eight larger as keys have it
        grow = 1.0 + 3.0 * (torch.arange(dim, device="cuda") % 8 == 0).float()
        d.k, d.v = normal(rows, kv, dim) * grow, normal(rows, kv, dim)
        past = {"k": normal(pool, block, kv, dim) * grow, "v": normal(pool, block, kv, dim)}
        keep = torch.zeros(pool, dtype=torch.long)
        for s, o in enumerate(old):
            if o % block:
                keep[t[s, o // block]] = o % block
        inside = (torch.arange(block)[None, :] < keep[:, None]).cuda()[:, :, None, None]
        for name, lay in (("k", _keys_in), ("v", _vals_in)):
            x = torch.where(inside, past[name], torch.zeros_like(past[name]))
            scale = _first_scale(x.abs().amax((1, 3)), fmt)
            c = _codes(x.double() / scale.double().clamp_min(1e-300)[:, None, :, None], fmt)
            d.__dict__[name + "_codes"] = lay(c).contiguous()
            d.__dict__[name + "_scale"] = scale.contiguous()
        return d

    heads = case["heads"]
    d.q = normal(rows, heads * dim) * (4.0 if case["cap"] else 1.0)
    for name in "kv":
        c = normal(pool, kv, block * dim)
        c = _codes(torch.round(c * 36).clamp(-127, 127), "int8") if fmt == "int8" else _codes((c * 110).clamp(-448, 448), fmt)
        # a block's largest value is 3 to 4.5 standard deviations
        s = torch.rand(pool, kv, generator=make, device="cuda") * 1.5 + 3
        d.__dict__[name + "_codes"] = c
        d.__dict__[name + "_scale"] = s / 127 if fmt == "int8" else s / 448
    d.scale = 1.0 / math.sqrt(dim)
    d.cap, d.window = float(case["cap"]), int(case["window"])
    d.slopes = None
    if case["slopes"]:
        d.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")
    # every other request has a prefix that is seen whole
    d.prefix = _ints([min(case["prefix"], n) if s % 2 == 0 else 0 for s, n in enumerate(new)]) if case["prefix"] else None
    return d


def prepare(case, seed):
    s = _inputs(case, seed)
    s.case = dict(case)
    empty = {"device": "cuda", "dtype": torch.int32}
    if case["kind"] == "plan":
        s.new_lens, s.new_n_free = torch.zeros_like(s.lens), torch.zeros_like(s.n_free)
        s.starts = torch.zeros(len(s.lens) + 1, **empty)
        s.slots, s.positions = torch.zeros(s.rows, **empty), torch.zeros(s.rows, **empty)
        s.refused = torch.zeros(1, **empty)
    elif case["kind"] == "append":
        shape = (len(s.held), case["kv"], case["dim"])
        s.k_held, s.v_held = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    else:
        s.o = torch.zeros_like(s.q)
    return s


# ---- one pass ----------------------------------------------------------------------
def run(s):
    kind = s.case["kind"]
    if own:
        return _own_run(s)
    return _plan(s) if kind == "plan" else _append(s) if kind == "append" else _attend(s)


def _plan(s):
    block = s.case["block"]
    lens, new, n_free = s.lens.long(), s.new.long(), s.n_free.long()
    valid = (lens >= 0) & (new >= 0) & (lens + new <= s.width * block)
    new = torch.where(valid, new, 0)
    had = (lens + block - 1) // block
    need = torch.where(valid, (lens + new + block - 1) // block - had, 0)
    upto = torch.cumsum(need, 0)
    ok = valid & ((new == 0) | (((need == 0) | (upto <= n_free)) & (torch.cumsum(new, 0) <= s.rows)))
    new, need = torch.where(ok, new, 0), torch.where(ok, need, 0)
    first = upto - need                                     # of the blocks handed out in order
    j = torch.arange(s.width, device="cuda")[None, :] - had[:, None]
    take = (j >= 0) & (j < need[:, None])
    at = (n_free - 1 - first[:, None] - j).clamp(0, len(s.free) - 1)
    s.tables.copy_(torch.where(take, s.free[at], s.tables))
    ends = torch.cumsum(new, 0)
    s.starts[0] = 0
    s.starts[1:] = ends.to(torch.int32)
    row = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(ends, row, right=True).clamp_max(len(lens) - 1)
    pos = lens[seq] + row - (ends - new)[seq]
    inside = row < ends[-1]
    entry = s.tables[seq, (pos // block).clamp(0, s.width - 1)].long()
    held = inside & (entry >= 0) & (entry < s.pool)
    s.slots.copy_(torch.where(held, entry * block + pos % block, -1))
    s.positions.copy_(torch.where(inside, pos, -1))
    s.new_lens.copy_(lens + new)
    s.new_n_free.copy_(n_free - need.sum())
    s.refused.copy_((~ok).sum().reshape(1))
    return _plan_out(s)


def _plan_out(s):
    return {"tables": s.tables, "lens": s.new_lens, "free": s.new_n_free, "starts": s.starts, "slots": s.slots,
            "positions": s.positions, "refused": s.refused}


def _append(s):
    fmt, block, dim = s.case["format"], s.case["block"], s.case["dim"]
    slots, held = s.slots.long(), s.held.long()
    b, o = slots // block, slots % block
    fresh = torch.zeros(s.pool, device="cuda").index_put((b,), (o == 0).float(), accumulate=True) > 0
    out = {}
    for name, x, codes, scale, lay, take in (("k", s.k, s.k_codes, s.k_scale, _keys_in, _keys_out),
                                             ("v", s.v, s.v_codes, s.v_scale, _vals_in, _vals_out)):
        kv = x.shape[1]
        top = torch.zeros(s.pool, kv, device="cuda").scatter_reduce(0, b[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
        old = torch.where(fresh[:, None], torch.zeros_like(scale), scale)
        d = _grown(top, old, fmt)
        now = torch.where(old > 0, torch.ldexp(old, d), _first_scale(top, fmt))
        c = torch.where(fresh[:, None, None, None], 0.0, _values(take(codes, dim), fmt))
        c = _codes(torch.ldexp(c, -d[:, None, :, None]), fmt)
        c[b, o] = _codes(x.double() / now[b].double().clamp_min(1e-300)[..., None], fmt)
        codes.copy_(lay(c))
        scale.copy_(now)
        out[name] = _values(c[held // block, held % block], fmt) * now[held // block][..., None]
        out[name + "_scale"] = scale
    return out


def _attend(s):
    c = s.case
    heads, kv, dim, block, fmt = c["heads"], c["kv"], c["dim"], c["block"], c["format"]
    n_seqs, group, most = c["seqs"], heads // kv, c["new"]
    lens, starts = s.lens.long(), s.starts.long()
    new = starts[1:] - starts[:-1]
    at = s.tables.long().clamp_min(0)
    length = s.width * block

    def cache(codes, scale, lay):
        x = _values(lay(codes[at.reshape(-1)], dim), fmt) * scale[at.reshape(-1)][:, None, :, None]
        return x.reshape(n_seqs, length, kv, dim)

    i = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + i[None, :]).clamp_max(s.rows - 1)            # (request, i)
    q = s.q[row].reshape(n_seqs, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n_seqs, kv, most * group, dim)
    k = cache(s.k_codes, s.k_scale, _keys_out).permute(0, 2, 3, 1).contiguous()
    t = (torch.matmul(q, k) * s.scale).reshape(n_seqs, kv, most, group, length)
    if s.cap:
        t = s.cap * torch.tanh(t / s.cap)
    p = (lens - new)[:, None] + i[None, :]                                   # (request, i)
    j = torch.arange(length, device="cuda")
    if s.slopes is not None:
        far = (p[:, :, None] - j).abs().float()                              # (request, i, key)
        t = t - s.slopes.reshape(1, kv, 1, group, 1) * far[:, None, :, None, :]
    end = p + 1 if s.prefix is None else torch.maximum(p + 1, s.prefix.long()[:, None])
    seen = (j < torch.minimum(end, lens[:, None])[:, :, None])
    if s.window:
        seen = seen & (j > (p - s.window)[:, :, None])
    t = t.masked_fill(~seen[:, None, :, None, :], -math.inf)
    w = torch.exp(t - t.amax(-1, keepdim=True).clamp_min(-1e30))
    w = (w / w.sum(-1, keepdim=True).clamp_min(1e-30)).reshape(n_seqs, kv, most * group, length)
    o = torch.matmul(w, cache(s.v_codes, s.v_scale, _vals_out).permute(0, 2, 1, 3).contiguous())
    o = o.reshape(n_seqs, kv, most, group, dim).permute(0, 2, 1, 3, 4).reshape(n_seqs * most, heads * dim)
    # the rows in their order: row r is number r - starts of its request
    r = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True).clamp_max(n_seqs - 1)
    s.o.copy_(o[seq * most + r - starts[seq]])
    return s.o


# ---- the library's calls --------------------------------------------------------------
_device = None


def _bind(s):
    """The calls of a pass with their arguments, as a program keeps them."""
    global _device
    import ctypes

    from aihost_amd import _native as nat
    from aihost_amd import compute
    if _device is None:
        _device = compute.HipComputeDevice(0)
    h, L, c = _device.handle, nat.lib(), s.case
    if c["kind"] == "plan":
        return [(L.aih_kv_plan, (h, s.lens.data_ptr(), s.new.data_ptr(), c["seqs"], s.tables.data_ptr(), s.width,
                                 c["block"], s.pool, s.free.data_ptr(), s.n_free.data_ptr(), s.new_lens.data_ptr(),
                                 s.new_n_free.data_ptr(), s.starts.data_ptr(), s.slots.data_ptr(),
                                 s.positions.data_ptr(), s.rows, s.refused.data_ptr()))]
    s.cache = nat.KvCache(format=nat.KV_INT8 if c["format"] == "int8" else nat.KV_E4M3, n_kv_heads=c["kv"],
                          head_dim=c["dim"], block_tokens=c["block"], n_blocks=s.pool, k=s.k_codes.data_ptr(),
                          v=s.v_codes.data_ptr(), k_scale=s.k_scale.data_ptr(), v_scale=s.v_scale.data_ptr())
    cache, wide = ctypes.byref(s.cache), c["kv"] * c["dim"]
    if c["kind"] == "append":
        return [(L.aih_kv_append, (h, cache, s.k.data_ptr(), wide, s.v.data_ptr(), wide, s.slots.data_ptr(), s.rows)),
                (L.aih_kv_read, (h, cache, s.held.data_ptr(), len(s.held), s.k_held.data_ptr(), wide,
                                 s.v_held.data_ptr(), wide))]
    floats = nat.check_size(L.aih_kv_attention_scratch_floats(h, cache, c["heads"], s.rows, c["seqs"], s.width),
                            "aih_kv_attention_scratch_floats")
    s.scratch = torch.zeros(max(4, floats), device="cuda")
    s.scores = nat.KvScores(cap=s.cap, window=s.window, slopes=s.slopes.data_ptr() if s.slopes is not None else None,
                            prefix=s.prefix.data_ptr() if s.prefix is not None else None)
    row = c["heads"] * c["dim"]
    return [(L.aih_kv_attention, (h, cache, s.q.data_ptr(), row, s.o.data_ptr(), row, s.rows, c["heads"], c["seqs"],
                                  s.starts.data_ptr(), s.lens.data_ptr(), s.tables.data_ptr(), s.width, s.scale,
                                  ctypes.byref(s.scores), s.scratch.data_ptr(), floats))]


def _own_run(s):
    calls = s.__dict__.get("calls")
    if calls is None:
        calls = s.calls = _bind(s)
        # the library has a stream of its own, which does not wait for torch's: what prepare queued has to be there first.
        # (The outputs are on that stream too; who reads them with torch waits for the device before.)
        torch.cuda.synchronize()
    for f, a in calls:
        status = f(*a)
        if status:
            raise RuntimeError("%s: status %d" % (f.__name__, status))
    if s.case["kind"] == "plan":
        return _plan_out(s)
    if s.case["kind"] == "append":
        return {"k": s.k_held, "k_scale": s.k_scale, "v": s.v_held, "v_scale": s.v_scale}
    return s.o


# ---- what a pass cannot do without -------------------------------------------------
def _seen(case):
    """(query, key) pairs that are looked at, and the cached tokens read, over all requests."""
    pairs = tokens = 0
    for s, (o, n) in enumerate(zip(*_lengths(case))):
        prefix = min(case["prefix"], n) if s % 2 == 0 else 0
        window, low = case["window"], o + n
        for p in (range(o, o + n)):
            a = max(0, p - window + 1) if window else 0
            pairs += max(p + 1, prefix) - a
            low = min(low, a)
        tokens += o + n - low
    return pairs, tokens


def work(case):
    old, new = _lengths(case)
    block = case["block"]
    if case["kind"] == "plan":
        taken = sum(_blocks(o + n, block) - _blocks(o, block) for o, n in zip(old, new))
        width = max(_blocks(o + n, block) for o, n in zip(old, new))
        ints = 5 * len(old) + 2 * taken + 2 * (sum(new) + 3)
        return {"bytes": 4 * ints, "flops": 10 * len(old) + 4 * sum(new) + width}
    wide = case["kv"] * case["dim"]
    if case["kind"] == "append":
        rows = sum(new)
        held = sum(o + n - o // block * block for o, n in zip(old, new))
        scales = sum(_blocks(o + n, block) - o // block for o, n in zip(old, new)) * case["kv"]
        # rows in, their codes and scales out; then codes and scales in, values out
        return {"bytes": 2 * (rows * wide * 5 + held * wide * 5 + 3 * 4 * scales) + 4 * (rows + held),
                "flops": 2 * (rows * wide * 4 + held * wide)}
    pairs, tokens = _seen(case)
    rows = sum(new)
    return {"bytes": 2 * tokens * wide + 8 * rows * case["heads"] * case["dim"] + 8 * tokens // block * case["kv"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- the same in 64 bits, from the definitions -------------------------------------
def _byte_at(token, head, d, block, dim, kv, keys):
    """Index of the code of `token` (slot number), `head`, dimension d."""
    b, o = token // block, token % block
    base = (b * kv + head) * block * dim + o // 16 * 16 * dim
    o = o % 16
    if keys:
        unit = ((o // 4 * (dim // 64) + d // 64) * 4 + o % 4) * 4 + d % 64 // 16
        return base + unit * 16 + d % 16
    return base + d * 16 + o


def _rows64(codes, scale, slots, case, keys):
    """The values at `slots` in 64 bits: (len(slots), kv, dim)."""
    block, dim, kv = case["block"], case["dim"], case["kv"]
    at = _byte_at(slots[:, None, None], torch.arange(kv, device="cuda")[None, :, None],
                  torch.arange(dim, device="cuda")[None, None, :], block, dim, kv, keys)
    c = codes.reshape(-1)[at]
    c = c.view(torch.int8).double() if case["format"] == "int8" else c.view(torch.float8_e4m3fn).double()
    return c * scale.double()[slots // block][:, :, None]


def _exact_append(d, case):
    """Block by block: what its tokens are, then the rule for the scale."""
    block, fmt = case["block"], case["format"]
    old, new = _lengths(case)
    tables = d.tables.cpu().long()
    out = {"k": [], "v": []}
    scales = {"k": d.k_scale.double().clone(), "v": d.v_scale.double().clone()}
    first_row = 0
    for s, (o, n) in enumerate(zip(old, new)):
        for name, x in (("k", d.k), ("v", d.v)):
            at = o
            while at < o + n:
                b, start = int(tables[s, at // block]), at // block * block
                end = min(start + block, o + n)
                rows = x[first_row + at - o:first_row + end - o].double()
                top = rows.abs().amax((0, 2))
                scale, codes = scales[name][b], d.__dict__[name + "_codes"]
                if at == start:
                    scale, before = torch.zeros_like(scale), rows[:0]
                else:
                    slots = b * block + torch.arange(at - start, device="cuda")
                    before = _rows64(codes, d.__dict__[name + "_scale"], slots, case, name == "k") / scale.clamp_min(1e-300)[None, :, None]
                most = MOST[fmt]
                if fmt == "int8":
                    begin = torch.clamp((top / 127).float().double(), min=TINY)
                else:
                    begin = torch.clamp(2.0 ** torch.ceil(torch.log2(top.clamp_min(1e-300) / 448)), min=TINY)
                begin = torch.where(top > 0, begin, torch.zeros_like(top))
                up = torch.clamp(torch.ceil(torch.log2((top / (most * scale.clamp_min(1e-300))).clamp_min(1e-300))), min=0)
                up = torch.where(scale > 0, up, torch.zeros_like(up))
                now = torch.where(scale > 0, scale * 2.0 ** up, begin)
                c = torch.cat([before * 2.0 ** -up[None, :, None], rows / now.clamp_min(1e-300)[None, :, None]])
                c = torch.round(c).clamp(-127, 127) if fmt == "int8" else c.to(torch.float8_e4m3fn).double()
                out[name].append(c * now[None, :, None])
                scales[name][b] = now
                at = end
        first_row += n
    return {"k": torch.cat(out["k"]), "k_scale": scales["k"], "v": torch.cat(out["v"]), "v_scale": scales["v"]}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "plan":
        return None
    if case["kind"] == "append":
        return _exact_append(d, case)
    heads, kv, dim, block = case["heads"], case["kv"], case["dim"], case["block"]
    group = heads // kv
    old, new = _lengths(case)
    out = torch.empty(d.rows, heads, dim, device="cuda", dtype=torch.float64)
    first_row = 0
    for s, (o, n) in enumerate(zip(old, new)):
        j = torch.arange(o + n, device="cuda")
        slots = d.tables[s].long()[j // block] * block + j % block
        k, v = (_rows64(c, sc, slots, case, keys) for c, sc, keys in ((d.k_codes, d.k_scale, True), (d.v_codes, d.v_scale, False)))
        p = torch.arange(o, o + n, device="cuda")
        end = p + 1
        if d.prefix is not None:
            end = torch.clamp(end, min=int(d.prefix[s]))
        hidden = j[None, :] >= end[:, None]
        if d.window:
            hidden |= j[None, :] <= (p - d.window)[:, None]
        q = d.q[first_row:first_row + n].double().reshape(n, heads, dim)
        for h in range(heads):
            t = q[:, h].contiguous() @ k[:, h // group].T.contiguous() * d.scale
            if d.cap:
                t = d.cap * torch.tanh(t / d.cap)
            if d.slopes is not None:
                t = t - d.slopes[h].double() * (p[:, None] - j[None, :]).abs()
            out[first_row:first_row + n, h] = torch.softmax(t.masked_fill(hidden, -math.inf), -1) @ v[:, h // group].contiguous()
        first_row += n
    return out.reshape(d.rows, heads * dim)
