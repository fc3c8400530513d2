"""The operators of decoding over a quantised block cache, as cases that can be
timed and compared: norms of query and key heads with rotary positions of
several axes, the quantised cache write, reading rows back, and attention of
one new token a request with capped scores, distance biases, windows and
documents.

``listed()`` holds representative cases, ``draw`` gives others of the same
ranges, ``prepare`` makes what a program has in hand before the call, ``run``
is one pass, ``work`` the bytes and operations that a pass cannot do without
and ``exact`` the same outputs in float64.  With ``own`` false ``run`` computes
the plain form in torch, with ``own`` true it calls this package.

Sizes: the 4B-shaped model of ``runtime.ModelConfig`` (32 query heads of 128,
8 KV groups, 32 rotary dims), the batches of its benchmark (up to 128 rows, 256
in the long horizon), and caches of 16- to 64-token blocks.

A quantised cache keeps a row's values in runs of 32 that share a power of two
2^(s - 127), the smallest at which none of them is past the largest code (448
of e4m3, 6 of e2m1; s is at least 16): keys and values [blocks, G, block, D] in
float8_e4m3fn, or [blocks, G, block, D / 2] bytes of two e2m1 codes, the even
dim in the low half; scales s [blocks, G, D / 32, block] bytes.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROW = {"bf16": 2.0, "fp16": 2.0, "fp8": 1.0 + 1 / 32, "fp4": 0.5 + 1 / 32}     # bytes of a cached value
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one interactive session's token: the latency of a call
        {"name": "rope_b1", "kind": "rope", "tokens": 1, "h": 32, "g": 8, "d": 128, "rotary": 32, "axes": 1,
         "interleaved": False, "far": 5000, "dtype": "bf16"},
        # a packed prefill of text and images at full rotary width, positions up to a million
        {"name": "rope_prefill_axes", "kind": "rope", "tokens": 65521, "h": 32, "g": 8, "d": 128, "rotary": 128,
         "axes": 3, "interleaved": True, "far": 1000000, "dtype": "bf16"},
        # the serving batch's new tokens, some rows of the captured batch idle, and their rows back
        {"name": "write_b128_fp8", "kind": "write", "tokens": 128, "kept": 0.9, "block": 16, "g": 8, "d": 128,
         "fmt": "fp8", "dtype": "bf16"},
        # the keys and values of a packed prefill, and their rows back
        {"name": "write_prefill_fp4", "kind": "write", "tokens": 65521, "kept": 1.0, "block": 64, "g": 8, "d": 128,
         "fmt": "fp4", "dtype": "bf16"},
        # one request's cached prefix for the prefill that continues it
        {"name": "read_prefix_fp4", "kind": "read", "requests": 1, "len_lo": 777, "len_hi": 777, "block": 16, "g": 8,
         "d": 128, "fmt": "fp4", "dtype": "fp16"},
        # the prefixes of a refill
        {"name": "read_refill_fp8", "kind": "read", "requests": 16, "len_lo": 1000, "len_hi": 32768, "block": 64,
         "g": 8, "d": 128, "fmt": "fp8", "dtype": "bf16"},
        # one interactive session: the latency of a call
        {"name": "attn_b1_fp8", "kind": "attn", "requests": 1, "idle": 0, "len_lo": 5000, "len_hi": 5000, "block": 16,
         "window": 0, "doc": 0.0, "cap": 0.0, "slopes": False, "gate": True, "h": 32, "g": 8, "d": 128, "fmt": "fp8",
         "dtype": "bf16"},
        # the serving batch, gated as the model's attention, capped scores, some rows of the captured batch idle
        {"name": "attn_b128_fp8", "kind": "attn", "requests": 128, "idle": 5, "len_lo": 200, "len_hi": 20000,
         "block": 16, "window": 0, "doc": 0.0, "cap": 50.0, "slopes": False, "gate": True, "h": 32, "g": 8, "d": 128,
         "fmt": "fp8", "dtype": "bf16"},
        # four-bit caches, very ragged contexts
        {"name": "attn_b64_fp4", "kind": "attn", "requests": 64, "idle": 0, "len_lo": 37, "len_hi": 65536, "block": 32,
         "window": 0, "doc": 0.0, "cap": 0.0, "slopes": False, "gate": False, "h": 32, "g": 8, "d": 128, "fmt": "fp4",
         "dtype": "bf16"},
        # a 16-bit cache with capped scores and a window, heads of 256
        {"name": "attn_b32_window", "kind": "attn", "requests": 32, "idle": 0, "len_lo": 900, "len_hi": 30000,
         "block": 64, "window": 4096, "doc": 0.0, "cap": 30.0, "slopes": False, "gate": False, "h": 16, "g": 8,
         "d": 256, "fmt": "fp16", "dtype": "fp16"},
        # long contexts with a bias that falls with distance
        {"name": "attn_long_b8_fp8", "kind": "attn", "requests": 8, "idle": 0, "len_lo": 30000, "len_hi": 131000,
         "block": 64, "window": 0, "doc": 0.0, "cap": 0.0, "slopes": True, "gate": False, "h": 32, "g": 8, "d": 128,
         "fmt": "fp8", "dtype": "bf16"},
        # packed documents, one key head for many query heads
        {"name": "attn_docs_fp4", "kind": "attn", "requests": 48, "idle": 3, "len_lo": 1, "len_hi": 40000, "block": 16,
         "window": 0, "doc": 0.3, "cap": 0.0, "slopes": False, "gate": False, "h": 20, "g": 1, "d": 64, "fmt": "fp4",
         "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return a, b


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "attn", "attn", "attn"])
    if kind == "rope":
        d = rng.choice([64, 128, 128, 256])
        g = rng.choice([1, 2, 5, 8])
        h = g * rng.choice([1, 3, 4])
        most = min(65521, 65521 * 40 * 128 // ((h + g) * d))
        return {"kind": kind, "tokens": _log(rng, 1, most), "h": h, "g": g, "d": d,
                "rotary": rng.choice([16, 32, d // 2, 3 * d // 4, d]), "axes": rng.choice([1, 2, 3, 3, 4]),
                "interleaved": rng.random() < 0.5, "far": _log(rng, 1, 1000000), "dtype": rng.choice(["bf16", "fp16"])}
    fmt = rng.choice(["fp8", "fp4"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "write":
        d, g = rng.choice([32, 64, 96, 128, 128, 256]), rng.choice([1, 2, 5, 8])
        return {"kind": kind, "tokens": _log(rng, 1, min(65521, 65521 * 1024 // (g * d))),
                "kept": rng.choice([0.2, 0.6, 1.0]), "block": rng.choice([1, 16, 24, 64, 1024]), "g": g, "d": d,
                "fmt": fmt, "dtype": dtype}
    if kind == "read":
        d, g = rng.choice([32, 64, 96, 128, 128, 256]), rng.choice([1, 2, 5, 8])
        n = _log(rng, 1, 64)
        lo, hi = _span(rng, 1, max(1, min(32768, 140000 * 1024 // (n * g * d))))
        return {"kind": kind, "requests": n, "len_lo": lo, "len_hi": hi, "block": rng.choice([1, 16, 24, 64]),
                "g": g, "d": d, "fmt": rng.choice([fmt, fmt, dtype]), "dtype": dtype}
    g = rng.choice([1, 2, 4, 8, 8])
    h = g * rng.choice([1, 2, 3, 4, 4, 7, 8, 20])
    d = rng.choice([64, 128, 128, 256])
    lo, hi = _span(rng, 1, 131000)
    fmt = rng.choice([fmt, fmt, dtype])
    # within the cost of the largest listed case
    most = max(1, min(256, int(5.5e8 // (hi * g * d * max(1, ROW[fmt]))), int(1.7e7 // (hi * h))))
    return {"kind": kind, "requests": _log(rng, 1, most), "idle": rng.choice([0, 0, 1, 3]), "len_lo": lo, "len_hi": hi,
            "block": rng.choice([1, 8, 16, 16, 24, 48, 64, 256]), "window": rng.choice([0, 0, 1, 100, 1000, 4096]),
            "doc": rng.choice([0.0, 0.0, 0.5, 0.9]), "cap": rng.choice([0.0, 0.0, 15.0, 50.0]),
            "slopes": rng.random() < 0.3, "gate": rng.random() < 0.4, "h": h, "g": g, "d": d, "fmt": fmt,
            "dtype": dtype}


# --- inputs -------------------------------------------------------------------

def _spread(lo, hi, n):
    """n sizes from lo to hi, evenly over their logarithm, whatever the seed."""
    if n == 1 or lo == hi:
        return [hi] * n
    return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _quantise(x, fmt):
    """x [..., D] -> (codes [..., D or D / 2], scales s [..., D / 32])."""
    y = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(y.abs().amax(-1))                # m 2^e with m in [1/2, 1)
    top, most = (9, 0.875) if fmt == "fp8" else (3, 0.75)
    s = (e - top + (m > most).to(e.dtype)).clamp_min(-111)
    y = torch.ldexp(y, -s[..., None]).flatten(-2)
    if fmt == "fp8":
        return y.to(torch.float8_e4m3fn), (s + 127).to(torch.uint8)
    a = y.abs()                                         # nearest code, ties to the even one
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = (code + 8 * (y < 0)).to(torch.uint8).unflatten(-1, (-1, 2))
    return code[..., 0] + 16 * code[..., 1], (s + 127).to(torch.uint8)


def _values(codes, scales):
    """Codes [..., D or D / 2] and scales [..., D / 32] -> float32 [..., D]."""
    if codes.dtype == torch.float8_e4m3fn:
        y = codes.float()
    else:
        both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
        y = table[both.int()]
    return torch.ldexp(y.unflatten(-1, (-1, 32)), scales.to(torch.int32)[..., None] - 127).flatten(-2)


class _Make:
    """Seeded inputs: sizes and orders on the host, values on the device."""

    def __init__(self, seed):
        self.dev = "cuda" if torch.cuda.is_available() else "cpu"
        self.host = torch.Generator().manual_seed(int(seed))
        self.gen = torch.Generator(device=self.dev).manual_seed(int(seed) + 1)

    def normal(self, *shape, dtype=torch.bfloat16, std=1.0):
        return (torch.randn(*shape, device=self.dev, generator=self.gen, dtype=torch.float32) * std).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.host)

    def sizes(self, lo, hi, n):
        return torch.tensor(_spread(lo, hi, n), dtype=torch.int64)[self.order(n)]

    def empty(self, blocks, g, block, d, fmt):
        """An empty cache: keys, values and, of a quantised one, their scales."""
        if fmt in DTYPES:
            return [torch.zeros(blocks, g, block, d, dtype=DTYPES[fmt], device=self.dev) for _ in range(2)] + [None] * 2
        shape, dt = ((d,), torch.float8_e4m3fn) if fmt == "fp8" else ((d // 2,), torch.uint8)
        data = [torch.zeros(blocks, g, block, *shape, dtype=torch.uint8, device=self.dev).view(dt) for _ in range(2)]
        return data + [torch.zeros(blocks, g, d // 32, block, dtype=torch.uint8, device=self.dev) for _ in range(2)]

    def cache(self, blocks, g, block, d, fmt):
        """A cache of drawn keys and values, a few channels of the keys larger, as trained ones have them."""
        c = self.empty(blocks, g, block, d, fmt)
        loud = 1 + 3 * (torch.arange(d, device=self.dev) % 37 == 5)
        step = max(1, 2 ** 27 // (g * block * d))
        for i in range(0, blocks, step):
            for which in range(2):
                x = torch.randn(min(step, blocks - i), g, block, d, device=self.dev, generator=self.gen)
                x = x if which else x * loud
                if fmt in DTYPES:
                    c[which][i:i + step] = x.to(DTYPES[fmt])
                else:
                    codes, scales = _quantise(x, fmt)
                    c[which][i:i + step] = codes
                    c[2 + which][i:i + step] = scales.transpose(2, 3)
        return c

    def tables(self, lengths, block):
        """Shuffled blocks for each request: (tables [R, columns], blocks in all)."""
        held = -(-lengths // block)
        blocks, columns = int(held.sum()) + 1, max(1, int(held.max()))
        order, first, c = self.order(blocks), held.cumsum(0) - held, torch.arange(columns)
        tables = torch.full((lengths.numel(), columns), -1, dtype=torch.int64)
        mine = c < held[:, None]
        tables[mine] = order[(first[:, None] + c)[mine]]
        return tables, blocks


def prepare(case, seed):
    m = _Make(seed)
    return {"rope": _prepare_rope, "write": _prepare_write, "read": _prepare_read, "attn": _prepare_attn}[case["kind"]](
        case, m)


def _sections(pairs, axes):
    """Pairs of each axis: the first a little more, as time has in such models."""
    rest = [pairs // axes - (1 if pairs // axes > 1 and axes > 2 else 0)] * (axes - 1)
    return [pairs - sum(rest)] + rest


def _prepare_rope(case, m):
    n, h, g, d, rd, axes = (case[x] for x in ("tokens", "h", "g", "d", "rotary", "axes"))
    dt = DTYPES[case["dtype"]]
    # runs of text, where all axes count on, and images, whose axes after the first are rows and columns
    pos, at, parts = case["far"], 0, []
    while at < n:
        size = 1 + int(torch.randint(0, 700, (), generator=m.host))
        i = torch.arange(min(size, n - at))
        wide = 1 + int(torch.randint(0, 40, (), generator=m.host))
        image = axes > 1 and bool(torch.randint(0, 2, (), generator=m.host))
        ways = [torch.zeros_like(i), i // wide, i % wide, i // 4][:axes] if image else [i] * axes
        parts.append(torch.stack(ways) + pos)
        pos = int(parts[-1].max()) + 1
        at += size
    positions = torch.cat(parts, 1)
    # the projection of gated attention: a head's query and gate side by side, keys after all of them
    proj = m.normal(n, 2 * h * d + 2 * g * d, dtype=dt)
    half = rd // 2
    freq = 1.0 / (1.0e7 ** (torch.arange(half, device=m.dev, dtype=torch.float32) / half))
    return SimpleNamespace(kind="rope", q=proj[:, :2 * h * d].view(n, h, 2 * d)[..., :d],
                           k=proj[:, 2 * h * d:2 * h * d + g * d].view(n, g, d), q_w=m.normal(d, dtype=dt, std=0.1),
                           k_w=m.normal(d, dtype=dt, std=0.1), freq=freq,
                           positions=(positions[0] if axes == 1 else positions).to(m.dev),
                           sections=None if axes == 1 else _sections(half, axes), interleaved=case["interleaved"])


def _prepare_write(case, m):
    n, block, g, d, dt = case["tokens"], case["block"], case["g"], case["d"], DTYPES[case["dtype"]]
    blocks = -(-n // block) + 3
    slots = m.order(blocks * block)[:n]
    kept = torch.rand(n, generator=m.host) < case["kept"]
    # keys come normed and rotated, values as columns of the projection that made both
    kv = m.normal(n, 2 * g * d, dtype=dt)
    return SimpleNamespace(kind="write", k=m.normal(n, g, d, dtype=dt), v=kv[:, g * d:].view(n, g, d),
                           slots=torch.where(kept, slots, torch.full_like(slots, -1)).to(m.dev), fmt=case["fmt"],
                           cache=m.empty(blocks, g, block, d, case["fmt"]), block=block, dtype=dt)


def _prepare_read(case, m):
    block = case["block"]
    lengths = m.sizes(case["len_lo"], case["len_hi"], case["requests"])
    tables, blocks = m.tables(lengths, block)
    r = torch.repeat_interleave(torch.arange(lengths.numel()), lengths)
    p = torch.arange(r.numel()) - (lengths.cumsum(0) - lengths)[r]
    slots = tables[r, p // block] * block + p % block
    return SimpleNamespace(kind="read", slots=slots.to(m.dev), block=block, dtype=DTYPES[case["dtype"]],
                           cache=m.cache(blocks, case["g"], block, case["d"], case["fmt"]))


def _prepare_attn(case, m):
    n, h, g, d = (case[x] for x in ("requests", "h", "g", "d"))
    dt = DTYPES[case["dtype"]]
    lengths = torch.cat((m.sizes(case["len_lo"], case["len_hi"], n), torch.zeros(case["idle"], dtype=torch.int64)))
    lengths = lengths[m.order(lengths.numel())]
    tables, blocks = m.tables(lengths, case["block"])
    rows = lengths.numel()
    # where each request's own document begins
    starts = (lengths * case["doc"]).long() if case["doc"] else None
    return SimpleNamespace(kind="attn", q=m.normal(rows, h, d, dtype=dt, std=1.5), lengths=lengths.to(m.dev),
                           longest=int(lengths.max()), tables=tables.to(torch.int32).to(m.dev),
                           starts=None if starts is None else starts.to(m.dev), window=case["window"] or None,
                           cap=case["cap"] or None, block=case["block"],
                           slopes=torch.exp2(-8 * torch.arange(1, h + 1, device=m.dev) / h) if case["slopes"] else None,
                           gate=m.normal(rows, h, d, dtype=dt) if case["gate"] else None,
                           cache=m.cache(blocks, g, case["block"], d, case["fmt"]))


# --- one pass -----------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attn": _plain_attn}[s.kind](s)


def _own(s):
    from yanchor_amd import layers
    if s.kind == "rope":
        return layers.qk_norm_rope(s.q, s.k, s.q_w, s.k_w, s.positions, s.freq, 1e-6, sections=s.sections,
                                   interleaved=s.interleaved)
    if s.kind == "write":
        layers.cache_write_quantized(s.k, s.v, s.slots, *s.cache)
        return layers.cache_read(s.slots, *s.cache, dtype=s.dtype)
    if s.kind == "read":
        return layers.cache_read(s.slots, *s.cache, dtype=s.dtype)
    keys, values, key_scales, value_scales = s.cache
    return layers.decode_attention(s.q, keys, values, s.tables, s.lengths, key_scales=key_scales,
                                   value_scales=value_scales, starts=s.starts, window=s.window, softcap=s.cap,
                                   slopes=s.slopes, gate=s.gate, max_length=s.longest)


def _axis_of_pair(pairs, sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = len(sections)
    return [j % axes if j < axes * sections[j % axes] else 0 for j in range(pairs)]


def _plain_rope(s):
    half = s.freq.numel()
    pos = s.positions if s.positions.ndim == 2 else s.positions[None]
    axis = torch.tensor(_axis_of_pair(half, s.sections or [half], s.interleaved), device=pos.device)
    angle = pos[axis].T.double() * s.freq.double()      # far positions need more than float32's 24 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def one(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * (1 + w.float())
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]), -1).to(x.dtype)
    return one(s.q, s.q_w), one(s.k, s.k_w)


def _plain_read(s):
    keys, values, key_scales, value_scales = s.cache
    live = s.slots >= 0
    slot = s.slots.clamp_min(0)
    b, row = slot // s.block, slot % s.block

    def one(data, scales):
        if scales is None:
            y = data[b, :, row].float()
        else:
            y = data.view(torch.uint8)[b, :, row].view(data.dtype)
            y = _values(y, scales[b, :, :, row])
        return torch.where(live[:, None, None], y, 0.0).to(s.dtype)
    return one(keys, key_scales), one(values, value_scales)


def _plain_write(s):
    live = s.slots >= 0
    slot = s.slots[live]
    b, row = slot // s.block, slot % s.block
    for x, data, scales in zip((s.k, s.v), s.cache[:2], s.cache[2:]):
        codes, sc = _quantise(x[live], s.fmt)
        data.view(torch.uint8)[b, :, row] = codes.view(torch.uint8)
        scales[b, :, :, row] = sc
    return _plain_read(s)


def _plain_attn(s):
    r, h, d = s.q.shape
    g, c, block = s.cache[0].shape[1], s.tables.shape[1], s.block
    dev = s.q.device
    p = torch.arange(s.longest, device=dev)
    blk = s.tables[:, p // block % c].clamp_min(0).long()

    def rows(data, scales):
        if scales is None:
            return data[blk, :, p % block].float().permute(0, 2, 1, 3)
        y = _values(data.view(torch.uint8)[blk, :, p % block].view(data.dtype), scales[blk, :, :, p % block])
        return y.permute(0, 2, 1, 3)
    q = s.q.float().view(r, g, h // g, d) * d ** -0.5
    x = q @ rows(s.cache[0], s.cache[2]).transpose(2, 3)
    if s.cap is not None:
        x = s.cap * torch.tanh(x / s.cap)
    back = (s.lengths - 1)[:, None] - p
    if s.slopes is not None:
        x = x - s.slopes.view(g, h // g, 1) * back[:, None, None].float()
    seen = back >= 0
    if s.window is not None:
        seen = seen & (back < s.window)
    if s.starts is not None:
        seen = seen & (p >= s.starts[:, None])
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(3, keepdim=True).clamp_min(-1e30)).exp_()
    den = x.sum(3, keepdim=True)
    o = (x @ rows(s.cache[1], s.cache[3])) / torch.where(den > 0, den, 1.0)   # a row that sees nothing: zeros
    o = o.reshape(r, h, d)
    if s.gate is not None:
        o = o * torch.sigmoid(s.gate.float())
    return o.to(s.q.dtype)


# --- what a pass cannot do without -----------------------------------------------

def work(case):
    kind, g, d = case["kind"], case["g"], case["d"]
    if kind == "rope":
        n, h = case["tokens"], case["h"]
        return {"bytes": 2 * 2 * n * (h + g) * d + 8 * n * case["axes"], "flops": n * (h + g) * (5 * d + 3 * case["rotary"])}
    if kind == "write":      # rows in, codes out and in again, rows out
        rows = case["tokens"] * (case["kept"] * (2 + 2 * ROW[case["fmt"]]) + 2) * 2 * g * d
        return {"bytes": rows + 16 * case["tokens"], "flops": 6 * case["tokens"] * g * d}
    if kind == "read":
        n = sum(_spread(case["len_lo"], case["len_hi"], case["requests"]))
        return {"bytes": n * (8 + 2 * g * d * (ROW[case["fmt"]] + 2)), "flops": 2 * n * g * d}
    h = case["h"]
    span = 0
    for x in _spread(case["len_lo"], case["len_hi"], case["requests"]):
        first = int(x * case["doc"])
        span += min(x - first, case["window"] or x)
    io = (case["requests"] + case["idle"]) * h * d * 2 * (3 if case["gate"] else 2)
    return {"bytes": io + span * (2 * g * d * ROW[case["fmt"]] + 4 / case["block"]), "flops": 4 * d * h * span}


# --- float64, from the definitions -----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_write, "read": _exact_read, "attn": _exact_attn}[s.kind](s)


def _exact_rope(s):
    f = torch.float64
    half = s.freq.numel()
    pos = s.positions if s.positions.ndim == 2 else s.positions[None]
    sections = s.sections or [half]
    turn = torch.zeros(pos.shape[1], half, dtype=f, device=pos.device)
    begin = 0
    for a, n in enumerate(sections):
        if s.interleaved and len(sections) > 1:
            if a == 0:
                turn[:] = pos[0][:, None]
            else:
                turn[:, a:len(sections) * n:len(sections)] = pos[a][:, None].to(f)
        else:
            turn[:, begin:begin + n] = pos[a][:, None].to(f)
        begin += n
    unit = torch.polar(torch.ones_like(turn), turn * s.freq.to(f))[:, None]
    out = []
    for x, w in ((s.q, s.q_w), (s.k, s.k_w)):
        y = x.to(f)
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.to(f))
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * unit
        out.append(torch.cat((z.real, z.imag, y[..., 2 * half:]), -1))
    return tuple(out)


def _code_values(fmt, device):
    """The values of the non-negative codes, ascending, by their definition."""
    f = torch.float64
    if fmt == "fp4":
        return torch.tensor(E2M1, dtype=f, device=device)
    small = torch.arange(8, dtype=f, device=device) / 8 * 2.0 ** -6
    rest = [(1 + torch.arange(8, dtype=f, device=device) / 8) * 2.0 ** e for e in range(-6, 9)]
    return torch.cat([small] + rest)[:127]


def _nearest(y, table):
    """The table's nearest value, of two equally near the one of even index."""
    hi = torch.searchsorted(table, y).clamp_max(table.numel() - 1)
    lo = (hi - 1).clamp_min(0)
    up, down = table[hi] - y, y - table[lo]
    take_lo = (down < up) | ((down == up) & (lo % 2 == 0))
    return torch.where(take_lo, table[lo], table[hi])


def _exact_write(s):
    f = torch.float64
    live = s.slots >= 0
    out = []
    for x in (s.k, s.v):
        n, g, d = x.shape
        table = _code_values(s.fmt, x.device)
        res = torch.zeros(n, g, d, dtype=f, device=x.device)
        for i in range(0, n, 8192):
            y = x[i:i + 8192].to(f).view(-1, g, d // 32, 32)
            top = y.abs().amax(-1, keepdim=True)
            s2 = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / table[-1]))
            s2 = torch.where(top > table[-1] * torch.exp2(s2), s2 + 1, s2)      # log2 may be off by its rounding
            s2 = torch.where(top <= table[-1] * torch.exp2(s2 - 1), s2 - 1, s2).clamp_min(-111)
            unit = torch.exp2(s2)
            z = _nearest((y / unit).abs(), table) * unit * torch.sign(y)
            res[i:i + 8192] = z.view(-1, g, d) * live[i:i + 8192, None, None]
        out.append(res)
    return tuple(out)


def _exact_rows(data, scales, b, row):
    """Rows of a cache as float64 [n, G, D]."""
    f = torch.float64
    if scales is None:
        return data[b, :, row].to(f)
    raw = data.view(torch.uint8)[b, :, row]
    if data.dtype == torch.float8_e4m3fn:
        y = raw.view(data.dtype).to(f)
    else:
        table = _code_values("fp4", data.device)
        y = torch.empty(*raw.shape[:-1], 2 * raw.shape[-1], dtype=f, device=raw.device)
        for part, code in ((0, raw % 16), (1, raw // 16)):
            y[..., part::2] = torch.where(code < 8, 1.0, -1.0) * table[(code % 8).long()]
    return y * torch.exp2(scales[b, :, :, row].to(f) - 127).repeat_interleave(32, -1)


def _exact_read(s):
    b, row = s.slots // s.block, s.slots % s.block
    out = []
    for data, scales in zip(s.cache[:2], s.cache[2:]):
        parts = [_exact_rows(data, scales, b[i:i + 16384], row[i:i + 16384]) for i in range(0, b.numel(), 16384)]
        out.append(torch.cat(parts))
    return tuple(out)


def _exact_attn(s):
    f = torch.float64
    r, h, d = s.q.shape
    g, block = s.cache[0].shape[1], s.block
    out = torch.zeros(r, h, d, dtype=f, device=s.q.device)
    starts = s.starts.tolist() if s.starts is not None else [0] * r
    for i, length in enumerate(s.lengths.tolist()):
        first = max(starts[i], length - s.window if s.window else 0, 0)
        if first >= length:
            continue
        p = torch.arange(first, length, device=s.q.device)
        b = s.tables[i].long()[p // block]
        keys = _exact_rows(s.cache[0], s.cache[2], b, p % block)
        values = _exact_rows(s.cache[1], s.cache[3], b, p % block)
        for kv in range(g):
            heads = slice(kv * (h // g), (kv + 1) * (h // g))
            w = keys[:, kv].contiguous() @ s.q[i, heads].to(f).T.contiguous() / math.sqrt(d)
            if s.cap is not None:
                w = s.cap * torch.tanh(w / s.cap)
            if s.slopes is not None:
                w = w - s.slopes[heads].to(f) * (length - 1 - p)[:, None]
            out[i, heads] = torch.softmax(w, 0).T.contiguous() @ values[:, kv].contiguous()
    if s.gate is not None:
        out = out * torch.sigmoid(s.gate.to(f))
    return out
