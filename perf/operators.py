"""Operators of a quantized KV cache, as they are measured.

Three operators, each over caches [B, T, Hkv, D] whose head rows are stored as q8_0 (34-byte) or q4_0 (18-byte) blocks of
32 values (an f16 scale, then the codes), kept contiguous, as a ring of T rows, or in pages behind a page table:

  * "cache":     new rows are quantized as they are appended, and logical steps are read back as f16 / f32
                 (`aion_cuda_sequence_append` with a quantized cache, `aion_cuda_sequence_read`);
  * "attention": grouped-query attention whose K / V are such a cache (`aion_cuda_attention` with quantized K / V);
  * "rope":      RMSNorm of every query and key head, rotary positions, and the append of K and V to their caches, in one
                 pass over the projection's output (`aion_cuda_qk_norm_rope_append`).

`own = False` computes them with elementary torch operations in 32 bits (64 where a border or a long sum needs it);
`own = True` calls the C ABI of the library through its ctypes binding, with the step records made once per state.
"""
import ctypes

import numpy as np
import torch

own = False

BLOCK = {"q8_0": 34, "q4_0": 18}
TORCH = {"f32": torch.float32, "f16": torch.float16}
BASE_FREQUENCY = 10000.0
EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------

def cache_case(name, **kw):
    c = dict(op="cache", batch=1, t_cap=2048, heads=1, dim=256, new=1, read=1, dtype="q8_0", src="f32", out="f16", layout="plain", page=64)
    c.update(kw)
    return dict(c, name=name) if name else c


def attention_case(name, **kw):
    c = dict(op="attention", batch=1, t_cap=2048, new=1, heads=8, kv_heads=1, dim=256, k="q8_0", v="q8_0", q="f32", layout="plain", page=64,
             left=-1, cap=0.0, ragged=True)
    c.update(kw)
    return dict(c, name=name) if name else c


def rope_case(name, **kw):
    c = dict(op="rope", batch=1, t_cap=2048, new=1, heads=8, kv_heads=1, dim=256, k="q8_0", v="q8_0", layout="plain", page=64, proportion=1.0)
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # A decode step of the synthetic decoder (8 query heads over 1 kv head of 256, context 2048): 64 requests add one row each.
        cache_case("append-step", batch=64),
        # Four prompts of an odd length go into a paged q4 cache and are read back, as when a prefix is checked or moved.
        cache_case("append-prompt-paged", batch=4, t_cap=4096, heads=4, dim=128, new=1531, read=1531, dtype="q4_0", src="f16", layout="paged"),
        # Long prefixes of different lengths leave a q4 cache as f16 (migration to an f16 cache, a prefix handed on); most of the
        # work of this operator is here.
        cache_case("read-prefixes", batch=24, t_cap=4100, heads=4, dim=256, new=0, read=4097, dtype="q4_0"),
        # One request in the middle of a conversation: nothing but latency.
        attention_case("decode-one", t_cap=1024, ragged=False),
        # The decoder's own decode batch at its full context, lengths mixed, one slot empty.
        attention_case("decode-batch", batch=64, k="q4_0", v="q4_0"),
        # Few requests with a very long paged context, 32 query heads over 8 kv heads, K in 8 bits and V in 4.
        attention_case("decode-long-paged", batch=6, t_cap=65536, heads=32, kv_heads=8, dim=128, v="q4_0", layout="paged"),
        # Five drafted tokens per request are verified against a sliding window in a ring cache, with capped logits.
        attention_case("verify-window", batch=16, t_cap=1500, new=5, heads=16, kv_heads=4, dim=64, k="q4_0", v="q4_0", q="f16", layout="rolling",
                       left=1023, cap=50.0),
        # A chunk of a long prompt (8 query heads over 4 kv heads of 256): bound by arithmetic.
        attention_case("prompt-chunk", t_cap=8192, new=1024, kv_heads=4, ragged=False),
        # The decoder's step with normed heads into f16 caches: 64 rows.
        rope_case("rope-step", batch=64, k="f16", v="f16"),
        # 512 requests, K in 8 bits and V in 4, pages of 64 rows.
        rope_case("rope-step-paged", batch=512, t_cap=256, v="q4_0", layout="paged"),
        # A batch of prompts, 32 query heads over 8 kv heads of 128, half of every head rotated.
        rope_case("rope-prompt", batch=3, t_cap=2048, new=1999, heads=32, kv_heads=8, dim=128, proportion=0.5),
        # A long prompt into q4 caches, 8 query heads over 4 kv heads of 256.
        rope_case("rope-prompt-long", t_cap=16384, new=16000, kv_heads=4, k="q4_0", v="q4_0"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "rope"])
    dim = rng.choice([64, 128, 256])
    layout = rng.choice(["plain", "paged", "rolling"])
    page = rng.choice([16, 64, 96, 128])
    if op == "cache":
        heads = rng.choice([1, 2, 3, 4, 8])
        batch = _spread(rng, 1, 64)
        room = 90_000_000 // (batch * heads * dim)  # values read back: no more than the largest listed case reads
        new = min(_spread(rng, 1, 2000), max(1, room // 2))
        read = min(rng.choice([new, _spread(rng, 1, 8000)]), max(1, room // 2))
        t_cap = max(new, read) + rng.randrange(0, 500)
        return cache_case(None, batch=batch, t_cap=t_cap, heads=heads, dim=dim, new=new, read=read, dtype=rng.choice(["q8_0", "q4_0"]),
                          src=rng.choice(["f32", "f16"]), out=rng.choice(["f32", "f16"]), layout=layout, page=page)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    k, v = rng.choice(["q8_0", "q4_0"]), rng.choice(["q8_0", "q4_0"])
    if op == "attention":
        new = rng.choice([1, 1, rng.randrange(2, 12), _spread(rng, 12, 700)])
        batch = _spread(rng, 1, 96)
        # Cache rows of all heads, and (row, key, head) products: within the largest listed cases.
        room = min(250_000_000 // (batch * kv_heads * dim), 10_000_000_000 // (batch * new * heads * dim))
        t_cap = _spread(rng, 16, max(17, min(40000, room)))
        t_cap = max(t_cap, new + rng.randrange(1, 60))
        left = rng.choice([-1, -1, _spread(rng, 8, 2000)])
        return attention_case(None, batch=batch, t_cap=t_cap, new=new, heads=heads, kv_heads=kv_heads, dim=dim, k=k, v=v, q=rng.choice(["f32", "f16"]),
                              layout=layout, page=page, left=left, cap=rng.choice([0.0, 0.0, 30.0]), ragged=rng.choice([True, True, False]))
    batch = _spread(rng, 1, 256)
    room = 60_000_000 // (batch * (heads + 2 * kv_heads) * dim)  # values of the projection: no more than the longest prompt has
    new = max(1, min(rng.choice([1, _spread(rng, 2, 4000)]), room))
    t_cap = min(new + rng.randrange(1, 300), max(new + 1, 200_000_000 // (batch * kv_heads * dim)))
    return rope_case(None, batch=batch, t_cap=t_cap, new=new, heads=heads, kv_heads=kv_heads, dim=dim, k=rng.choice([k, "f16"]), v=rng.choice([v, "f16"]),
                     layout=layout, page=page, proportion=rng.choice([1.0, 0.5, 0.25]))


# ---- what every case says about its requests --------------------------------------------

def held(c):
    """Logical steps that each request holds when the operator reads its cache (the new rows of an attention step among them)."""
    T, n = c["t_cap"], c["batch"]
    if c["op"] == "cache":
        if c["new"]:  # read back right after the append
            start = starts(c)
            return [s + c["new"] for s in start]
        return [0 if n >= 8 and b == n - 1 else T - (b * 173) % (T // 2 + 1) for b in range(n)]
    if c["layout"] == "rolling":
        return [T + (b * 37) % T for b in range(n)]  # the ring has come round
    if not c["ragged"]:
        return [T] * n
    least = min(T, c["new"])
    return [0 if n >= 8 and b == n - 1 else max(least, T - (b * 7919) % (3 * T // 4 + 1)) for b in range(n)]


def starts(c):
    """Logical step of each request's first new row."""
    T, L, n = c["t_cap"], c["new"], c["batch"]
    if c["layout"] == "rolling":
        return [(b * 97) % (2 * T) for b in range(n)]
    return [(b * 31) % (T - L + 1) for b in range(n)]


def read_starts(c):
    """First logical step that is read back: the new rows' first, or as many as are read up to the newest."""
    if c["new"]:
        return [max(0, h - c["read"]) for h in held(c)]
    return [0] * c["batch"]


def visible(c, h, first, row):
    """Keys [lo, hi) that row `row` of a request with `h` steps sees: causal, `left` back, and what a ring still has."""
    pos = first + row
    hi = min(h, pos + 1)
    lo = max(0, pos - c["left"]) if c["left"] >= 0 else 0
    if c["layout"] == "rolling":
        lo = max(lo, h - c["t_cap"])
    return lo, max(lo, hi)


def first_position(c, h):
    return max(0, h - c["new"])


def row_bytes(dtype, dim):
    return dim // 32 * BLOCK[dtype] if dtype in BLOCK else dim * 2


def work(case):
    c = case
    D = c["dim"]
    if c["op"] == "cache":
        new_values = c["batch"] * c["new"] * c["heads"] * D
        rows_held = 0
        for h, s in zip(held(c), read_starts(c)):
            lo = max(s, h - c["t_cap"] if c["layout"] == "rolling" else 0)
            rows_held += max(0, min(h, s + c["read"]) - lo)
        row = c["heads"] * row_bytes(c["dtype"], D)
        out = c["batch"] * c["read"] * c["heads"] * D
        b = new_values * (4 if c["src"] == "f32" else 2) + c["batch"] * c["new"] * row + rows_held * row + out * (4 if c["out"] == "f32" else 2)
        return {"bytes": b, "flops": 4 * new_values + rows_held * c["heads"] * D}
    rows = c["batch"] * c["new"]
    if c["op"] == "rope":
        values = rows * (c["heads"] + 2 * c["kv_heads"]) * D
        stored = rows * c["kv_heads"] * (row_bytes(c["k"], D) + row_bytes(c["v"], D))
        back = 0  # a quantized cache is handed back as f16 values: read again, and written
        for t in (c["k"], c["v"]):
            if t in BLOCK:
                back += rows * c["kv_heads"] * (row_bytes(t, D) + 2 * D)
        return {"bytes": values * 4 + rows * c["heads"] * D * 4 + stored + back, "flops": 10 * values}
    keys, pairs = 0, 0
    for h in held(c):
        first = first_position(c, h)
        spans = [visible(c, h, first, l) for l in range(c["new"])]
        pairs += sum(hi - lo for lo, hi in spans)
        some = [s for s in spans if s[1] > s[0]]
        keys += max(s[1] for s in some) - min(s[0] for s in some) if some else 0
    kv = keys * c["kv_heads"] * (row_bytes(c["k"], D) + row_bytes(c["v"], D))
    q_bytes = 4 if c["q"] == "f32" else 2
    return {"bytes": kv + rows * c["heads"] * D * (q_bytes + 4), "flops": 4 * pairs * c["heads"] * D}


# ---- the block formats -------------------------------------------------------------------

def _away(x):
    """Nearest whole number, halves away from zero (in 64 bits: x + 0.5 must not round)."""
    x = x.double()
    return torch.sign(x) * torch.floor(x.abs() + 0.5)


def quantize(x, dtype):
    """f32 [..., D] -> bytes [..., D / 32 * block]: the codes are chosen in f32, each step rounded once."""
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = blocks.abs().amax(-1, keepdim=True)
    one = torch.ones_like(amax)
    top = torch.full_like(amax, 127.0 if dtype == "q8_0" else 7.0)  # a tensor: a division by a number multiplies by its reciprocal
    scale = torch.where(amax == 0, one, amax / top)
    half = scale.half()
    if dtype == "q8_0":
        eff = half.float()
        inv = torch.where((amax == 0) | (eff == 0), torch.zeros_like(eff), one / eff)
        codes = _away(blocks * inv).clamp(-128, 127).to(torch.int8).view(torch.uint8)
    else:
        n = (_away(blocks / scale).clamp(-8, 7) + 8).to(torch.uint8)
        codes = n[..., 0::2] | (n[..., 1::2] << 4)
    packed = torch.cat([half.view(torch.uint8), codes], -1)
    return packed.reshape(*x.shape[:-1], -1)


def values(packed, dtype):
    """bytes [..., D / 32 * block] -> f32 [..., D]: code x scale, exact in 32 bits."""
    if dtype == "f16":
        return packed.float()
    size = BLOCK[dtype]
    blocks = packed.reshape(*packed.shape[:-1], packed.shape[-1] // size, size)
    scale = blocks[..., :2].contiguous().view(torch.float16).float()
    codes = blocks[..., 2:]
    if dtype == "q8_0":
        n = codes.contiguous().view(torch.int8).float()
    else:
        n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    return (n * scale).flatten(-2)


# ---- states ------------------------------------------------------------------------------

def _pages(c, gen):
    """A page table [B, pages per request] over a pool with a few pages to spare, in an order of its own."""
    per = -(-c["t_cap"] // c["page"])
    pool = c["batch"] * per + 3
    return torch.randperm(pool, generator=gen, device="cuda")[: c["batch"] * per].to(torch.int32).reshape(c["batch"], per), pool


def _empty_cache(c, dtype, heads, pool):
    rows = (pool, c["page"]) if c["layout"] == "paged" else (c["batch"], c["t_cap"])
    if dtype == "f16":
        return torch.zeros(*rows, heads, c["dim"], dtype=torch.float16, device="cuda")
    return torch.zeros(*rows, heads, row_bytes(dtype, c["dim"]), dtype=torch.uint8, device="cuda")


def _filled_cache(c, dtype, heads, pool, gen, scale):
    """A cache whose every row holds the blocks of normal values, head by head of a different size."""
    cache = _empty_cache(c, dtype, heads, pool)
    flat = cache.view(-1, heads, cache.shape[-1])
    size = scale * (0.5 + torch.rand(heads, 1, generator=gen, device="cuda"))
    step = max(1, (1 << 26) // (heads * c["dim"]))
    for at in range(0, flat.shape[0], step):
        n = min(step, flat.shape[0] - at)
        flat[at:at + n] = quantize(torch.randn(n, heads, c["dim"], generator=gen, device="cuda") * size, dtype)
    return cache


def frequencies(c):
    """Angle per position of each rotated pair: repeated f32 products, as the rotary step of the library builds its table."""
    pairs = c["dim"] // 2
    step = np.float32(float(BASE_FREQUENCY) ** float(np.float32(-2.0) / np.float32(c["dim"])))
    table = np.empty(pairs, dtype=np.float32)
    f = np.float32(1.0)
    for i in range(pairs):
        table[i] = f
        f = np.float32(f * step)
    return table[: int(np.floor(np.float32(c["proportion"]) * np.float32(pairs)))]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    B, L, D = c["batch"], c["new"], c["dim"]
    s = {"case": c, "table": None, "pool": 0}
    if c["layout"] == "paged":
        s["table"], s["pool"] = _pages(c, gen)
    if c["op"] == "cache":
        s["held"], s["read_start"] = i32(held(c)), i32(read_starts(c))
        s["out"] = torch.empty(B, c["read"], c["heads"], D, dtype=TORCH[c["out"]], device="cuda")
        s["cache"] = _filled_cache(c, c["dtype"], c["heads"], s["pool"], gen, 1.5)
        if L:
            s["new"] = (randn(B, L, c["heads"], D) * 1.5).to(TORCH[c["src"]])
            s["start"] = i32(starts(c))
    elif c["op"] == "attention":
        h = held(c)
        s["held"] = i32(h)
        s["positions"] = i32([[first_position(c, x) + l for l in range(L)] for x in h])
        s["q"] = (randn(B, L, c["heads"], D) * 1.2).to(TORCH[c["q"]])
        s["k"] = _filled_cache(c, c["k"], c["kv_heads"], s["pool"], gen, 1.0)
        s["v"] = _filled_cache(c, c["v"], c["kv_heads"], s["pool"], gen, 0.8)
        s["out"] = torch.empty(B, L, c["heads"], D, device="cuda")
        s["scale"] = float(D) ** -0.5
    else:
        begin = starts(c)
        s["start"] = i32(begin)
        s["positions"] = i32([[x + l for l in range(L)] for x in begin])
        s["qkv"] = randn(B, L, (c["heads"] + 2 * c["kv_heads"]) * D) * 0.9
        s["q_gamma"] = 1.0 + 0.2 * randn(D)
        s["k_gamma"] = 1.0 + 0.2 * randn(D)
        s["frequencies"] = torch.from_numpy(frequencies(c)).cuda()
        s["k"] = _empty_cache(c, c["k"], c["kv_heads"], s["pool"])
        s["v"] = _empty_cache(c, c["v"], c["kv_heads"], s["pool"])
        s["q_out"] = torch.empty(B, L, c["heads"], D, device="cuda")
        for t in "kv":
            if c[t] in BLOCK:
                s[t + "_out"] = torch.empty(B, L, c["kv_heads"], D, dtype=torch.float16, device="cuda")
    return s


# ---- the plain forms -----------------------------------------------------------------------

def _cache_rows(s, steps, cache):
    """Index of the cache row (of all requests' rows, or of the pool's) that holds logical step steps[b, t]."""
    c = s["case"]
    if c["layout"] == "paged":
        page = torch.gather(s["table"].long(), 1, steps // c["page"])
        return page * c["page"] + steps % c["page"]
    if c["layout"] == "rolling":
        steps = steps % c["t_cap"]
    return torch.arange(c["batch"], device="cuda")[:, None] * c["t_cap"] + steps


def _append(s, cache, rows, dtype):
    """Rows f32 [B, L, H, D] into the cache from each request's start."""
    c = s["case"]
    steps = s["start"].long()[:, None] + torch.arange(c["new"], device="cuda")
    if c["new"] > c["t_cap"]:
        raise ValueError("more new rows than the cache holds")
    at = _cache_rows(s, steps, cache).reshape(-1)
    packed = rows.half() if dtype == "f16" else quantize(rows, dtype)
    cache.view(-1, *cache.shape[2:])[at] = packed.reshape(-1, *cache.shape[2:])


def _read(s, cache, start, length, count, dtype, out):
    """Logical steps start[b] .. start[b] + count as values; zeros where the request does not hold the step."""
    c = s["case"]
    steps = start.long()[:, None] + torch.arange(count, device="cuda")
    length = length.long()[:, None]
    oldest = torch.clamp(length - c["t_cap"], min=0)
    live = (steps < length) & (steps >= oldest)
    at = _cache_rows(s, torch.where(live, steps, torch.zeros_like(steps)), cache)
    rows = cache.view(-1, *cache.shape[2:])[at.reshape(-1)].reshape(*at.shape, *cache.shape[2:])
    got = values(rows, dtype)
    return torch.where(live[:, :, None, None], got, torch.zeros_like(got)).to(out)


def _attend(s):
    c = s["case"]
    B, L, H, G, D, T = c["batch"], c["new"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["t_cap"]
    k, v = s["k"], s["v"]
    if c["layout"] == "paged":
        k = k[s["table"].long()].flatten(1, 2)[:, :T]
        v = v[s["table"].long()].flatten(1, 2)[:, :T]
    length = s["held"].long()[:, None]
    step = torch.arange(T, device="cuda")[None, :]
    oldest = torch.zeros_like(length)
    if c["layout"] == "rolling":
        step = step + T * torch.div(length - 1 - step, T, rounding_mode="floor")  # the newest step that the ring row holds
        oldest = torch.clamp(length - T, min=0)
    pos = s["positions"].long()[:, :, None]
    seen = ((step >= oldest) & (step < length))[:, None, :] & (step[:, None, :] <= pos)
    if c["left"] >= 0:
        seen = seen & (step[:, None, :] >= pos - c["left"])
    kf = values(k, c["k"]).permute(0, 2, 3, 1)
    q = s["q"].float().reshape(B, L, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * L, D)
    x = (q @ kf).reshape(B, H, G, L, T) * s["scale"]
    del kf
    if c["cap"] > 0:
        x = c["cap"] * torch.tanh(x / c["cap"])
    x = torch.where(seen[:, None, None], x, torch.full_like(x, -float("inf")))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -float("inf"), torch.zeros_like(top), top)
    p = torch.exp(x - top)
    del x
    total = p.sum(-1).reshape(B, H, G * L, 1)
    vf = values(v, c["v"]).permute(0, 2, 1, 3)
    o = p.reshape(B, H, G * L, T) @ vf
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.reshape(B, H, G, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H * G, D)


def _norm(x, gamma):
    """(x * 1 / sqrt(mean(x^2) + eps)) * gamma per head: the statistic in 64 bits, two rounded products."""
    inv = (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()
    return (x * inv) * gamma


def _rotate(s, x):
    """Rotary positions on pairs (i, D / 2 + i); each product and sum rounds once."""
    c = s["case"]
    f = s["frequencies"]
    n, half = f.numel(), c["dim"] // 2
    angle = (s["positions"].float()[:, :, None] * f).double()
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    lo, hi = x[..., :half], x[..., half:]
    a, b = lo[..., :n], hi[..., :n]
    return torch.cat([a * cos - b * sin, lo[..., n:], a * sin + b * cos, hi[..., n:]], -1)


def _plain(s):
    c = s["case"]
    if c["op"] == "attention":
        return _attend(s)
    if c["op"] == "cache":
        if c["new"]:
            _append(s, s["cache"], s["new"].float(), c["dtype"])
        return _read(s, s["cache"], s["read_start"], s["held"], c["read"], c["dtype"], s["out"].dtype)
    B, L, D = c["batch"], c["new"], c["dim"]
    x = s["qkv"].reshape(B, L, c["heads"] + 2 * c["kv_heads"], D)
    q, k, v = x.split([c["heads"], c["kv_heads"], c["kv_heads"]], 2)
    q = _rotate(s, _norm(q, s["q_gamma"]))
    k = _rotate(s, _norm(k, s["k_gamma"]))
    _append(s, s["k"], k, c["k"])
    _append(s, s["v"], v, c["v"])
    return {"q": q, "k": _stored(s, "k"), "v": _stored(s, "v")}


def _stored(s, t):
    """An f16 cache is returned as it is; the new rows of a quantized one as the values that they stand for."""
    c = s["case"]
    if c[t] == "f16":
        return s[t]
    return _read(s, s[t], s["start"], s["start"] + c["new"], c["new"], c[t], torch.float16)


# ---- the library's calls ---------------------------------------------------------------------

_backend = None


def _calls(s):
    """The step records of one pass, made once per state, as a program keeps them."""
    global _backend
    from aion_b200 import capi
    from aion_b200.backend import CudaBackend

    if _backend is None:
        _backend = CudaBackend(torch.cuda.current_device())
    lib, c = capi.load(), s["case"]
    dtypes = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "q8_0": capi.DTYPE_Q8_0, "q4_0": capi.DTYPE_Q4_0}
    none = capi.Operand(0, 0, 0)
    op = lambda t: none if t is None else capi.Operand(t.data_ptr(), 0, t.numel() * t.element_size())  # noqa: E731
    rolling = int(c["layout"] == "rolling")
    paged = dict(page_table=op(s["table"]), page_tokens=c["page"] if s["pool"] else 0, pool_pages=s["pool"])
    calls = []

    def read(cache, heads, start, lengths, count, dtype, out):
        calls.append((lib.aion_cuda_sequence_read, capi.SequenceRead(
            out=op(out), cache=op(cache), start_index=op(start), lengths=op(lengths), batch=c["batch"], t_cap=c["t_cap"], heads=heads,
            head_dim=c["dim"], out_len=count, dtype=dtypes[dtype], out_dtype=dtypes["f32" if out.dtype == torch.float32 else "f16"],
            rolling=rolling, **paged)))

    if c["op"] == "attention":
        unbounded = capi.WINDOW_UNBOUNDED
        calls.append((lib.aion_cuda_attention, capi.Attention(
            out=op(s["out"]), q=op(s["q"]), k=op(s["k"]), v=op(s["v"]), query_positions=op(s["positions"]), kv_lengths=op(s["held"]),
            q_dtype=dtypes[c["q"]], k_dtype=dtypes[c["k"]], v_dtype=dtypes[c["v"]], rolling=rolling, batch=c["batch"], l_q=c["new"],
            h_q=c["heads"], h_kv=c["kv_heads"], d_k=c["dim"], d_v=c["dim"], t_cap=c["t_cap"], scale=s["scale"], soft_cap=c["cap"],
            window_left=c["left"] if c["left"] >= 0 else unbounded, window_right=0, window_chunk=0, flags=0, **paged)))
        s["result"] = s["out"]
    elif c["op"] == "cache":
        if c["new"]:
            calls.append((lib.aion_cuda_sequence_append, capi.SequenceAppend(
                cache=op(s["cache"]), new_kv=op(s["new"]), end_index=op(s["start"]), batch=c["batch"], t_cap=c["t_cap"], heads=c["heads"],
                head_dim=c["dim"], new_len=c["new"], dtype=dtypes[c["dtype"]], new_dtype=dtypes[c["src"]], rolling=rolling, **paged)))
        read(s["cache"], c["heads"], s["read_start"], s["held"], c["read"], c["dtype"], s["out"])
        s["result"] = s["out"]
    else:
        calls.append((lib.aion_cuda_qk_norm_rope_append, capi.QKNormRopeAppend(
            q_out=op(s["q_out"]), qkv=op(s["qkv"]), q_gamma=op(s["q_gamma"]), k_gamma=op(s["k_gamma"]), positions=op(s["positions"]),
            end_index=op(s["start"]), k_cache=op(s["k"]), v_cache=op(s["v"]), batch=c["batch"], len=c["new"], h_q=c["heads"],
            h_kv=c["kv_heads"], head_dim=c["dim"], t_cap=c["t_cap"], eps=EPS, base_frequency=BASE_FREQUENCY, scale_factor=1.0,
            proportion=c["proportion"], k_dtype=dtypes[c["k"]], v_dtype=dtypes[c["v"]], rolling=rolling, **paged)))
        s["result"] = {"q": s["q_out"], "k": s["k"], "v": s["v"]}
        for t in "kv":
            if c[t] in BLOCK:
                read(s[t], c["kv_heads"], s["start"], None, c["new"], c[t], s[t + "_out"])
                s["result"][t] = s[t + "_out"]
                if rolling:  # a ring that has come round holds its newest steps: the read has to know how many there are
                    s["ends"] = s["start"] + c["new"]
                    calls[-1][1].lengths = op(s["ends"])
    s["calls"] = [(fn, ctypes.byref(rec), rec) for fn, rec in calls]


def run(state):
    if not own:
        return _plain(state)
    if "calls" not in state:
        _calls(state)
    for fn, rec, _ in state["calls"]:
        if fn(_backend.handle, rec):
            raise RuntimeError("the library refused a call")
    return state["result"]


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_blocks(x, dtype):
    """What quantizing f64 values that are f32 numbers leaves of them. The format is defined by roundings to f32 and f16: each is
    made here from the 64-bit quotient or product (correctly rounded, as 53 bits are more than 2 x 24 + 1)."""
    f32 = lambda t: t.float().double()  # noqa: E731
    n = x.shape[-1] // 32
    v = x.unflatten(-1, (n, 32))
    m = v.abs().max(-1).values[..., None]
    d = f32(m / (127.0 if dtype == "q8_0" else 7.0))
    d[m == 0] = 1.0
    stored = d.to(torch.float16).double()
    if dtype == "q8_0":
        r = f32(1.0 / stored)
        r[(m == 0) | (stored == 0)] = 0.0
        y, low, high = f32(v * r), -128, 127
    else:
        y, low, high = f32(v / d), -8, 7
    whole = torch.where(y < 0, -torch.floor(0.5 - y), torch.floor(0.5 + y)).clamp(low, high)
    return (whole * stored).flatten(-2)


def _exact_values(raw, dtype):
    """Blocks [..., bytes] as f64 values."""
    size = BLOCK[dtype]
    b = raw.unflatten(-1, (raw.shape[-1] // size, size))
    d = (b[..., 0].int() + 256 * b[..., 1].int()).to(torch.int16).view(torch.float16).double()[..., None]
    if dtype == "q8_0":
        code = b[..., 2:].double()
        code = code - 256.0 * (code > 127)
    else:
        low, high = b[..., 2:].int() % 16, b[..., 2:].int() // 16
        code = torch.stack((low, high), -1).reshape(*b.shape[:-1], 32).double() - 8.0
    return (code * d).flatten(-2)


def _request_rows(s, cache, b, steps):
    """The stored rows of one request's logical steps."""
    c = s["case"]
    if c["layout"] == "paged":
        return cache[s["table"][b].long()[steps // c["page"]], steps % c["page"]]
    return cache[b][steps % c["t_cap"]]


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, L, D = c["batch"], c["new"], c["dim"]
    count = lambda n: torch.arange(n, device="cuda")  # noqa: E731
    if c["op"] == "cache":
        out = torch.zeros(B, c["read"], c["heads"], D, dtype=torch.float64, device="cuda")
        fresh = _exact_blocks(s["new"].double(), c["dtype"]) if L else None
        for b, (h, r) in enumerate(zip(held(c), read_starts(c))):
            oldest = max(0, h - c["t_cap"])
            lo, hi = max(r, oldest), max(r, min(h, r + c["read"]))
            if hi <= lo:
                continue
            row = _exact_values(_request_rows(s, s["cache"], b, lo + count(hi - lo)), c["dtype"])
            if L:  # steps at and after the start are the new ones
                first = starts(c)[b]
                if hi > first:
                    a = max(lo, first)
                    row[a - lo:] = fresh[b, a - first:hi - first]
            out[b, lo - r:hi - r] = row
        return out
    if c["op"] == "attention":
        G = c["heads"] // c["kv_heads"]
        out = torch.zeros(B, L, c["heads"], D, dtype=torch.float64, device="cuda")
        if sum(held(c)) * L * c["heads"] * D > 2e11:
            return None
        for b, h in enumerate(held(c)):
            first = first_position(c, h)
            spans = [visible(c, h, first, l) for l in range(L)]
            lo, hi = min(x[0] for x in spans), max(x[1] for x in spans)
            if hi <= lo:
                continue
            steps = lo + count(hi - lo)
            k = _exact_values(_request_rows(s, s["k"], b, steps), c["k"])
            v = _exact_values(_request_rows(s, s["v"], b, steps), c["v"])
            a = torch.tensor([x[0] for x in spans], device="cuda")[:, None]
            z = torch.tensor([x[1] for x in spans], device="cuda")[:, None]
            hidden = (steps[None] < a) | (steps[None] >= z)
            for g in range(c["kv_heads"]):
                q = s["q"][b, :, g * G:(g + 1) * G].double()
                y = torch.einsum("lgd,td->lgt", q, k[:, g]) * s["scale"]
                if c["cap"]:
                    y = c["cap"] * torch.tanh(y / c["cap"])
                y = y.masked_fill(hidden[:, None], -float("inf"))
                w = torch.nan_to_num(torch.softmax(y, -1))
                out[b, :, g * G:(g + 1) * G] = torch.einsum("lgt,td->lgd", w, v[:, g])
        return out
    x = s["qkv"].double().unflatten(-1, (-1, D))
    heads = [x[:, :, :c["heads"]], x[:, :, c["heads"]:c["heads"] + c["kv_heads"]], x[:, :, c["heads"] + c["kv_heads"]:]]
    f = frequencies(c)
    # The angle is position x frequency rounded to f32 by definition; what follows is in 64 bits.
    angle = (s["positions"].float()[..., None] * torch.from_numpy(f).cuda()).double()[:, :, None]
    turned = []
    for y, gamma in ((heads[0], s["q_gamma"]), (heads[1], s["k_gamma"])):
        y = y * (y.pow(2).sum(-1, keepdim=True) / D + EPS).rsqrt() * gamma.double()
        n, half = len(f), D // 2
        z = torch.complex(y[..., :half], y[..., half:])
        z[..., :n] = z[..., :n] * torch.polar(torch.ones_like(angle), angle)
        turned.append(torch.cat([z.real, z.imag], -1))
    got = {"q": turned[0]}
    for t, y in (("k", turned[1]), ("v", heads[2])):
        if c[t] != "f16":
            # The codes are chosen from f32 values: a key that lies on a border has no value of its own in 64 bits, so keys are
            # rounded to f32 first and the few that fall on the other side of a border are one code off.
            got[t] = _exact_blocks(y.float().double(), c[t])
            continue
        whole = torch.zeros(s[t].shape, dtype=torch.float64, device="cuda")
        for b, first in enumerate(starts(c)):
            steps = first + count(L)
            if c["layout"] == "paged":
                whole[s["table"][b].long()[steps // c["page"]], steps % c["page"]] = y[b]
            else:
                whole[b, steps % c["t_cap"]] = y[b]
        got[t] = whole
    return got
