"""What the K/V-cache operators are measured on: the quantised cache of the rollout's attention (written, read back, attended to).

The cache of one layer holds the keys and values of ``E`` episodes in blocks of 32 numbers along the head dimension, each block
with one power of two as its scale:

* ``codes``  uint8 (2, E, kv_heads, S, dim * bits / 8): 4-bit e2m1 numbers, two a byte (the even dimension in the low half), or
  8-bit e4m3 numbers; index 0 holds the keys, 1 the values; S is the window's capacity;
* ``scales`` uint8 (2, E, kv_heads, S, 4): byte b is the exponent (biased by 127) of block b's scale, 255 = the block is not a number.

The scale of a block is the smallest 2^e, -100 <= e <= 100, at which its largest magnitude is at most 6 (e2m1) or 448 (e4m3);
numbers are rounded to the nearest code, ties to the even one.

Four kinds of cases: ``append`` (write new steps and read them back), ``read`` (read a whole history back), ``attend`` (attention of
``steps`` new positions over the cached keys and values) and ``step`` (append one position and attend to it in one call).
"""
import math

import torch

own = False

BLOCK = 32
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, kind, bits, dtype, rows, steps, heads, kv_heads, dim, capacity, low, high, window=0, causal=True):
    return dict(name=name, kind=kind, bits=bits, dtype=dtype, rows=rows, steps=steps, heads=heads, kv_heads=kv_heads, dim=dim,
                capacity=capacity, low=low, high=high, window=window, causal=causal)


def listed():
    return [
        # one control step of 64 running episodes: the new keys and values of one layer enter the cache (latency)
        _case("append_step", "append", 4, "float32", 64, 1, 8, 8, 96, 32, 0, 31),
        # 512 episodes whose windows of 32 slid by one: all rows of one layer are written again
        _case("append_windows", "append", 8, "float32", 512, 32, 8, 8, 96, 32, 0, 0),
        # long histories handed over from a 16-bit model, an odd number of steps each
        _case("append_long", "append", 4, "bfloat16", 16, 4093, 8, 8, 128, 8192, 0, 4099),
        # a server moves 24 episodes away: their whole histories, of different lengths, come back in 16 bits
        _case("read_long", "read", 4, "float16", 24, 6001, 8, 8, 64, 6144, 1700, 6001),
        # the policy's cached step at its own sizes: 512 episodes somewhere in a window of 32
        _case("step_policy", "step", 4, "float32", 512, 1, 8, 8, 96, 32, 0, 31),
        # one robot with a history of about nine minutes at 15 Hz: few rows, one long axis
        _case("step_single_long", "step", 8, "float32", 1, 1, 8, 8, 96, 8192, 8190, 8191),
        # many long episodes in 4 bits, four query heads to a key head
        _case("attend_decode_gqa", "attend", 4, "bfloat16", 48, 1, 32, 8, 128, 16384, 7001, 16383),
        # the same in 8 bits and shorter, odd lengths, only the last 1000 positions looked at
        _case("attend_decode_local", "attend", 8, "float16", 160, 1, 16, 4, 64, 4096, 300, 4095, 1000),
        # the recompute of 64 windows of 32 positions in the policy's own arithmetic
        _case("attend_windows", "attend", 4, "float32", 64, 32, 8, 8, 96, 32, 0, 0),
        # whole long windows at once, odd in length, 16-bit activations
        _case("attend_whole", "attend", 4, "bfloat16", 8, 2047, 12, 12, 64, 2048, 0, 0),
        # a chunk of 500 new steps after a cached history, grouped heads
        _case("attend_chunk_gqa", "attend", 4, "bfloat16", 8, 500, 32, 8, 128, 8192, 2500, 7600),
        # patch or prompt tokens that all see each other (no causal order)
        _case("attend_full_view", "attend", 8, "float16", 32, 577, 16, 16, 64, 640, 0, 0, 0, False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "step", "step", "attend", "attend", "attend"])
    bits, dtype = rng.choice([4, 4, 8]), rng.choice(sorted(_DTYPES))
    dim = rng.choice([32, 64, 96, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8])
    window, causal = 0, True
    if kind in ("append", "read"):
        heads = kv_heads
        steps = _spread(rng, 1, 6001)
        rows = _spread(rng, 1, max(1, min(512, 36_000_000 // (steps * kv_heads * dim))))
        capacity = steps + rng.randrange(0, 700)
        low, high = (steps // 3, steps) if kind == "read" else (0, capacity - steps)
    elif kind == "step" or rng.random() < 0.5:                   # one new position a row
        steps = 1
        capacity = _spread(rng, 4, 16384)
        rows = _spread(rng, 1, max(1, min(1024, 300_000_000 // (capacity * kv_heads * dim))))
        low, high = rng.choice([0, capacity // 3, capacity - 1]), capacity - 1
        window = rng.choice([0, 0, 0, 1 + rng.randrange(capacity)])
    else:
        steps = _spread(rng, 2, 2047)
        capacity = steps + rng.choice([0, rng.randrange(0, 6000)])
        rows = _spread(rng, 1, max(1, min(256, 3_000_000_000 // (steps * capacity * heads * dim))))
        causal = rng.random() < 0.75
        low, high = 0, capacity - steps
        window = rng.choice([0, 0, 1 + rng.randrange(capacity)]) if causal else 0
    return _case("", kind, bits, dtype, rows, steps, heads, kv_heads, dim, capacity, low, high, window, causal)


# ---------------------------------------------------------------------------------------------------- plain form
def _power(e):
    """2^e for whole e in [-126, 127], from the exponent's bits."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _tables():
    """What a program keeps for 4-bit numbers: the value of each code, and the code of each magnitude's double (0, 1, 2, 3, 4, 6, 8, 12)."""
    code = torch.zeros(13, dtype=torch.uint8)
    code[[int(2 * v) for v in _E2M1]] = torch.arange(8, dtype=torch.uint8)
    return torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device="cuda"), code.cuda()


def _encode(x, bits, tables):
    """x (..., dim) -> codes uint8 (..., dim * bits / 8), scales uint8 (..., 4)."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1)
    mantissa, e = torch.frexp(top)                               # top = mantissa 2^e, 0.5 <= mantissa < 1
    e = e - 3 + (mantissa > 0.75).int() if bits == 4 else e - 9 + (mantissa > 0.875).int()
    e = e.clamp(-100, 100)
    y = x * _power(-e).unsqueeze(-1)
    if bits == 4:
        m = y.abs().clamp(max=6.0)
        m = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), torch.round(m / 2) * 2))
        c = tables[1][(2 * m).to(torch.int32)] | (torch.signbit(y).to(torch.uint8) << 3)
        c = c.flatten(-2)
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
    else:
        codes = y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    scales = torch.zeros(*top.shape[:-1], 4, dtype=torch.uint8, device=x.device)
    scales[..., :top.shape[-1]] = torch.where(torch.isfinite(top), e + 127, 255).to(torch.uint8)
    return codes, scales


def _decode(codes, scales, bits, tables):
    """-> float32 (..., dim)."""
    if bits == 4:
        y = torch.stack([tables[0][(codes & 15).to(torch.int32)], tables[0][(codes >> 4).to(torch.int32)]], -1).flatten(-2)
    else:
        y = codes.view(torch.float8_e4m3fn).float()
    y = y.unflatten(-1, (-1, BLOCK))
    s = _power(scales[..., :y.shape[-2]].to(torch.int32) - 127)
    return (y * s.unsqueeze(-1)).flatten(-2)


def _places(s):
    """Positions (rows, steps) of the new steps in their episodes' windows."""
    return s["pos"].long()[s["idx"].long()][:, None] + torch.arange(s["steps"], device=s["pos"].device)


def _plain_write(s, k, v):
    e, at = s["idx"].long()[:, None], _places(s)
    for j, x in enumerate((k, v)):
        codes, scales = _encode(x, s["bits"], s["tables"])
        s["codes"][j][e, :, at] = codes
        s["scales"][j][e, :, at] = scales


def _plain_read(s, steps, start):
    """Keys and values (rows, steps, kv_heads, dim) of positions start .. start + steps - 1, float32."""
    e, at = s["idx"].long()[:, None], start + torch.arange(steps, device=s["pos"].device)
    return [_decode(s["codes"][j][e, :, at], s["scales"][j][e, :, at], s["bits"], s["tables"]) for j in (0, 1)]


def _plain_attend(s, q):
    n, t, heads, dim = q.shape
    keys = s["max_len"]
    e = s["idx"].long()
    k, v = [_decode(s["codes"][j][e, :, :keys], s["scales"][j][e, :, :keys], s["bits"], s["tables"]) for j in (0, 1)]   # (n, kv, keys, dim)
    kv = k.shape[1]
    q = q.float().view(n, t, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    p = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    at = _places(s) if s["causal"] else _places(s)[:, -1:].expand(n, t)
    at = at.repeat_interleave(heads // kv, 1)[:, None, :, None]
    key = torch.arange(keys, device=q.device)
    seen = key <= at
    if s["window"]:
        seen = seen & (key > at - s["window"])
    p = p.masked_fill(~seen, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v)
    return o.view(n, kv, t, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(n, t, heads, dim)


# ---------------------------------------------------------------------------------------------------- inputs
def _numbers(g, shape, dtype):
    """Activations as projections give them: normal numbers, a few channels several times larger than the rest."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    gain = 1.0 + 7.0 * (torch.rand(shape[-2:], generator=g, device="cuda") > 0.97)
    return (x * gain).to(dtype)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    n, t, h, kv, d, cap = (case[f] for f in ("rows", "steps", "heads", "kv_heads", "dim", "capacity"))
    episodes = n + n // 8                                        # some of the server's episodes take no part in the call
    dtype = _DTYPES[case["dtype"]]
    s = dict(case, dtype=dtype, tables=_tables())
    s["idx"] = torch.randperm(episodes, generator=g, device="cuda")[:n].to(torch.int32)
    ends = torch.randint(case["low"], case["high"] + 1, (episodes,), generator=g, device="cuda", dtype=torch.int32)
    bytes_a_row = d * case["bits"] // 8
    s["codes"] = torch.zeros(2, episodes, kv, cap, bytes_a_row, dtype=torch.uint8, device="cuda")
    s["scales"] = torch.zeros(2, episodes, kv, cap, 4, dtype=torch.uint8, device="cuda")
    if case["kind"] != "append":                                 # the history, and behind it what earlier episodes left there
        for j in (0, 1):
            for e in range(0, episodes, 8):
                x = _numbers(g, (min(8, episodes - e), cap, kv, d), torch.float32).transpose(1, 2)
                s["codes"][j, e:e + 8], s["scales"][j, e:e + 8] = _encode(x, case["bits"], s["tables"])
    if case["kind"] == "read":
        s["count"], s["pos"] = ends[s["idx"].long()].contiguous(), torch.zeros_like(ends)
    else:
        s["pos"] = ends
        s["max_len"] = case["high"] + t                          # what the caller's own counters say: no window is longer
    if case["kind"] in ("append", "step"):                       # one product's output holds q | k | v of every new step
        s["new"] = _numbers(g, (n, t, h + 2 * kv, d), dtype)
        s["q"], s["k"], s["v"] = s["new"][:, :, :h], s["new"][:, :, h:h + kv], s["new"][:, :, h + kv:]
    elif case["kind"] == "attend":
        s["q"] = _numbers(g, (n, t, h, d), dtype)
    return s


def run(s):
    kind = s["kind"]
    if own:
        from otter_amd import ops
        codes, scales, idx, pos = s["codes"], s["scales"], s["idx"], s["pos"]
        if kind == "append":
            ops.kv_cache_write(s["k"], s["v"], codes, scales, pos, idx)
            return ops.kv_cache_read(codes, scales, s["dim"], s["steps"], pos, idx, dtype=s["dtype"])
        if kind == "read":
            return ops.kv_cache_read(codes, scales, s["dim"], s["steps"], None, idx, s["count"], dtype=s["dtype"])
        if kind == "attend":
            return ops.attn_cache(s["q"], codes, scales, pos, idx, causal=s["causal"], window=s["window"], max_len=s["max_len"])
        out = ops.attn_cache_rows(s["q"][:, 0], s["k"][:, 0], s["v"][:, 0], codes, scales, pos, idx, window=s["window"], max_len=s["max_len"])
        return out, ops.kv_cache_read(codes, scales, s["dim"], 1, pos, idx, dtype=s["dtype"])
    if kind == "append":
        _plain_write(s, s["k"], s["v"])
        return tuple(x.to(s["dtype"]) for x in _plain_read(s, s["steps"], s["pos"][s["idx"].long()][:, None]))
    if kind == "read":
        left = (torch.arange(s["steps"], device="cuda") < s["count"][:, None])[:, :, None, None]
        return tuple(torch.where(left, x, 0.0).to(s["dtype"]) for x in _plain_read(s, s["steps"], torch.zeros_like(s["idx"])[:, None]))
    if kind == "attend":
        return _plain_attend(s, s["q"]).to(s["dtype"])
    _plain_write(s, s["k"], s["v"])
    out = _plain_attend(s, s["q"])[:, 0].to(s["dtype"])
    return out, tuple(x.to(s["dtype"]) for x in _plain_read(s, 1, s["pos"][s["idx"].long()][:, None]))


# ---------------------------------------------------------------------------------------------------- sizes
def work(case):
    """Lengths at the middle of their range: what one pass reads, writes and multiplies."""
    n, t, h, kv, d = (case[f] for f in ("rows", "steps", "heads", "kv_heads", "dim"))
    size = 4 if case["dtype"] == "float32" else 2
    token = 2 * kv * (d * case["bits"] // 8 + d // BLOCK)        # one cached position: codes and scales of its keys and values
    plain = 2 * kv * d * size                                    # the same as numbers
    if case["kind"] == "append":
        return {"bytes": n * t * (plain + 2 * token + plain), "flops": n * t * kv * d * 2 * 4}
    middle = (case["low"] + case["high"]) / 2
    if case["kind"] == "read":
        return {"bytes": int(n * (middle * token + t * plain)), "flops": int(n * middle * kv * d * 2)}
    last = middle + t
    keys = min(last, case["window"] + t - 1) if case["window"] else last            # positions that any of the queries looks at
    if not case["causal"]:
        pairs = t * last
    elif case["window"]:
        pairs = sum(min(middle + i + 1, case["window"]) for i in range(t))
    else:
        pairs = t * middle + t * (t + 1) / 2
    moved = n * (keys * token + 2 * t * h * d * size)
    if case["kind"] == "step":
        moved += n * (2 * plain + 2 * token)
    return {"bytes": int(moved), "flops": int(4 * n * h * d * pairs)}


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def _value64(byte_codes, exponents, bits, dim):
    """Numbers that the stored bytes stand for, decoded field by field."""
    raw = byte_codes.to(torch.int64)
    if bits == 4:
        raw = torch.stack((raw % 16, raw // 16), -1).reshape(*raw.shape[:-1], dim)
        sign, ex, frac, low, width = raw // 8, (raw // 2) % 4, raw % 2, 1, 2.0
    else:
        sign, ex, frac, low, width = raw // 128, (raw // 8) % 16, raw % 8, 7, 8.0
    normal = (1.0 + frac.double() / width) * torch.exp2((ex - low).double())
    tiny = frac.double() / width * 2.0 ** (1 - low)
    value = torch.where(ex > 0, normal, tiny) * (1 - 2 * sign).double()
    return value * torch.exp2(exponents[..., : dim // BLOCK].double() - 127.0).repeat_interleave(BLOCK, -1)


def _nearest64(x, bits):
    """The representable number next to each of x (..., dim)."""
    shape = x.shape
    x = x.double().reshape(-1, BLOCK)
    most, digits, lowest = (6.0, 1, 0) if bits == 4 else (448.0, 3, -6)
    top = x.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(torch.where(top > 0, top / most, 2.0 ** -200))).clamp(-100, 100)
    e = torch.where(top <= most * torch.exp2(e - 1), e - 1, e)   # the logarithm's own rounding, next to a power of two
    e = torch.where(top > most * torch.exp2(e), e + 1, e).clamp(-100, 100)
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** lowest))) - digits)
    y = (torch.round(y / step) * step).clamp(-most, most)
    return (y * torch.exp2(e)).reshape(shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind, dim, bits, idx = case["kind"], case["dim"], case["bits"], s["idx"].tolist()
    if kind == "append":
        return tuple(_nearest64(s[f], bits) for f in ("k", "v"))
    if kind == "read":
        both = []
        for j in (0, 1):
            x = torch.zeros(case["rows"], case["steps"], case["kv_heads"], dim, dtype=torch.float64, device="cuda")
            for i, e in enumerate(idx):
                m = min(int(s["count"][i]), case["steps"])
                x[i, :m] = _value64(s["codes"][j, e, :, :m], s["scales"][j, e, :, :m], bits, dim).transpose(0, 1)
            both.append(x)
        return tuple(both)
    t, group = case["steps"], case["heads"] // case["kv_heads"]
    out = torch.zeros(case["rows"], t, case["heads"], dim, dtype=torch.float64, device="cuda")
    new = [_nearest64(s[f], bits) for f in ("k", "v")] if kind == "step" else None
    pos = s["pos"].tolist()
    for i, e in enumerate(idx):
        m = pos[e] + t
        k, v = (_value64(s["codes"][j, e, :, :m], s["scales"][j, e, :, :m], bits, dim) for j in (0, 1))
        if new:
            k[:, pos[e]], v[:, pos[e]] = new[0][i, 0], new[1][i, 0]
        last = torch.arange(pos[e], m, device="cuda")[:, None] if case["causal"] else torch.full((t, 1), m - 1, device="cuda")
        key = torch.arange(m, device="cuda")
        hidden = key > last
        if case["window"]:
            hidden |= key <= last - case["window"]
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        a = (s["q"][i].double().transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(dim)).masked_fill(hidden, -math.inf)
        out[i] = (torch.softmax(a, -1) @ v).transpose(0, 1)
    return (out[:, 0], tuple(new)) if new else out
