"""The quantised K/V cache on the GPU: written, read back and attended to, against a plain implementation in 64 bits."""
import math

import pytest
import torch

import kv_plain as P

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from otter_amd import _lib
    _lib.load()
    return torch.device("cuda:0")


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _new(dev, episodes, heads, capacity, d, bits, fill=0):
    return (torch.full((2, episodes, heads, capacity, d * bits // 8), fill, dtype=torch.uint8, device=dev),
            torch.full((2, episodes, heads, capacity, 4), fill, dtype=torch.uint8, device=dev))


def _filled(dev, seed, episodes, heads, capacity, d, bits):
    """A cache full of quantised random numbers with a few louder channels -> (codes, scales, k, v as doubles on the CPU)."""
    x = _randn(seed, 2, episodes, heads, capacity, d)
    x[..., ::13] *= 6
    codes, scales = P.quantise(x, bits)
    return codes.to(dev), scales.to(dev), *P.dequantise(codes, scales, bits)


# ---------------------------------------------------------------------------------------------------- write and read back
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("n,t,h", [(3, 1, 8), (2, 7, 1), (5, 33, 3)])
def test_write_then_read(dev, bits, dtype, d, n, t, h):
    from otter_amd import ops
    e, s = n + 2, t + 9
    k, v = _randn(1, n, t, h, d).to(dtype), (_randn(2, n, t, h, d) * 37).to(dtype)
    idx, pos = torch.randperm(e, generator=torch.Generator().manual_seed(3))[:n], torch.arange(e) % 10
    codes, scales = _new(dev, e, h, s, d, bits, fill=0x5a)
    before = codes.clone(), scales.clone()
    ops.kv_cache_write(k.to(dev), v.to(dev), codes, scales, _i32(pos.tolist(), dev), _i32(idx.tolist(), dev))
    want_c, want_s = before[0].cpu(), before[1].cpu()
    nb = d // 32
    for i, ep in enumerate(idx.tolist()):
        for j, x in enumerate((k, v)):
            c, sc = P.quantise(x[i].transpose(0, 1), bits)
            at = slice(int(pos[ep]), int(pos[ep]) + t)
            want_c[j, ep, :, at] = c
            want_s[j, ep, :, at, :nb] = sc[..., :nb]
    assert torch.equal(codes.cpu(), want_c)                                    # every stored byte, and nothing else touched
    assert torch.equal(scales.cpu()[..., :nb], want_s[..., :nb]) and torch.equal(scales.cpu()[..., nb:], before[1].cpu()[..., nb:])
    for out in DTYPES:
        gk, gv = ops.kv_cache_read(codes, scales, d, t, _i32(pos.tolist(), dev), _i32(idx.tolist(), dev), dtype=out)
        for got, x in ((gk, k), (gv, v)):
            assert got.dtype == out and tuple(got.shape) == (n, t, h, d)
            assert torch.equal(got.cpu(), P.dequantise(*P.quantise(x, bits), bits).to(out))


@pytest.mark.parametrize("bits", [4, 8])
def test_rounding_limits_and_non_finite_blocks(dev, bits):
    """Ties, the ends of the range, tiny and huge blocks, zeros, and blocks with a NaN or an infinity."""
    from otter_amd import ops
    d = 128
    g = P.grid(bits)
    ties = (g[1:] + g[:-1]) / 2                                                # half way between neighbours
    rows = [torch.cat([ties, -ties, g, -g, ties * (1 + 2.0 ** -20), ties * (1 - 2.0 ** -20)])]
    rows = [torch.cat([rows[0], torch.zeros(-len(rows[0]) % 31)]).view(-1, 31)]
    x = torch.cat([rows[0], torch.full((len(rows[0]), 1), float(g[-1]))], 1)   # 31 numbers and the largest code: scale 1
    x = torch.cat([x, x * 2.0 ** -90, x * 2.0 ** 99, x * 2.0 ** 110, x * 2.0 ** -120, torch.zeros(1, 32, dtype=torch.float64)])
    for top in (1.0, 1.5, 1.5 * (1 + 2.0 ** -23), 1.75, 1.75 * (1 + 2.0 ** -23), 2 - 2.0 ** -23, 1e-45, 1e-38, 3.4e38):
        x = torch.cat([x, torch.linspace(-1, 1, 32, dtype=torch.float64)[None] * top])
    for bad in (math.nan, math.inf, -math.inf):
        y = torch.ones(1, 32, dtype=torch.float64)
        y[0, 17] = bad
        x = torch.cat([x, y])
    x = torch.cat([x, torch.zeros(-len(x) % 4, 32, dtype=torch.float64)]).view(1, -1, 1, d).float()
    t = x.shape[1]
    codes, scales = _new(dev, 1, 1, t, d, bits)
    ops.kv_cache_write(x.to(dev), -x.to(dev), codes, scales)
    k, v = ops.kv_cache_read(codes, scales, d, t)
    want = P.dequantise(*P.quantise(x, bits), bits).float()
    torch.testing.assert_close(k.cpu(), want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(v.cpu(), -want, rtol=0, atol=0, equal_nan=True)
    c, s = P.quantise(x, bits)
    finite = (s != 255).repeat_interleave(codes.shape[-1] // 4, -1)
    assert torch.equal(codes[0, 0, 0].cpu()[finite[0, :, 0]], c[0, :, 0][finite[0, :, 0]]) and torch.equal(scales[0, 0, 0].cpu(), s[0, :, 0])
    h16, _ = ops.kv_cache_read(codes, scales, d, t, dtype=torch.float16)       # cut at the largest fp16 number, NaN kept
    torch.testing.assert_close(h16.cpu(), want.clamp(-65504, 65504).half(), rtol=0, atol=0, equal_nan=True)


def test_write_skips_what_lies_outside(dev):
    """Counts, positions before and behind the window, episodes that do not exist, and an episode listed twice."""
    from otter_amd import ops
    bits, d, h, s, e, t = 4, 64, 2, 10, 4, 6
    k, v = _randn(5, 6, t, h, d), _randn(6, 6, t, h, d)
    idx, pos, count = [2, -1, 0, 2, 4, 1], [8, -3, 1, 0], [6, 6, 4, 5, 6, 99]
    codes, scales = _new(dev, e, h, s, d, bits, fill=0x11)
    ops.kv_cache_write(k.to(dev), v.to(dev), codes, scales, _i32(pos, dev), _i32(idx, dev), _i32(count, dev))
    want = torch.full_like(codes.cpu(), 0x11)
    for i, ep in enumerate(idx):
        if not 0 <= ep < e or ep in idx[i + 1:]:
            continue
        for step in range(min(count[i], t)):
            at = pos[ep] + step
            if 0 <= at < s:
                want[0, ep, :, at], want[1, ep, :, at] = P.quantise(k[i, step], bits)[0], P.quantise(v[i, step], bits)[0]
    assert torch.equal(codes.cpu(), want)
    gk, gv = ops.kv_cache_read(codes, scales, d, t, _i32(pos, dev), _i32(idx, dev), _i32(count, dev))
    for i, ep in enumerate(idx):
        for step in range(t):
            at = pos[ep] + step if 0 <= ep < e else -1
            live = 0 <= at < s and step < count[i]
            ref = P.dequantise(codes[0, ep, :, at].cpu(), scales[0, ep, :, at].cpu(), bits).float() if live else torch.zeros(h, d)
            assert torch.equal(gk[i, step].cpu(), ref)
    assert tuple(ops.kv_cache_read(codes, scales, d, 0)[0].shape) == (e, 0, h, d)
    empty = torch.zeros(0, t, h, d, device=dev)
    ops.kv_cache_write(empty, empty, codes, scales, idx=_i32([], dev))
    assert torch.equal(codes.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_operands(dev, dtype):
    """Keys and values as slices of a wider buffer, in other dimension orders, and at addresses no vector load takes."""
    from otter_amd import ops
    n, t, h, d, bits = 2, 5, 3, 96, 4
    want = None
    base = _randn(7, n, t, 2, h, d).to(dtype)
    flat = torch.zeros(base.numel() + 64, dtype=dtype, device=dev)
    for form in range(4):
        if form == 0:
            x = base.to(dev)
            k, v = x[:, :, 0], x[:, :, 1]
        elif form == 1:
            k, v = (base[:, :, j].permute(2, 1, 0, 3).contiguous().to(dev).permute(2, 1, 0, 3) for j in (0, 1))
        elif form == 2:                                                         # one element off any 16-byte boundary
            flat[1:1 + base.numel()] = base.reshape(-1).to(dev)
            x = flat[1:1 + base.numel()].view(base.shape)
            k, v = x[:, :, 0], x[:, :, 1]
        else:                                                                   # rows of an odd length
            wide = torch.zeros(n, t, 2, h, d + 1, dtype=dtype, device=dev)
            wide[..., :d] = base.to(dev)
            k, v = wide[:, :, 0, :, :d], wide[:, :, 1, :, :d]
        codes, scales = _new(dev, n, h, t, d, bits)
        ops.kv_cache_write(k, v, codes, scales)
        q = k.expand(n, t, h, d)
        out = ops.attn_cache(q, codes, scales)
        if want is None:
            want = codes, scales, out
            assert torch.equal(codes[0].cpu(), P.quantise(base[:, :, 0].transpose(1, 2), bits)[0])
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(out, want[2])
    # a cache that is a slice of a larger one
    big_c, big_s = _new(dev, 5, 2 * h, t + 3, d, bits, fill=7)
    part_c, part_s = big_c[:, 1:4:2, h:], big_s[:, 1:4:2, h:]
    ops.kv_cache_write(base[:, :, 0].to(dev), base[:, :, 1].to(dev), part_c, part_s)
    assert torch.equal(part_c[:, :, :, :t], want[0]) and bool((big_c[:, ::2] == 7).all()) and bool((big_c[:, :, :h] == 7).all())
    assert torch.equal(ops.attn_cache(base[:, :, 0].to(dev), part_c, part_s), want[2])


# ---------------------------------------------------------------------------------------------------- attention
def _check(dev, seed, bits, dtype, d, n, t, heads, kv_heads, capacity, pos, idx=None, count=None, causal=True, window=0, max_len=None, scale=None,
           episodes=None):
    from otter_amd import ops
    episodes = episodes or n
    codes, scales, k, v = _filled(dev, seed, episodes, kv_heads, capacity, d, bits)
    q = _randn(seed + 1, n, t, heads, d).to(dtype)
    got = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), None if idx is None else _i32(idx, dev), None if count is None else _i32(count, dev),
                         causal=causal, window=window, max_len=max_len, scale=scale)
    assert got.dtype == dtype and tuple(got.shape) == tuple(q.shape)
    for i in range(n):
        e = i if idx is None else idx[i]
        if not 0 <= e < episodes:
            assert bool((got[i] == 0).all())
            continue
        out, a_, b_ = P.attend(q[i], k[e], v[e], pos[e], t if count is None else min(max(count[i], 0), t), causal, window,
                               capacity if max_len is None else max_len, d ** -0.5 if scale is None else scale)
        off = (got[i].double().cpu() - out).abs()
        tol = P.tolerance(out, a_, b_, dtype)
        assert bool((off <= tol).all()), (i, float((off / tol).max()), float(off.max()))
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2), (7, 1), (40, 2)])
def test_attend_one_position(dev, bits, dtype, d, heads, kv_heads):
    """Lengths from one key to a few tiles, on, before and behind a tile's end."""
    lengths = [0, 1, 30, 31, 32, 33, 63, 64, 95, 130]
    _check(dev, 11, bits, dtype, d, len(lengths), 1, heads, kv_heads, 131, lengths)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("t,heads,kv_heads,capacity", [(2, 2, 2, 3), (5, 12, 3, 70), (17, 2, 2, 33), (50, 6, 2, 64), (33, 4, 4, 257)])
def test_attend_many_positions(dev, bits, dtype, d, t, heads, kv_heads, capacity):
    pos = [0, capacity - t, (capacity - t) // 2]
    _check(dev, 12, bits, dtype, d, 3, t, heads, kv_heads, capacity, pos)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000])
@pytest.mark.parametrize("t", [1, 40])
def test_attend_window(dev, dtype, window, t):
    _check(dev, 13, 4, dtype, 96, 4, t, 4, 2, 300, [0, 20, 150, 260], window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_all_see_all_and_ragged_counts(dev, dtype):
    t = 37
    _check(dev, 14, 8, dtype, 64, 5, t, 4, 4, 80, [0, 10, 43, 3, 0], causal=False)
    _check(dev, 15, 4, dtype, 64, 5, t, 4, 4, 80, [0, 10, 43, 3, 0], count=[0, 1, 37, 36, 17], causal=False)
    got = _check(dev, 16, 4, dtype, 64, 5, t, 4, 2, 80, [0, 10, 43, 3, 0], count=[0, 1, 37, 36, 99])
    assert bool((got[0] == 0).all()) and bool((got[1, 1:] == 0).all()) and bool((got[3, 36:] == 0).all())


@pytest.mark.parametrize("t", [1, 20])
def test_attend_rows_that_see_nothing(dev, t):
    """Positions before the window, beyond the capacity and beyond max_len; episodes that do not exist or repeat."""
    _check(dev, 17, 4, torch.float32, 64, 7, t, 2, 2, 50, [-5, -30, 49, 60, 2000000000, -2000000000], idx=[3, 0, -1, 1, 6, 0, 2], episodes=6)
    _check(dev, 18, 4, torch.bfloat16, 64, 4, t, 2, 2, 50, [0, 5, 20, 40], max_len=18, window=6)
    _check(dev, 19, 8, torch.float16, 32, 4, t, 2, 2, 50, [4, 5, 20, 40], max_len=1, scale=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits,d,heads,kv_heads,t", [(4, 128, 4, 1, 1), (8, 96, 2, 2, 1), (4, 64, 2, 1, 9), (4, 96, 16, 1, 7)])
def test_attend_split_keys(dev, dtype, bits, d, heads, kv_heads, t):
    """Few rows over long histories: the keys are shared by waves and workgroups, some of them past the row's length."""
    for pos, cap, kw in (([2999, 5, 600], 3200, {}), ([3100, 255, 2047], 3200, {"window": 700}), ([1500, 0, 900], 3200, {"max_len": 1501})):
        _check(dev, 20, bits, dtype, d, 3, t, heads, kv_heads, cap, pos, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits,d,heads,kv_heads,t,capacity,kw", [
    (4, 64, 2, 2, 130, 1500, {}), (8, 96, 4, 2, 101, 1300, {"window": 333}), (4, 128, 3, 1, 67, 2100, {}), (8, 32, 2, 1, 200, 900, {"max_len": 800}),
    (4, 96, 2, 2, 140, 700, {"causal": False})])
def test_attend_chunk_after_a_long_history(dev, dtype, bits, d, heads, kv_heads, t, capacity, kw):
    """Many columns, few rows: workgroups that convert the tiles together, and several of them share the keys."""
    _check(dev, 26, bits, dtype, d, 2, t, heads, kv_heads, capacity, [capacity - t, capacity // 3], **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,heads,kv_heads,t", [(2, 3, 3, 150), (17, 7, 1, 40), (63, 2, 2, 130), (64, 4, 2, 129), (65, 2, 2, 130)])
def test_attend_chunks_after_histories_of_any_length(dev, dtype, n, heads, kv_heads, t):
    """Workgroups are dealt out by the length of their row's history: none, equal, differing ones, some before the window or past its end,
    rows that do not exist, short counts; every output of every row is there."""
    rng = torch.Generator().manual_seed(n)
    cap = 420
    pos = torch.randint(0, cap - t + 1, (n,), generator=rng).tolist()
    _check(dev, 33, 4, dtype, 64, n, t, heads, kv_heads, cap, pos)
    _check(dev, 34, 8, dtype, 32, n, t, heads, kv_heads, cap, [0] * n)
    idx = torch.randperm(n, generator=rng).tolist()
    idx[n // 2], idx[n - 1] = -1, n + 5
    odd = [(-2000000000, -40, cap - 1, cap + 7, 2000000000)[j % 5] if j % 3 == 0 else p for j, p in enumerate(pos)]
    count = torch.randint(-1, t + 2, (n,), generator=rng).tolist()
    _check(dev, 35, 4, dtype, 96, n, t, heads, kv_heads, cap, odd, idx=idx, count=count, max_len=cap - 50)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,heads", [(1, 2), (40, 2), (3, 4), (100, 4)])
def test_not_a_number_in_masked_places(dev, dtype, t, heads):
    """Rows that a query must not see hold NaN (and codes and scales that the writer never makes): before its window, behind its
    position, behind the length, in other episodes.  Where it does see one, its output is NaN as the formula's is."""
    from otter_amd import ops
    bits, d, h, s, n = 4, 64, 2, 220, 3
    pos, window = [10, 40, 110], 25
    codes, scales, k, v = _filled(dev, 21, n, h, s, d, bits)
    q = _randn(22, n, t, heads, d).to(dtype)
    want = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), window=window)
    for i in range(n):
        first, last = max(0, pos[i] - window + 1), pos[i] + t - 1
        hidden = torch.ones(s, dtype=torch.bool)
        hidden[first:last + 1] = False
        scales[:, i, :, hidden.to(dev)] = 255
        scales[:, i, :, s - 1] = 254
        codes[:, i, :, hidden.to(dev)] = 0x77
    got = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), window=window)
    assert torch.equal(got, want)
    # a value row of the last query only: everyone else keeps its result, the last one is NaN in that block and nowhere else
    saved = scales.clone()
    for i in range(n):
        scales[1, i, :, pos[i] + t - 1, 1] = 255
    got = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), window=window)
    assert torch.equal(got[:, :-1], want[:, :-1])
    assert torch.equal(got[:, -1, :, :32], want[:, -1, :, :32]) and bool(torch.isnan(got[:, -1, :, 32:]).all())
    scales.copy_(saved)
    for i in range(n):
        scales[0, i, :, pos[i] + t - 1, 0] = 255                               # a key row: its score, hence the whole output
    got = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), window=window)
    assert torch.equal(got[:, :-1], want[:, :-1]) and bool(torch.isnan(got[:, -1]).all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,heads,kv_heads", [(1, 2, 2), (1, 8, 2), (50, 2, 2), (200, 4, 2)])
@pytest.mark.parametrize("power", [-60, -22, -12, 8, 12, 30])
def test_values_of_any_magnitude(dev, bits, dtype, t, heads, kv_heads, power):
    """Value blocks (and, at the small powers, key blocks) whose scales leave the range of one operand type or another: all of
    them, and single rows among ordinary ones."""
    from otter_amd import ops
    d, s, n = 64, 260, 2
    pos = [s - t, 0]
    x = _randn(27, 2, n, kv_heads, s, d)
    x[1, 0] *= 2.0 ** power                                                     # episode 0: every value
    x[1, 1, :, 3::17] *= 2.0 ** power                                           # episode 1: some rows
    if power < 0:
        x[0, 1, :, 2::19] *= 2.0 ** power
    codes, scales = P.quantise(x, bits)
    k, v = P.dequantise(codes, scales, bits)
    q = _randn(28, n, t, heads, d).to(dtype)
    got = ops.attn_cache(q.to(dev), codes.to(dev), scales.to(dev), _i32(pos, dev))
    for i in range(n):
        out, a_, b_ = P.attend(q[i], k[i], v[i], pos[i], t, True, 0, s, d ** -0.5)
        tol = P.tolerance(out, a_, b_, dtype)
        fits = out.abs() <= torch.finfo(dtype).max * 0.999
        assert bool(((got[i].double().cpu() - out).abs() <= tol)[fits].all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,heads", [(1, 2), (1, 4), (1, 16), (40, 2), (3, 4), (100, 4)])
def test_codes_that_are_no_numbers_in_masked_places(dev, dtype, t, heads):
    """8 bits have codes for NaN, which the writer makes only in blocks whose scale says so.  Memory that nobody has written may
    hold them with any scale: before the window and behind the end it changes nothing."""
    from otter_amd import ops
    bits, d, h, s, n = 8, 96, 2, 420, 3
    pos, window = [10, 75, 310], 25
    codes, scales, k, v = _filled(dev, 31, n, h, s, d, bits)
    q = _randn(32, n, t, heads, d).to(dtype)
    want = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), window=window)
    for i in range(n):
        hidden = torch.ones(s, dtype=torch.bool)
        hidden[max(0, pos[i] - window + 1):pos[i] + t] = False
        codes[:, i, :, hidden.to(dev)] = 0x7f if i % 2 else 0xff
        scales[:, i, :, hidden.to(dev)] = 255 if i == 2 else 130
    got = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev), window=window)
    assert torch.equal(got, want)


@pytest.mark.parametrize("t,heads", [(1, 2), (1, 8), (20, 2), (100, 2)])
def test_half_precision_outputs_are_cut(dev, t, heads):
    """Outputs past fp16's largest number: that number, as a read gives it, with one split of the keys and with several."""
    from otter_amd import ops
    for s in (64, 2200):
        codes, scales = _new(dev, 1, 2, s, 64, 4)
        codes[:, :, :, :, ::2], codes[:, :, :, :, 1::2] = 0x77, 0xff                    # 6, 6, -6, -6, ...
        scales[0], scales[1] = 127, 127 + 14
        q = torch.zeros(1, t, heads, 64, dtype=torch.float16, device=dev)
        got = ops.attn_cache(q, codes, scales, _i32([s - t], dev))
        sign = torch.tensor([1.0, 1.0, -1.0, -1.0]).repeat(16)
        want = (65504.0 * sign).repeat(1, t, heads, 1)
        want[:, :max(0, t - s)] = 0                                                     # steps before position 0 see nothing
        assert torch.equal(got.float().cpu(), want)


# ---------------------------------------------------------------------------------------------------- append and attend in one call
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,capacity", [(96, 8, 8, 32), (64, 4, 4, 130), (128, 8, 2, 1100), (32, 40, 1, 600)])
def test_append_and_attend_is_write_then_attend(dev, bits, dtype, d, heads, kv_heads, capacity):
    from otter_amd import ops
    lengths = [0, 1, capacity - 1, capacity // 2, 31, capacity, -1, 5]          # the sixth is full, the seventh before the window
    e = len(lengths)
    idx = [3, 0, 7, 9, 5, 6, 2, 1, 4, 7]                                        # 9 does not exist, 7 comes twice
    codes, scales, _, _ = _filled(dev, 23, e, kv_heads, capacity, d, bits)
    fresh = _randn(24, len(idx), heads + 2 * kv_heads, d).to(dtype).to(dev)
    q, k, v = fresh[:, :heads], fresh[:, heads:heads + kv_heads], fresh[:, heads + kv_heads:]
    c2, s2 = codes.clone(), scales.clone()
    ops.kv_cache_write(k.unsqueeze(1), v.unsqueeze(1), c2, s2, _i32(lengths, dev), _i32(idx, dev))
    for kw in ({}, {"window": 20}, {"max_len": capacity // 2 + 1}):
        want = ops.attn_cache(q.unsqueeze(1), c2, s2, _i32(lengths, dev), _i32(idx, dev), **kw).squeeze(1)
        c1, s1 = codes.clone(), scales.clone()
        got = ops.attn_cache_rows(q, k, v, c1, s1, _i32(lengths, dev), _i32(idx, dev), **kw)
        assert torch.equal(c1, c2) and torch.equal(s1, s2)
        assert torch.equal(got, want)


def test_a_run_of_steps_as_a_rollout_makes_them(dev):
    """Episodes of different lengths grow step by step through the fused call; the result of every step, and the cache at the end,
    are those of the plain implementation on the numbers that went in."""
    from otter_amd import ops
    bits, d, h, s, e = 4, 96, 2, 40, 3
    codes, scales = _new(dev, e, h, s, d, bits, fill=255)                       # never written: must never be seen
    lens = [0, 0, 0]
    hist = [[[], []] for _ in range(e)]
    for step in range(36):
        rows = [i for i in range(e) if (step + i) % (i + 1) == 0]
        x = _randn(100 + step, len(rows), 3 * h, d)
        got = ops.attn_cache_rows(*(x[:, j * h:(j + 1) * h].to(dev) for j in range(3)), codes, scales, _i32(lens, dev), _i32(rows, dev))
        for i, ep in enumerate(rows):
            for j in (0, 1):
                hist[ep][j].append(P.dequantise(*P.quantise(x[i, (1 + j) * h:(2 + j) * h], bits), bits))
            k, v = (torch.stack(hist[ep][j], 1) for j in (0, 1))
            out, a_, b_ = P.attend(x[i:i + 1, :h], k, v, lens[ep], 1, True, 0, s, d ** -0.5)
            assert bool(((got[i].double().cpu() - out[0]).abs() <= P.tolerance(out, a_, b_, torch.float32)[0]).all())
            lens[ep] += 1
    k, v = ops.kv_cache_read(codes, scales, d, s, count=_i32(lens, dev))
    for ep in range(e):
        assert torch.equal(k[ep, :lens[ep]].double().cpu(), torch.stack(hist[ep][0], 0)) and bool((v[ep, lens[ep]:] == 0).all())


def test_captured_and_replayed(dev):
    """The calls record into a HIP graph (with the split path's scratch in the graph's own pool), follow the lengths of each
    replay, and two graphs replayed on two streams do not disturb each other."""
    from otter_amd import ops
    bits, d, h, s, n = 4, 64, 2, 2048, 2
    graphs = []
    for seed in (1, 2):
        codes, scales, _, _ = _filled(dev, 30 + seed, n, h, s, d, bits)
        x = _randn(40 + seed, n, 3 * h, d).to(dev)
        pos = _i32([0, 0], dev)
        args = (x[:, :h], x[:, h:2 * h], x[:, 2 * h:], codes, scales, pos)
        ops.attn_cache_rows(*args)                                              # code objects loaded before the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.attn_cache_rows(*args)
            back = ops.kv_cache_read(codes, scales, d, 1, pos)
        graphs.append((g, args, out, back, torch.cuda.Stream()))
    for lengths in ([5, 2047], [1000, 1], [2000, 1999], [31, 32]):
        for g, args, *_ in graphs:
            args[5].copy_(_i32(lengths, dev))
            args[0].add_(0.125)
        torch.cuda.synchronize()
        for g, args, out, back, stream in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for g, args, out, back, stream in graphs:
            c, sc = args[3].clone(), args[4].clone()
            assert torch.equal(out, ops.attn_cache_rows(*args[:3], c, sc, args[5]))
            want = ops.kv_cache_read(c, sc, d, 1, args[5])
            assert torch.equal(back[0], want[0]) and torch.equal(back[1], want[1])


def test_runs_on_the_current_stream(dev):
    from otter_amd import ops
    codes, scales, _, _ = _filled(dev, 50, 2, 2, 300, 64, 4)
    q = _randn(51, 2, 1, 2, 64).to(dev)
    want = ops.attn_cache(q, codes, scales, _i32([299, 100], dev))
    side = torch.cuda.Stream()
    pos, late = _i32([0, 0], dev), _i32([299, 100], dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        pos.copy_(late)
        got = ops.attn_cache(q, codes, scales, pos)
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_past_32_bits(dev):
    """An episode whose rows lie more than 4 GiB into the cache."""
    from otter_amd import ops
    bits, d, h, s = 8, 128, 2, 1 << 20
    e = 20                                                                      # 5.4 GB of key codes
    codes = torch.zeros(2, e, h, s, d, dtype=torch.uint8, device=dev)
    scales = torch.zeros(2, e, h, s, 4, dtype=torch.uint8, device=dev)
    x = _randn(60, 1, 300, 3 * h, d).to(dev)
    pos = torch.zeros(e, dtype=torch.int32, device=dev)
    pos[e - 1] = s - 300
    idx = _i32([e - 1], dev)
    ops.kv_cache_write(x[:, :, h:2 * h], x[:, :, 2 * h:], codes, scales, pos, idx)
    got = ops.attn_cache(x[:, :, :h], codes, scales, pos, idx, window=300)
    small = _new(dev, 1, h, 300, d, bits)
    ops.kv_cache_write(x[:, :, h:2 * h], x[:, :, 2 * h:], *small)
    assert torch.equal(codes[:, -1, :, -300:], small[0][:, 0]) and int(codes[:, :-1].max()) == 0
    back = ops.kv_cache_read(codes, scales, d, 300, pos, idx)
    assert torch.equal(back[0], ops.kv_cache_read(*small, d, 300)[0])
    k, v = P.dequantise(small[0].cpu(), small[1].cpu(), bits)
    for t in (0, 150, 299):                                                     # the histories before them are zeros outside the window's reach
        out, a_, b_ = P.attend(x[0, t:t + 1, :h].cpu(), torch.cat([torch.zeros(h, 300, d, dtype=torch.float64), k[0]], 1),
                               torch.cat([torch.zeros(h, 300, d, dtype=torch.float64), v[0]], 1), 300 + t, 1, True, 300, 600, d ** -0.5)
        assert bool(((got[0, t:t + 1].double().cpu() - out).abs() <= P.tolerance(out, a_, b_, torch.float32)).all())


def test_the_compiled_way_and_the_other_agree(dev, monkeypatch):
    """The same calls with the binding and without: equal outputs and caches; ordinary calls are taken by it, refusals raise the same."""
    from otter_amd import _lib, ops

    class Taken:
        def __init__(self, inner):
            self.inner, self.none = inner, 0

        def __getattr__(self, name):
            def call(*a):
                got = getattr(self.inner, name)(*a)
                self.none += got is None
                return got
            return call

    class Never:
        def __getattr__(self, name):
            return lambda *a: None

    n, t, h, hq, d, cap = 5, 3, 2, 4, 96, 700
    pos, idx, count = _i32([0, 650, 690, 3, 100, 50], dev), _i32([4, 0, 2, -1, 5], dev), _i32([3, 2, 0, 1, 9], dev)
    wide = _randn(41, n, t, hq + 2 * h, d).to(dev)

    def run(dtype, bits):
        codes, scales = _new(dev, 6, h, cap, d, bits)
        x = wide.to(dtype)
        q, k, v = x[:, :, :hq], x[:, :, hq:hq + h], x[:, :, hq + h:]
        ops.kv_cache_write(k, v, codes, scales, pos, idx, count)
        ops.kv_cache_write(k, v, codes[:, :5], scales[:, :5])
        out = [*ops.kv_cache_read(codes, scales, d, t, pos, idx, count, dtype=dtype), *ops.kv_cache_read(codes, scales, d, 2), *ops.kv_cache_read(codes, scales, d, 2, n_rows=4)]
        out += [ops.attn_cache(q, codes, scales, pos, idx, count), ops.attn_cache(q, codes, scales, pos, idx, causal=False, window=9, scale=0.3, max_len=600),
                ops.attn_cache(q, codes, scales), ops.attn_cache(q[:1, :1], codes, scales, pos, window=1 << 40, max_len=1 << 30)]
        out += [ops.attn_cache_rows(q[:, 0], k[:, 0], v[:, 0], codes, scales, pos, idx, window=5), ops.attn_cache_rows(q[:, 1], k[:, 1], v[:, 1], codes, scales, scale=1)]
        return [*out, codes, scales]

    taken = Taken(_lib.kv_binding())
    for dtype in DTYPES:
        for bits in (4, 8):
            monkeypatch.setattr(_lib, "_binding", taken)
            got = run(dtype, bits)
            monkeypatch.setattr(_lib, "_binding", Never())
            want = run(dtype, bits)
            assert len(got) == len(want) and all(a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b) for a, b in zip(got, want))
    assert taken.none == 1 * 6                                                   # (the window past 31 bits is left to the other way)
    monkeypatch.setattr(_lib, "_binding", taken)
    codes, scales = _new(dev, 2, h, 8, d, 4)
    q, k = torch.zeros(2, 1, hq, d, device=dev), torch.zeros(2, 1, h, d, device=dev)
    for call, error in ((lambda: ops.kv_cache_write(k[:, :, :1], k, codes, scales), ValueError), (lambda: ops.kv_cache_write(k, k.half(), codes, scales), TypeError),
                        (lambda: ops.kv_cache_write(k, k, codes, scales, _i32([0], dev)), ValueError), (lambda: ops.kv_cache_read(codes, scales, 64, 1), ValueError),
                        (lambda: ops.attn_cache(q, codes, scales, scale=-1.0), ValueError), (lambda: ops.attn_cache(q[:, :, :3], codes, scales), ValueError),
                        (lambda: ops.attn_cache(q, codes, scales, max_len=0), ValueError), (lambda: ops.attn_cache(q, codes, scales, window=-1), ValueError),
                        (lambda: ops.kv_cache_write(k, k, codes[:, :1].expand(-1, 2, -1, -1, -1), scales[:, :1].expand(-1, 2, -1, -1, -1)), ops.OtterHipError),
                        (lambda: ops.attn_cache_rows(q[:, 0], k[:, 0], k[:1, 0], codes, scales), ValueError), (lambda: ops.kv_cache_write(k, k, codes.cpu(), scales), ops.OtterHipError)):
        with pytest.raises(error):
            call()
    assert ops.attn_cache(q[:0], codes, scales).shape == (0, 1, hq, d) and ops.kv_cache_read(codes, scales, d, 0)[0].shape == (2, 0, h, d)
    assert bool((codes == 0).all())
