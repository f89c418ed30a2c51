"""Blocks whose scale byte alone says that they are no numbers (255; their codes may be anything), seen by some queries: every form of the
attention gives what the formula gives on what a read returns."""
import math

import pytest
import torch

import kv_plain as P
from test_gpu_kv_cache import DTYPES, _filled, _i32, _randn, dev  # noqa: F401

pytestmark = pytest.mark.gpu


# (one position on the vector unit, one with a group's heads on the matrix unit, up to 32 columns, and more: four waves a tile)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("t,heads", [(1, 2), (1, 8), (3, 4), (40, 2), (100, 4)])
def test_a_marked_block_that_is_seen(dev, bits, dtype, d, t, heads):
    """Key and value blocks with ordinary codes and scale byte 255, at the first, a middle and the last position that a row sees: the
    columns that see them are NaN (a value block: in that block), the others are the formula's."""
    from otter_amd import ops
    h, s, n = 2, 260, 3
    pos = [s - t, 150, 0]
    codes, scales, k, v = _filled(dev, 71, n, h, s, d, bits)
    q = _randn(72, n, t, heads, d).to(dtype)
    spots = {0: 130, 1: 150 + t - 1, 2: 0}
    want = {i: P.attend(q[i], k[i], v[i], pos[i], t, True, 0, s, d ** -0.5) for i in spots}
    for kv in (0, 1):
        for block in {0, d // 32 - 1}:
            sc = scales.clone()
            for i, at in spots.items():
                sc[kv, i, :, at, block] = 255
            read = ops.kv_cache_read(codes, sc, d, s)
            got = ops.attn_cache(q.to(dev), codes, sc, _i32(pos, dev)).double().cpu()
            for i, at in spots.items():
                numbers = read[kv][i].cpu()
                assert bool(torch.isnan(numbers[at, :, 32 * block:32 * block + 32]).all()) and int(torch.isnan(numbers).sum()) == h * 32
                out, a_, b_ = want[i]
                sees = (pos[i] + torch.arange(t) >= at)[:, None, None].expand(t, heads, d)
                gone = sees if kv == 0 else sees & ((torch.arange(d) // 32) == block)
                assert torch.equal(torch.isnan(got[i]), gone), (kv, block, i)
                off = (got[i] - out).abs()
                assert bool((off <= P.tolerance(out, a_, b_, dtype))[~gone].all()), (kv, block, i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,heads", [(1, 2), (1, 8), (40, 2), (100, 4)])
def test_marked_by_the_plain_writer(dev, dtype, t, heads):
    """The plain writer stores an infinity as the largest code under the byte 255, this library's as a NaN code: read and attended to alike."""
    from otter_amd import ops
    bits, d, h, s, n = 8, 64, 2, 130, 2
    x = _randn(73, 2, n, h, s, d)
    x[0, 0, :, 20, 5], x[0, 1, :, 70, 40] = math.inf, -math.inf
    codes, scales = (y.to(dev) for y in P.quantise(x, bits))
    c2, s2 = torch.zeros_like(codes), torch.zeros_like(scales)
    ops.kv_cache_write(x[0].transpose(1, 2).to(dev), x[1].transpose(1, 2).to(dev), c2, s2)
    assert torch.equal(s2, scales) and not torch.equal(c2, codes)
    q = _randn(74, n, t, heads, d).to(dtype).to(dev)
    pos = _i32([s - t, 20], dev)
    for a, b in zip(ops.kv_cache_read(codes, scales, d, s), ops.kv_cache_read(c2, s2, d, s)):
        assert torch.equal(a.nan_to_num(7e9), b.nan_to_num(7e9))
    one, two = ops.attn_cache(q, codes, scales, pos), ops.attn_cache(q, c2, s2, pos)
    assert bool(torch.isnan(one[0]).all()) and torch.equal(one.nan_to_num(6e4), two.nan_to_num(6e4))
