"""Blocks at the lowest exponent, -100: zeros, or numbers up to 448 * 2^-100 (8 bits) and 6 * 2^-100 (4 bits).  bf16 and fp32 outputs hold
such numbers, and every form of the attention returns them."""
import pytest
import torch

import kv_plain as P
from test_gpu_kv_cache import DTYPES, _i32, _randn, dev  # noqa: F401

pytestmark = pytest.mark.gpu
POWER = {4: -99, 8: -95}                                                        # of the numbers that get the scale byte 27


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("t,heads", [(1, 2), (1, 8), (3, 4), (40, 2), (100, 4)])
def test_values_at_the_lowest_exponent(dev, bits, dtype, d, t, heads):
    """Every value of episode 0; the last block of 32 of episode 1's values, with zeros in some rows; the values of one row of episode 2,
    whose others are zeros; episode 3: ordinary values between rows of zeros.  Its bits do not change with what stands for the zeros."""
    from otter_amd import ops
    h, s, n = 2, 200, 4
    pos = [s - t, 100, 90, 70]
    x = _randn(81, 2, n, h, s, d)
    x[1, 0] *= 2.0 ** POWER[bits]
    x[1, 1, :, :, d - 32:] *= 2.0 ** POWER[bits]
    x[1, 1, :, 5::9] = 0
    one = x[1, 2, :, 60].clone() * 2.0 ** POWER[bits]
    x[1, 2] = 0
    x[1, 2, :, 60] = one
    x[1, 3, :, ::3] = 0
    codes, scales = P.quantise(x, bits)
    assert int(scales[1, 0, :, :, 0].float().mode().values.max()) == 27 and int(scales[1, 2, 0, 60, 0]) == 27 and int(scales[1, 3, 0, 0, 0]) == 27
    k, v = P.dequantise(codes, scales, bits)
    q = _randn(82, n, t, heads, d).to(dtype)
    got = ops.attn_cache(q.to(dev), codes.to(dev), scales.to(dev), _i32(pos, dev))
    for i in range(n):
        out, a_, b_ = P.attend(q[i], k[i], v[i], pos[i], t, True, 0, s, d ** -0.5)
        off = (got[i].double().cpu() - out).abs()
        tol = P.tolerance(out, a_, b_, dtype)
        assert bool((off <= tol).all()), (i, float((off / tol).max()))
    # (the blocks of zeros in ordinary scales: the same numbers, so the same bits)
    s2 = scales.clone()
    zero_rows = (x[1, 3] == 0).all(-1)                                          # (h, s)
    s2[1, 3][zero_rows] = torch.tensor([127] * (d // 32) + [0] * (4 - d // 32), dtype=torch.uint8)
    again = ops.attn_cache(q.to(dev), codes.to(dev), s2.to(dev), _i32(pos, dev))
    assert torch.equal(again, got)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("t", [1, 40, 100])
def test_keys_at_the_lowest_exponent(dev, bits, t):
    """Keys of that size under a scale that makes their scores ordinary numbers again."""
    from otter_amd import ops
    d, h, s = 64, 2, 150
    x = _randn(83, 2, 1, h, s, d)
    x[0] *= 2.0 ** POWER[bits]
    x[0, 0, :, 7::11] = 0
    codes, scales = P.quantise(x, bits)
    assert int(scales[0, 0, :, :, :2].max()) <= 28
    k, v = P.dequantise(codes, scales, bits)
    q = _randn(84, 1, t, h, d)
    scale = 2.0 ** -POWER[bits] / 8
    for dtype in DTYPES:
        qd = q.to(dtype)
        got = ops.attn_cache(qd.to(dev), codes.to(dev), scales.to(dev), _i32([s - t], dev), scale=scale)
        out, a_, b_ = P.attend(qd[0], k[0], v[0], s - t, t, True, 0, s, scale)
        off = (got[0].double().cpu() - out).abs()
        tol = P.tolerance(out, a_, b_, dtype)
        assert bool((off <= tol).all()), (dtype, float((off / tol).max()))
