"""Calls of the quantised K/V history as programs make them: very many rows, recorded into graphs, on two streams, again and again; and the
arithmetic of the forms that hold the weights in two terms."""
import pytest
import torch

import kv_plain as P
from test_gpu_kv_cache import DTYPES, _filled, _i32, _new, _randn, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_dimension(dev):
    """70001 episodes: the writer's and the reader's rows go round the grid's third dimension, listed in another order and not."""
    from otter_amd import ops
    n, h, d, s, bits = 70001, 1, 32, 2, 4
    x = _randn(91, 3, n, 1, h, d).to(dev)
    codes, scales = _new(dev, n, h, s, d, bits)
    pos = (torch.arange(n, dtype=torch.int32) % 2).to(dev)
    ops.kv_cache_write(x[1], x[2], codes, scales, pos)
    want_c, want_s = P.quantise(x[1, :, 0].cpu(), bits)
    at = pos.long().cpu()
    assert torch.equal(codes[0].cpu()[torch.arange(n), :, at], want_c) and torch.equal(scales[0].cpu()[torch.arange(n), :, at, 0], want_s[..., 0])
    back = ops.kv_cache_read(codes, scales, d, 1, pos)
    assert torch.equal(back[0][:, 0].cpu(), P.dequantise(want_c, want_s, bits).float())
    out = ops.attn_cache(x[0], codes, scales, pos, window=1)                     # one key: its value row
    torch.testing.assert_close(out, back[1], rtol=2.0 ** -20, atol=0)
    idx = torch.randperm(n, generator=torch.Generator().manual_seed(92)).to(torch.int32).to(dev)
    some = idx[:66000].contiguous()
    c2, s2 = _new(dev, n, h, s, d, bits)
    ops.kv_cache_write(x[1][some.long()], x[2][some.long()], c2, s2, pos, some)
    left = idx[66000:].long()
    assert torch.equal(c2[:, some.long()], codes[:, some.long()]) and int(c2[:, left].max()) == 0


def _set(codes, scales, k, v, bits):
    for j, x in enumerate((k, v)):
        c, s = P.quantise(x, bits)
        codes[j].copy_(c)
        scales[j].copy_(s)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_columns_captured_and_replayed(dev, bits, dtype):
    """A chunk's attention in a graph: histories of other lengths and values of another size -- ordinary, past the range of one operand type,
    with zeros -- in every replay give what an eager call gives."""
    from otter_amd import ops
    n, t, h, d, s = 3, 70, 2, 64, 300
    codes, scales = _new(dev, n, h, s, d, bits)
    x = _randn(93, 2, n, h, s, d)
    _set(codes, scales, x[0], x[1], bits)
    q, pos = _randn(94, n, t, 2 * h, d).to(dtype).to(dev), _i32([0, 100, 230], dev)
    ops.attn_cache(q, codes, scales, pos)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.attn_cache(q, codes, scales, pos)
    for lengths, power, zeros in (([0, 100, 230], 0, 0), ([230, 0, 31], 30, 0), ([5, 64, 200], 0, 7), ([1, 2, 3], -60, 7), ([0, 100, 230], 0, 0)):
        y = x.clone()
        y[1] *= 2.0 ** power
        if zeros:
            y[:, :, :, ::zeros] = 0
        _set(codes, scales, y[0], y[1], bits)
        pos.copy_(_i32(lengths, dev))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attn_cache(q, codes, scales, pos))
        k, v = P.dequantise(codes, scales, bits)[0], P.dequantise(codes, scales, bits)[1]
        want, a_, b_ = P.attend(q[1].cpu(), k[1], v[1], lengths[1], t, True, 0, s, d ** -0.5)
        fits = want.abs() <= torch.finfo(dtype).max * 0.999
        assert bool(((out[1].double().cpu() - want).abs() <= P.tolerance(want, a_, b_, dtype))[fits].all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,heads,kv_heads,s", [(1, 2, 2, 3000), (1, 8, 2, 3000), (20, 2, 2, 900), (150, 4, 2, 1500)])
def test_calls_repeat_bit_for_bit_on_two_streams(dev, dtype, t, heads, kv_heads, s):
    """One cache attended to from two streams at once, several times, with the keys split and not: always the same bits."""
    from otter_amd import ops
    codes, scales, _, _ = _filled(dev, 95, 2, kv_heads, s, 64, 8)
    q, pos = _randn(96, 2, t, heads, 64).to(dtype).to(dev), _i32([s - t, s // 3], dev)
    want = ops.attn_cache(q, codes, scales, pos)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(ops.attn_cache(q, codes, scales, pos))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("t,heads,kv_heads", [(1, 2, 2), (1, 4, 2), (1, 16, 2), (16, 2, 2), (8, 8, 2)])
def test_two_terms_a_weight_in_the_forms_for_few_columns(dev, bits, d, t, heads, kv_heads):
    """Up to 32 columns, and one position, bf16 activations: a weight is fp32 on the vector unit and two bf16 terms on the matrix unit.  The
    first is off by at most half a step, 2^-8 of the weight, the second by 2^-8 of that: 2^-16, where more columns have 2^-11."""
    from otter_amd import ops
    n, s = 3, 333
    codes, scales, k, v = _filled(dev, 97, n, kv_heads, s, d, bits)
    q, pos = _randn(98, n, t, heads, d).bfloat16(), [s - t, 100, 0]
    got = ops.attn_cache(q.to(dev), codes, scales, _i32(pos, dev))
    for i in range(n):
        out, a_, b_ = P.attend(q[i], k[i], v[i], pos[i], t, True, 0, s, d ** -0.5)
        tol = a_ * (2 * b_ + 2.0 ** -16) * 1.01 + out.abs() * 2.0 ** -8 + torch.finfo(torch.bfloat16).tiny
        assert bool(((got[i].double().cpu() - out).abs() <= tol).all())
