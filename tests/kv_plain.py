"""Plain 64-bit restatement of the quantised K/V cache and of the attention over it, for the tests (CPU tensors throughout)."""
import math

import torch

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def grid(bits):
    """Every non-negative number a code can stand for, in order (the even ones are the codes with an even mantissa)."""
    if bits == 4:
        return torch.tensor(E2M1, dtype=torch.float64)
    return torch.tensor([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:-1], dtype=torch.float64)


def quantise(x, bits):
    """x (..., dim) -> (codes uint8 (..., dim * bits / 8), scale bytes uint8 (..., 4)): the definition, by search over the grid."""
    x = x.double().cpu()
    blocks = x.unflatten(-1, (-1, BLOCK))
    g = grid(bits)
    top = blocks.abs().amax(-1)
    ok = torch.isfinite(blocks).all(-1)
    top = torch.where(ok, top, 0.0)
    powers = 2.0 ** torch.arange(-100, 101, dtype=torch.float64)
    e = torch.searchsorted(g[-1] * powers, top.contiguous()).clamp(max=200)            # first power with top <= largest code * power
    y = torch.where(ok.unsqueeze(-1), blocks, 0.0) / powers[e].unsqueeze(-1)
    mag = y.abs().clamp(max=float(g[-1]))
    above = torch.searchsorted(g, mag.contiguous()).clamp(max=len(g) - 1)
    below = (above - 1).clamp(min=0)
    da, db = g[above] - mag, mag - g[below]
    code = torch.where((da < db) | ((da == db) & (above % 2 == 0)), above, below)
    code = torch.where(g[above] == mag, above, code)
    code = code + torch.signbit(y).long() * (8 if bits == 4 else 128)
    code = code.flatten(-2).to(torch.uint8)
    codes = code[..., 0::2] | (code[..., 1::2] << 4) if bits == 4 else code
    scales = torch.zeros(*top.shape[:-1], 4, dtype=torch.uint8)
    scales[..., : top.shape[-1]] = torch.where(ok, e - 100 + 127, 255).to(torch.uint8)
    return codes, scales


def dequantise(codes, scales, bits):
    codes, scales = codes.cpu(), scales.cpu()
    g = grid(bits)
    if bits == 4:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
        y = g[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    else:
        c = codes.long()
        full = torch.cat([g, torch.tensor([math.nan], dtype=torch.float64)])
        y = full[c & 127] * torch.where(c >= 128, -1.0, 1.0)
    y = y.unflatten(-1, (-1, BLOCK))
    s = scales[..., : y.shape[-2]].long()
    p = torch.where(s == 255, math.nan, 2.0 ** (s.double() - 127))
    return (y * p.unsqueeze(-1)).flatten(-2)


def attend(q, k, v, pos, count, causal, window, max_len, scale):
    """One row: q (T, Hq, D), k / v (H, S, D) doubles -> out (T, Hq, D) and A = sum p |v|, B = a bound on the relative error of any p."""
    q = q.double().cpu()
    t_n, hq, d = q.shape
    h, s_n, _ = k.shape
    g = hq // h
    out, a_, b_ = torch.zeros(t_n, hq, d, dtype=torch.float64), torch.zeros(t_n, hq, d, dtype=torch.float64), torch.zeros(t_n, hq, 1, dtype=torch.float64)
    for t in range(min(t_n, count)):
        x = pos + t if causal else pos + count - 1
        hi = min(x, s_n - 1, max_len - 1)
        lo = max(x - window + 1, 0) if window else 0
        if lo > hi:
            continue
        for j in range(hq):
            kk, vv = k[j // g, lo:hi + 1], v[j // g, lo:hi + 1]
            s = (kk * q[t, j]).sum(-1) * scale
            z = s - s.max()
            p = torch.softmax(s, -1)
            out[t, j] = p @ vv
            a_[t, j] = p @ vv.abs()
            mass = (kk.abs() * q[t, j].abs()).sum(-1).max() * scale
            # fp32: the scores' sums of D products, the scaled argument of the exponential, the exponential, the sums over the keys
            b_[t, j] = 2.0 ** -24 * ((d + 8) * mass + 4 * z.abs().max() + 8 + 2 * len(s))
    return out, a_, b_


def tolerance(out, a_, b_, dtype):
    """|kernel - out| at most this: both sums (numerator and denominator) carry the relative error of p; the numerator's terms are
    also rounded to matrix operands, by at most half a step of the last one: bf16 activations one fp16 number (2^-11) or two bf16
    ones (2^-8 2^-8), fp16 activations two fp16 (2^-11 2^-11) or two bf16 ones, fp32 three bf16 ones (2^-24).  Then one rounding to
    the type.  (A bf16 output's own half step is 2^-8.)"""
    cut = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -16}[dtype]
    return a_ * (2 * b_ + cut) * 1.01 + out.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
