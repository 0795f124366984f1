"""The e4m3 operators in 64 bits, and how far a correct kernel may be from them.

Sums: products of two e4m3 values are exact in fp32 and a kernel adds them in
fp32, in any order.  An addition in fp32 is off by at most 2^-23 of its result
(truncation; half that when rounded), and a result is at most the sum of the
magnitudes A of what is added, so n additions are off by at most n * 2^-23 * A.

The MoE layer quantises its inner activations, so a sum that is off by that
much can tip a value to the other neighbour when it lies next to the midpoint
of two e4m3 values.  The worst case over all values would hide real mistakes;
instead the error of one sum is taken as 8 standard deviations of independent
roundings (8 * sqrt(n) * 2^-23 * root of the sum of squares of the terms), each
value within that of a midpoint is allowed one e4m3 step, and all others none.
"""
from __future__ import annotations

import math

import torch

G = 128
F8 = torch.float8_e4m3fn
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def groups(n: int) -> int:
    return -(-n // G)


def step_of(v: torch.Tensor) -> torch.Tensor:
    """Distance of neighbouring e4m3 values around fp64 v."""
    _, e = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=-6) - 3)


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    s = step_of(v)
    return torch.clamp(torch.round(v / s) * s, -448.0, 448.0)


def scale_of(amax: torch.Tensor, pow2: bool) -> torch.Tensor:
    """fp64 amax -> the group scale, an fp32 number held in fp64."""
    s = (amax / torch.full_like(amax, 448.0)).float().double()
    s = torch.where(s < 2.0 ** -126, torch.full_like(s, 2.0 ** -126), s)
    if pow2:
        m, e = torch.frexp(s)
        s = torch.where(torch.isfinite(s), torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e)), s)
    return s


def pad(x: torch.Tensor, r: int, k: int) -> torch.Tensor:
    out = torch.zeros((r, k), dtype=torch.float64, device=x.device)
    out[: x.shape[0], : x.shape[1]] = x.double()
    return out


def quantize(x: torch.Tensor, block_rows: int = 1, pow2: bool = False):
    """(q as fp64 values, scale fp64)."""
    R, K = x.shape
    p = pad(x, groups(R) * G if block_rows == G else R, groups(K) * G)
    b = p.view(-1, block_rows, groups(K), G)
    s = scale_of(b.abs().amax(dim=(1, 3)), pow2)
    r = b / s[:, None, :, None]
    q = torch.where(torch.isnan(r), r, round_e4m3(r))
    return q.reshape(p.shape)[:R, :K], s


def rows_dequant(x, pow2=False):
    q, s = quantize(x, 1, pow2)
    return q * s.repeat_interleave(G, dim=1)[:, : x.shape[1]]


def weight(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    n, k = q.shape[-2:]
    return q.double() * s.double().repeat_interleave(G, dim=-2).repeat_interleave(G, dim=-1)[..., :n, :k]


def linear(x_values: torch.Tensor, w_values: torch.Tensor, bias=None, out_dtype=torch.float32):
    """(y, allowed error) of y = x . W^T + bias from what the e4m3 operands stand for."""
    y = x_values @ w_values.t()
    mag = x_values.abs() @ w_values.abs().t()
    n = G + groups(x_values.shape[1]) + 16
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    return y, n * 2.0 ** -23 * mag + HALF_STEP[out_dtype] * y.abs() + 2.0 ** -24


def moe(x, gate_up, gate_up_scale, down, down_scale, ids, weights, limit, pow2=False, out_dtype=torch.float32):
    """(out, allowed error); ids are local expert ids, out of range = skipped."""
    T, H = x.shape
    E, _, _ = gate_up.shape
    I = down.shape[2]
    xv = rows_dequant(x, pow2)
    out = torch.zeros((T, H), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    extra = torch.zeros_like(out)
    sigma8 = 8.0 * 2.0 ** -23
    for t in range(T):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < E:
                continue
            w13, w2 = weight(gate_up[e], gate_up_scale[e]), weight(down[e], down_scale[e])
            rw = weights[t, j].double()
            h = w13 @ xv[t]
            dh = sigma8 * math.sqrt(G + groups(H) + 8) * torch.sqrt((w13 * w13) @ (xv[t] * xv[t]))
            g, u = h[:I].clamp(max=limit), h[I:].clamp(-limit, limit)
            sg = g * torch.sigmoid(g)
            a = sg * u
            # |d silu / dg| <= 1.1; exp, division and products: a few roundings
            da = 1.1 * u.abs() * dh[:I] + sg.abs() * dh[I:] + 2.0 ** -21 * a.abs()
            b, db = a.view(-1, G), da.view(-1, G)
            amax = b.abs().amax(dim=1, keepdim=True)
            dmax = db.amax(dim=1, keepdim=True)
            s = scale_of(amax, pow2)
            rel_s = dmax / amax.clamp(min=1e-300)
            if pow2:
                jump = scale_of(amax + dmax, True) != scale_of(amax - dmax, True)
                rel_s = torch.zeros_like(rel_s)
            r = b / s
            q = round_e4m3(r)
            st = step_of(r)
            dr = db / s + r.abs() * rel_s
            to_mid = st / 2 - (r - q).abs()               # distance to the nearest midpoint
            allow = torch.where(to_mid.abs() <= dr, st * s, torch.zeros_like(r)) + (q * s).abs() * rel_s
            if pow2:
                allow = torch.where(jump, 2 * st * s, allow)
            av = (q * s).reshape(-1)
            out[t] += rw * (w2 @ av)
            mag[t] += rw.abs() * (w2.abs() @ av.abs())
            extra[t] += rw.abs() * (w2.abs() @ allow.reshape(-1))
    n = G + groups(I) + ids.shape[1] + 16
    return out, n * 2.0 ** -23 * mag + extra + HALF_STEP[out_dtype] * out.abs() + 2.0 ** -24


def worst(got: torch.Tensor, want: torch.Tensor, allowed: torch.Tensor) -> float:
    """Largest error over what is allowed; <= 1 passes."""
    assert torch.isfinite(got.double()).all()
    return float(((got.double() - want).abs() / allowed).max())


def e4m3_weight(shape, seed, device, scale=0.02):
    """e4m3 weights as a checkpoint holds them, with block scales."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(shape, generator=g) * 109.0).clamp(-448, 448).to(F8)
    s = (0.5 + torch.rand((*shape[:-2], groups(shape[-2]), groups(shape[-1])), generator=g)) * (scale / 109.0)
    return q.to(device), s.to(device)


def activations(rows, cols, seed, dtype, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g)
    x = x * torch.where(torch.rand((cols,), generator=g) < 0.1, 20.0, 1.0)
    return x.to(dtype).to(device)
