"""Attention in 64 bits, from the formulas, with the error bounds the tests use.

u is half a step of the element type (bf16 2^-8, f16 2^-11).  A kernel that
multiplies 16-bit operands exactly, sums in f32 and rounds probabilities (and,
in the gradient, the derivative of the scores) to the element type once may be
off by, per output element:
  scores   ds = (dim + 4) 2^-24 scale |q||k|   (f32 sum of dim products)
  weights  p (2 ds + u + 2^-18)                (both halves of the quotient, one
                                                rounding, exp and the f32 sums)
           + 2^-25 for f16                     (subnormal weights)
  output   u |out| on top
and correspondingly for the gradients, where D_i = dout_i.out_i takes the rounded
out.  `weight_bits` below is that sum."""
import math

import torch

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def tiny(t):
    """What a weight may lose below the type's normal range, times what it is multiplied with:
    half a step of a subnormal f16; for bf16, which has the exponents of f32, a weight below
    2^-126 may become zero, and the factors in these tests (dout.v among them) stay below 2^6."""
    return 2.0 ** -25 if t == "f16" else 2.0 ** -120


def visible(n, keys, causal, device):
    if not causal:
        return torch.ones(n, keys, dtype=torch.bool, device=device)
    i = torch.arange(n, device=device)[:, None]
    return torch.arange(keys, device=device)[None, :] <= i + (keys - n)


def head(q, k, v, scale, see):
    """One query head in 64 bits: out, lse, weights, scores' error bound."""
    s = (q @ k.T) * scale
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    top = s.amax(1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), -math.inf, dtype=s.dtype, device=s.device)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf))[:, 0]
    return p @ v, lse, p


def score_error(q, k, scale):
    if q.shape[0] == 0 or k.shape[0] == 0:
        return 0.0
    return (q.shape[1] + 4) * 2.0 ** -24 * scale * float(q.norm(dim=1).max() * k.norm(dim=1).max())


def weight_bits(t, err):
    return 2 * err + U[t] + 2.0 ** -18


def forward(t, q, k, v, segs_q, segs_k, scale, causal):
    """q [rows][heads][dim], k, v [rows][kv_heads][dim] of any float type.  Returns out, lse and
    their error bounds; rows in no segment hold NaN in all four."""
    g = q.shape[1] // k.shape[1]
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64, device=q.device)
    tol_o, tol_l = out.clone(), lse.clone()
    for (qf, qn), (kf, kn) in zip(segs_q, segs_k):
        if qn == 0:
            continue
        see = visible(qn, kn, causal, q.device)
        for h in range(q.shape[1]):
            qh = q[qf:qf + qn, h].double()
            kh, vh = k[kf:kf + kn, h // g].double(), v[kf:kf + kn, h // g].double()
            o, l, p = head(qh, kh, vh, scale, see)
            err = score_error(qh, kh, scale)
            out[qf:qf + qn, h], lse[qf:qf + qn, h] = o, l
            tol_o[qf:qf + qn, h] = U[t] * o.abs() + weight_bits(t, err) * (p @ vh.abs()) \
                + tiny(t) * (1 + see.double() @ vh.abs())
            tol_l[qf:qf + qn, h] = 2 * err + kn * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * \
                torch.where(l == -math.inf, torch.zeros_like(l), l).abs()
    return out, lse, tol_o, tol_l


def gradient(t, q, k, v, dout, segs_q, segs_k, scale, causal):
    """dq, dk, dv and their error bounds; rows in no segment hold NaN."""
    g = q.shape[1] // k.shape[1]
    u = U[t]
    grads = [torch.full(x.shape, math.nan, dtype=torch.float64, device=q.device) for x in (q, k, v)]
    tols = [x.clone() for x in grads]
    for (qf, qn), (kf, kn) in zip(segs_q, segs_k):
        for x in (*grads[1:], *tols[1:]):
            x[kf:kf + kn] = 0
        for x in (grads[0], tols[0]):
            x[qf:qf + qn] = 0
        if qn == 0 or kn == 0:
            continue
        see = visible(qn, kn, causal, q.device)
        for h in range(q.shape[1]):
            qh, do = q[qf:qf + qn, h].double(), dout[qf:qf + qn, h].double()
            kh, vh = k[kf:kf + kn, h // g].double(), v[kf:kf + kn, h // g].double()
            o, _, p = head(qh, kh, vh, scale, see)
            d = (do * o).sum(1, keepdim=True)
            dp = do @ vh.T
            ds = p * (dp - d)
            grads[0][qf:qf + qn, h] = scale * ds @ kh
            grads[1][kf:kf + kn, h // g] += scale * ds.T @ qh
            grads[2][kf:kf + kn, h // g] += p.T @ do
            bits = weight_bits(t, score_error(qh, kh, scale)) + kn * 2.0 ** -24
            err_out = u * o.abs() + weight_bits(t, score_error(qh, kh, scale)) * (p @ vh.abs()) + \
                tiny(t) * (1 + see.double() @ vh.abs())
            err_d = (do.abs() * err_out).sum(1, keepdim=True)
            err_dp = (q.shape[2] + 4) * 2.0 ** -24 * do.norm(dim=1, keepdim=True) * vh.norm(dim=1)[None, :]
            err_ds = ds.abs() * bits + p * (err_d + 2 * err_dp) + tiny(t) * see.double()
            err_p = p * bits + tiny(t) * see.double()
            tols[0][qf:qf + qn, h] = scale * err_ds @ kh.abs()
            tols[1][kf:kf + kn, h // g] += scale * err_ds.T @ qh.abs()
            tols[2][kf:kf + kn, h // g] += err_p.T @ do.abs()
    # f32 sums over all rows (2^-20 of the sum of magnitudes is far above their error) are inside
    # `bits`; the last rounding is half a step.
    for x, tol in zip(grads, tols):
        tol += u * x.abs() + tiny(t)
    return grads, tols


def within(got, want, tol):
    """NaN in `want`: not compared here."""
    ok = ((got.double() - want).abs() <= tol) | (got.double() == want) | want.isnan()
    if bool(ok.all()):
        return
    bad = (~ok).nonzero()
    first = tuple(bad[0].tolist())
    raise AssertionError(f"{len(bad)} of {ok.numel()} outside, first {first}: "
                         f"{got[first].item()} for {want[first].item()} +- {tol[first].item()}")


def rotate(x, pos, freqs, rot, interleaved):
    """x [rows][heads][dim] rotated in 64 bits."""
    y = x.double().clone()
    half = rot // 2
    a = torch.arange(0, rot, 2) if interleaved else torch.arange(half)
    b = a + 1 if interleaved else a + half
    angle = (pos.double()[:, None] * freqs.double()[None, :])[:, None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    xa, xb = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y
