"""Causal attention of one head in float64, and how far a correct kernel with
FP16 inputs, outputs and probabilities may be from it, value by value.

u = 2^-11 is half a step of FP16 relative to the value, z = 2^-25 half a step
among its subnormals, w = 2^-24 half a step of FP32. A kernel rounds
  - each score: a sum of HD products in FP32 and its scaling, at most (HD + 4) w
    of the terms' magnitudes scale |q| |k|; the exponential adds 2^-21 (the
    hardware's 2^x, its argument's rounding). Both are relative errors of the
    probabilities, e = max over the scores;
  - probabilities and dS to FP16: u of the value, z below 2^-14 (a probability
    is rounded before the division by the sum l >= 1, so z is not enlarged);
  - the outputs to FP16: u of the value, z;
  - the sums of products in FP32: n w of the terms' magnitudes, below u / 4 of
    them up to 2,048 terms; they are counted by taking 1.25 u for u.
First-order terms add up; 1.05 covers their products."""

import torch

U, Z, W = 2.0 ** -11, 2.0 ** -25, 2.0 ** -24


def attend(q, k, v, scale, visible, dout=None):
    """q: n x HD, k, v: m x HD, visible: n x m, any float type. A dict of name ->
    (value, bound) for o, lse and with dout dq, dk, dv, all float64."""
    q, k, v = q.double(), k.double(), v.double()
    s = (scale * q @ k.T).masked_fill(~visible, float("-inf"))
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    o = p @ v
    u = 1.25 * U
    terms = abs(scale) * (q.abs() @ k.abs().T)
    err = torch.where(visible, (q.shape[1] + 4) * W * terms, 0.0)
    e = 2.0 ** -21 + err.max(1, keepdim=True).values      # of a row's probabilities
    mass = p @ v.abs()
    reach = visible.double()
    o_bound = (u + 2 * e) * mass + U * o.abs() + Z * (reach @ v.abs()) + Z
    out = dict(o=(o, 1.05 * o_bound), lse=(lse, 1.05 * (e[:, 0] + 4 * W * lse.abs() + 4 * W)))
    if dout is None:
        return out
    g = dout.double()
    pe = u + 2 * e + 4 * W * lse.abs()[:, None]          # of a probability in the backward
    dv = p.T @ g
    dv_bound = (pe * p).T @ g.abs() + Z * (reach.T @ g.abs()) + U * dv.abs() + Z
    dp = g @ v.T
    d = (g * o).sum(1, keepdim=True)
    ds = p * (dp - d)
    d_err = (g.abs() * o_bound).sum(1, keepdim=True) + q.shape[1] * W * (g.abs() * o.abs()).sum(
        1, keepdim=True)
    dp_err = q.shape[1] * W * (g.abs() @ v.abs().T)
    ds_err = pe * ds.abs() + p * (d_err + dp_err) + u * ds.abs() + Z * reach
    dq, dk = scale * ds @ k, scale * ds.T @ q
    dq_bound = abs(scale) * (ds_err @ k.abs()) + U * dq.abs() + Z
    dk_bound = abs(scale) * (ds_err.T @ q.abs()) + U * dk.abs() + Z
    out.update(dq=(dq, 1.05 * dq_bound), dk=(dk, 1.05 * dk_bound), dv=(dv, 1.05 * dv_bound))
    return out


def causal(n, cached=0):
    """New token t, at position cached + t, sees the positions up to its own."""
    return (torch.arange(cached + n)[None, :] <= torch.arange(cached, cached + n)[:, None])


def worst(got, value, bound):
    """The largest |got - value| / bound, and infinity where got is not finite."""
    ratio = (got.double() - value).abs() / bound
    return float(torch.where(torch.isfinite(got.double()), ratio, float("inf")).max())
