"""Attention with changed scores and masks from its definition, in float64, for one sequence (torch
tensors of any device)."""
import torch


def attention(q, k, v, have, length, causal=True, window=0, scale=None, softcap=0.0, slopes=None,
              first=None, prefix=0):
    """q [n, hq, d] (the last n positions of ``length`` tokens), k and v [held, heads, d], have [held]
    -> (out, lse, bound, lse_bound).

    bound is what a result may differ by before its own rounding, to first order. A weight rounded to
    float16 errs by 2^-11. A float32 score errs by 2^-23 times a few of its terms: the
    d products' magnitudes, itself, 90 (the exponent's own steps), the cap (tanh by way of an exponential errs by
    1.5 x 2^-23 of 1; caps above 128 by 2^-20 of the score) and the distance's share. A score's
    error e_j moves its weight by e_j of itself and the sum by the weighted mean of all."""
    n, hq, d = q.shape
    held, heads, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    lse, lse_bound = q.new_full((n, hq), -torch.inf), q.new_zeros((n, hq))
    if n == 0 or held == 0:
        return out, lse, bound, lse_bound
    j = torch.arange(held, device=q.device)
    p = length - n + torch.arange(n, device=q.device)[:, None]
    see = have[None, :].expand(n, held)
    if causal:
        see = see & ((j <= p) | (j < prefix))
    if window:
        see = see & (j > p - window)
    if first is not None:
        see = see & (j >= first[:, None])
    some = see.any(1)
    far = (p - j).abs().double()

    def weighed(w, y):
        """w @ y over the seen tokens: where a weight is not seen, what it would meet counts nothing."""
        clean = torch.where(torch.isnan(y), torch.zeros_like(y), y)
        bad = see.double() @ torch.isnan(y).double() > 0
        return torch.where(bad, torch.full_like(clean[:1], torch.nan), w @ clean)
    for h in range(hq):
        kk, vv = k[:, h * heads // hq], v[:, h * heads // hq]
        s = q[:, h] @ kk.t() * scale
        err = 4 * (q[:, h].abs() @ kk.abs().t()) * scale + 4 * s.abs() + 90
        if softcap:
            s = softcap * torch.tanh(s / softcap)
            err = err + (3 * softcap if softcap <= 128 else 8 * s.abs())
        if slopes is not None:
            s = s - slopes[h] * far
            err = err + 3 * abs(slopes[h]) * far + 3 * s.abs()
        s = torch.where(see, s, torch.full_like(s, -torch.inf))
        err = torch.where(see, err, torch.zeros_like(err)) * 2.0 ** -23
        m = torch.where(some, s.amax(1), torch.zeros_like(s[:, 0]))[:, None]
        w = torch.exp(s - m)
        total = torch.where(some, w.sum(1), torch.ones_like(m[:, 0]))
        w = w / total[:, None]
        mean = (w * err).sum(1)
        out[:, h] = weighed(w, vv)
        lse[:, h] = torch.where(some, m[:, 0] + total.log(), torch.full_like(total, -torch.inf))
        y = vv.abs().nan_to_num(0.0)
        bound[:, h] = 1.1 * ((2.0 ** -11 + mean)[:, None] * (w @ y) + (w * err) @ y)
        lse_bound[:, h] = 1.1 * mean + 2.0 ** -22 * (1 + lse[:, h].abs())
    return out, lse, bound, lse_bound
