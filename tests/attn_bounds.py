"""Attention in 64 bits with a bound of the kernels' error that stays small whatever
the scores' cap, a bias of masks or the number of keys are.

u is half a step of the element type (2^-11 fp16, 2^-8 bf16), p the exact weights,
o the exact output.  Of a row:
  * key j's exponent is off by slip_j at most, so its weight before the division by
    up to t_j = exp(x_j + slip_j - lse) - p_j.  A key whose weight is nothing (a bias
    of -inf, or of the type's lowest value among ordinary ones) adds nothing, however
    large its score is;
  * slip_j sums the fp32 errors of a score: head_dim products and sums (2^-24
    (head_dim + 4) scale sum |q||k|); the cap, within 16 * 2^-24 of its value in the
    form that holds for every cap, or, of caps up to 64, 9 * 2^-24 cap in the
    shorter form; the exponent, a fused multiply-add of the score and the running
    maximum, whose factor is rounded twice (2^-24 (6 |x_j| + 4 max |x| + 64), with the
    exponential's own last places and those of a rescaled sum's factors);
  * a weight is rounded to the type before it meets v, and may be summed as rounded: u
    of it, in both sums or in the products only.  fp16 weights are formed so that the
    row's largest is 2^8 at least, so below the normal range one is off by 2^-25 / 2^8
    of the largest;
  * sums over N keys grow by 16 at a time in fp32: N / 16 + 64 roundings of 2^-23.
Sums w_j (v_j) / sum w_j with w_j = p_j (1 + d_j) differ from o by
sum p_j d_j (v_j - o) / (1 + sum p_j d_j).  The output's own rounding is not part of
the bound (attn_ref.check_out adds it).
"""
import math

FAST_CAP = 64.0     # largest cap of the shorter form


def head(q, k, v, scale, cap=0.0, bias=None, seen=None):
    """One head: q [S, D], k and v [N, D], bias and seen [S, N] -> (p, output, bound of
    the output's error before its rounding)."""
    import torch
    dt = str(q.dtype)
    u = 2.0 ** -8 if "bfloat16" in dt else 2.0 ** -11
    q, k, v = q.double(), k.double(), v.double()
    S, N = q.shape[0], k.shape[0]
    seen = torch.ones(S, N, dtype=torch.bool, device=q.device) if seen is None else seen
    anyone = seen.any(0)[:, None]           # what nobody may look at must not count
    k, v = torch.where(anyone, k, 0.0), torch.where(anyone, v, 0.0)
    x = scale * (q @ k.T.contiguous())
    e = 2.0 ** -24
    slip = e * (q.shape[1] + 4) * scale * (q.abs() @ k.abs().T.contiguous())
    if cap:
        x = cap * torch.tanh(x / cap)
        slip = slip + e * (16 * x.abs() + (9 * cap if cap <= FAST_CAP else 0.0))
    if bias is not None:
        x = x + bias.double()
    x = torch.where(seen, x, -math.inf)
    top = x.amax(1, keepdim=True)
    some = top > -math.inf
    top = torch.where(some, top, 0.0)
    live = x > -math.inf
    x = torch.where(live, x, 0.0)
    z = torch.where(live, torch.exp(x - top), 0.0)
    total = z.sum(1, keepdim=True)
    total = torch.where(some, total, 1.0)
    p = z / total
    slip = slip + e * (6 * x.abs() + 4 * top.abs() + 64)
    t = torch.where(live, torch.exp(x - top + slip) / total - p, 0.0)
    assert t.sum(1).max().item() < 0.125, "scores too large for fp32: the bound says nothing"
    out = p @ v
    mass = p @ v.abs() + out.abs()
    bound = t @ v.abs() + t.sum(1, keepdim=True) * out.abs() + (u + (N / 16 + 64) * 2 * e) * mass
    if "bfloat16" not in dt:
        ones = live.double()
        bound = bound + 2.0 ** -33 * p.amax(1, keepdim=True) * (ones @ v.abs() + ones.sum(1, keepdim=True) * out.abs())
    return p, out, bound / (1 - t.sum(1, keepdim=True) - 2 * u)
