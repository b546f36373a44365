"""Plain attention in 64 bits, and how far a result in 16 bits may be from it.

Bounds, element by element, from the arithmetic of the operators (u = half a step
of the element type: 2^-11 fp16, 2^-8 bf16):
  * softmax weights are rounded to the type before they meet v, and may be summed
    as they were rounded.  With weights p (1 + d), |d| <= u, in both sums the
    result is off by sum p d (v - out) / (1 + sum p d), at most
    u (sum p |v| + |out|) (1 + 2 u);
  * an fp16 weight below the normal range is off by 2^-25 at most.  Weights are
    formed against a maximum that may be the row's by up to 2^3 larger, so the
    largest is at least 2^-3 before the division: 2^-22 of it;
  * scores are fp32 sums of head_dim products: off by 2^-24 (head_dim + 4) scale
    sum |q||k| at most, and a few roundings of the score itself (8 * 2^-24 |x|);
    a capped one, cap - 2 cap t with t = 1 / (1 + e^(2 y)), also by what t is off,
    twice cap times: 2^-23 for the reciprocal's last place, 2^-24 for the sum's
    rounding, 2^-24 at most for e's (2^-22 of it, t (1 - t) <= 1/4), and by its own
    rounding: 9 * 2^-24 cap; a weight follows its exponent's error
    e as e^e - 1, on both sides of the division;
  * the output is rounded once more: u of itself (2^-25 below fp16's normal range).
"""
import math

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def half_step(dtype):
    return HALF_STEP[str(dtype).split(".")[1]]


def head(q, k, v, scale, cap=0.0, bias=None, seen=None):
    """One head in 64 bits: q [S, D], k and v [N, D], bias and seen [S, N].  Returns
    (weights, output, bound of the weights' relative error, bound of the output's
    error before its own rounding)."""
    import torch
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    S, N = q.shape[0], k.shape[0]
    seen = torch.ones(S, N, dtype=torch.bool, device=q.device) if seen is None else seen
    # what nobody may look at must not count, whatever it holds
    k = torch.where(seen.any(0)[:, None], k, 0.0)
    v = torch.where(seen.any(0)[:, None], v, 0.0)
    x = scale * (q @ k.T.contiguous())
    mass = scale * (q.abs() @ k.abs().T.contiguous())
    slip = 2.0 ** -24 * (q.shape[1] + 4) * mass
    if cap:
        x = cap * torch.tanh(x / cap)
        slip = slip + 9 * 2.0 ** -24 * cap
    if bias is not None:
        x = x + bias.double()
    slip = slip + 8 * 2.0 ** -24 * torch.where(seen, x.abs(), 0.0)
    x = torch.where(seen, x, -math.inf)
    some = seen.any(1, keepdim=True) & (x.amax(1, keepdim=True) > -math.inf)
    p = torch.where(some, torch.softmax(torch.where(some, x, 0.0), 1), 0.0)
    slip = torch.where(seen, slip, 0.0).amax(1, keepdim=True).clamp(max=1.0)
    weight_bound = torch.expm1(2 * slip) + 4 * 2.0 ** -24
    u = half_step(dt)
    out = p @ v
    bound = (u + 2 * u * u + weight_bound) * (p @ v.abs()) + u * (1 + 2 * u) * out.abs()
    if str(dt) == "torch.float16":
        bound = bound + 2.0 ** -22 * N * (p.amax(1, keepdim=True) * v.abs().amax())
    return p, out, weight_bound, bound


def check_out(got, ref, bound, dtype, what=""):
    """got (16 bits) against ref, whose error before rounding is at most bound."""
    import torch
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    allowed = bound + half_step(dtype) * (ref.abs() + bound) + 2.0 ** -25
    worst = ((got - ref).abs() / allowed).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the allowed error"
