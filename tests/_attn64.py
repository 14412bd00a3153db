"""Attention in 64 bits, and how far a kernel that follows its contract may be from it."""
import math

import torch

FP32 = 2.0 ** -24  # half a step


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend64(q, k, v, visible, scale, dtype):
    """q [n, D], k and v [T, D], visible bool [n, T] -> (o, tol) [n, D] in 64 bits.

    The bound counts roundings of o = sum p v / sum p against A = sum p |v| / sum p:
    a weight is rounded to the dtype (half a step of A; below the dtype's normal range
    at most half its smallest step, absolute, of weights that are 1 at their maximum),
    the result too (half a step of |o|).  Everything else is fp32: a score is D products
    added (D half steps of scale * sum |q k|, which move a weight by as much, relatively,
    and the maximum's weight and the scaling by log2(e) again), the exponential and its
    argument (8 half steps, and the argument's own rounding of up to |argument| half
    steps, below), and the sums of T weights, rescaled once per 64 keys (T + T / 16
    half steps each)."""
    q, k, v = q.double(), k.double(), v.double()
    n, T, D = q.shape[0], k.shape[0], k.shape[1]
    if T == 0:
        return torch.zeros_like(q), torch.full_like(q, 1e-30)
    seen_v = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
    s = (q @ k.T) * scale
    s = torch.where(visible, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.where(visible, (s - torch.where(m.isinf(), torch.zeros_like(m), m)).exp(),
                    torch.zeros_like(s))
    l = p.sum(-1, keepdim=True)
    w = p / torch.where(l == 0, torch.ones_like(l), l)
    o = torch.empty(n, D, dtype=torch.float64, device=q.device)
    bad = ~v.isfinite().all(-1)
    if bool(bad.any()):  # 0 * inf must not enter where a row is not seen
        for i in range(n):
            o[i] = w[i, visible[i]] @ v[visible[i]]
    else:
        o = w @ v
    A = w @ seen_v.abs()
    big = torch.where(visible, (q.abs() @ k.abs().T) * scale, torch.zeros_like(s)).amax(-1, keepdim=True)
    u = half_step(dtype)
    e32 = FP32 * (2 * (D + 4) * big + 8 + 4 * big + 2 * (T + T / 16))
    tiny = 0.0 if dtype == torch.bfloat16 else 2.0 ** -25
    tol = u * o.abs() + (u + e32) * A + tiny * seen_v.abs().sum(0)
    return o, tol + 2.0 ** -24 * (dtype == torch.float16) + 1e-30


def check(got, o, tol):
    got = got.double()
    fine = o.isfinite()
    assert torch.equal(fine, got.isfinite()) and torch.equal(o.isnan(), got.isnan())
    inf = ~fine & ~o.isnan()
    assert torch.equal(got[inf], o[inf])
    d = (got - o).abs()[fine]
    over = (d / tol[fine]).max().item() if d.numel() else 0.0
    assert over <= 1.0, f"{over:.3f} of the bound"
    return over
