"""Inputs that leave of an adapter projection only what its rank-space vector
u = scale x A^T loses on the way to the second product, and the bounds.

x and A are small whole numbers, scale and B powers of two, so every product and
every partial sum is a multiple of 1/4 below 2^24 quarters: exact in f32 in any
order.  Output n takes rank value j = n mod R with a sign, and W's row n is the
negative of what that adds up to, so y is 0 wherever the row's adapter has rank
value j, and what was lost of u shows undiminished.  u itself has up to 17
bits: one f16 (11 bits) or one bf16 (8) cannot hold it; a pair of either does.
"""
import torch


def exact_inputs(dtype, rows, slots, ranks, inn, out, seed, device):
    """(x [m, inn], W [out, inn], A per slot, B per slot, scale per slot, slot of each row)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).to(torch.float64)
    assert inn * 64 * 8 < 1 << 22          # a sum of products, in quarters, below 2^24
    R = max(ranks)
    x, a = ints(-64, 64, sum(rows), inn), ints(-8, 8, R, inn)
    sign = ints(0, 1, out) * 2 - 1
    j = torch.arange(out) % R
    scale = [2.0 ** (s % 3 - 2) for s in range(len(ranks))]
    bs = []
    for s, r in enumerate(ranks):
        b = torch.zeros(out, R, dtype=torch.float64)
        b[torch.arange(out), j] = sign / 4 / scale[s]
        bs.append(b[:, :r])
    w = -sign[:, None] / 4 * a[j]
    owner = torch.repeat_interleave(torch.tensor(slots), torch.tensor(rows))
    put = lambda t: t.to(dtype).to(device)
    return put(x), put(w), [put(a[:r]) for r in ranks], [put(b) for b in bs], scale, owner.to(device)


def definition(x, w, a, b, scale, owner, held=lambda u: u):
    """(y in 64 bits, |u| |B|^T), u passed through `held` between the products."""
    xd = x.double()
    y = xd @ w.double().T
    part = torch.zeros_like(y)
    for s in range(len(a)):
        rows = (owner == s).nonzero()[:, 0]
        u = held(scale[s] * (xd[rows] @ a[s].double().T))
        y[rows] += u @ b[s].double().T
        part[rows] = u.abs() @ b[s].double().abs().T
    return y, part


def eps(dtype):
    """Half a step: what one rounding is off by, relative to the value."""
    return torch.finfo(dtype).eps / 2


def rank_limit(dtype, want, part, b_sum):
    """Largest error of y when u is a value and its remainder and all sums are
    exact: eps^2 of u (f16: its smallest step, 2^-24, halved), then y's rounding."""
    e = eps(dtype)
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    tol = e * e * part + floor * b_sum
    return tol + e * (want.abs() + tol) + floor


def rms(t):
    return float(t.double().square().mean().sqrt())


def one(dtype):
    return lambda u: u.to(dtype).double()


def pair(dtype):
    def held(u):
        hi = u.to(dtype).double()
        return hi + (u - hi).to(dtype).double()
    return held


def bits(n):
    """u to n significant bits."""
    def held(u):
        m, e = torch.frexp(u)
        return torch.ldexp(torch.round(m * 2.0 ** n) / 2.0 ** n, e)
    return held
