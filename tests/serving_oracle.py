"""Plain 64-bit forms of the operators over sequences of different lengths, with the bounds that a kernel of
32-bit sums and 16-bit outputs has to keep."""
import math

import torch


def frequencies(d, theta, scaling):
    """Angle per position of each pair from the formulas, and the amplitude."""
    s, L, lo, hi = scaling.factor, scaling.original, scaling.low, scaling.high
    f = [theta ** (-2.0 * i / d) for i in range(d // 2)]
    if scaling.kind == 1:
        f = [x / s for x in f]
    elif scaling.kind == 2:
        f = [(theta * s ** (d / (d - 2.0))) ** (-2.0 * i / d) for i in range(d // 2)]
    elif scaling.kind == 3:
        w = [min(1.0, max(0.0, (L * x / (2 * math.pi) - lo) / (hi - lo))) for x in f]
        f = [w_ * x + (1 - w_) * x / s for w_, x in zip(w, f)]
    elif scaling.kind == 4:
        pair = lambda n: d * math.log(L / (n * 2 * math.pi)) / (2 * math.log(theta))
        a, b = max(math.floor(pair(hi)), 0), min(math.ceil(pair(lo)), d - 1)
        w = [min(1.0, max(0.0, (i - a) / max(b - a, 0.001))) for i in range(d // 2)]
        f = [w_ * x / s + (1 - w_) * x for w_, x in zip(w, f)]
    return f, (0.1 * math.log(s) + 1.0 if scaling.kind == 4 else 1.0)


def rotate(x, positions, d, theta, half, scaling):
    """(rotated x [T, H, hd] in 64 bits, bound).  Bound: the turn's argument is a 32-bit float (2^-24 of at most
    pi) and sincospi and the amplitude's product are good to 2^-22; two products and a sum round by 2^-24 each; the
    result is rounded to fp16 (2^-11 of it, 2^-25 among the subnormals)."""
    f, amp = frequencies(d, theta, scaling)
    ang = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    c, s = (amp * ang.cos())[:, None], (amp * ang.sin())[:, None]
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    ia, ib = (slice(0, d // 2), slice(d // 2, d)) if half else (slice(0, d, 2), slice(1, d, 2))
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = amp * (a.abs() + b.abs())
    tol = size * (math.pi * 2.0 ** -24 + 2.0 ** -22 + 3 * 2.0 ** -24) + y.abs() * 2.0 ** -11 * 1.01 + 2.0 ** -25
    tol[..., d:] = 0
    return y, tol


def attend(q, k, v, scale, first):
    """(output [m, H, hd], bound) in 64 bits; row i of q sees the first `first + i` keys (all where None), none: 0.

    Bound, per element: a probability is rounded to fp16 (2^-11 of it, 2^-25 where it is subnormal, against a sum of at
    least sum exp(s - max)) and its score, a sum of hd products in fp32, is off by hd * 2^-23 of the sum of their sizes,
    and by 2^-22 of its distance from the maximum in the exponential; exp itself by 2^-18 (a polynomial of degree 4); the output's rounding is 2^-11
    of it.  fp32 sums over the keys add sqrt-like 2^-24s, covered by the factor 1.05."""
    m, H, hd = q.shape
    n, Hk = k.shape[:2]
    g = H // Hk
    q, k, v = q.double(), k.double(), v.double()
    out, tol = torch.zeros((m, H, hd), dtype=torch.float64, device=q.device), torch.zeros((m, H, hd), dtype=torch.float64, device=q.device)
    if n == 0:
        return out, tol
    seen = torch.ones((m, n), dtype=torch.bool, device=q.device)
    if first is not None:
        seen = torch.arange(n, device=q.device)[None] < first + torch.arange(m, device=q.device)[:, None]
    some = seen.any(1)
    for h in range(H):
        kh, vh = k[:, h // g], v[:, h // g]
        s = (q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf)
        size = (q[:, h].abs() @ kh.abs().T * abs(scale)).masked_fill(~seen, 0)
        top = s.amax(1, keepdim=True)
        top = torch.where(some[:, None], top, torch.zeros_like(top))
        e = torch.exp(s - top)
        l = e.sum(1, keepdim=True)
        l = torch.where(some[:, None], l, torch.ones_like(l))
        vh_ = torch.where(seen.any(0)[:, None], vh, torch.zeros_like(vh))  # what nobody sees does not count
        o = (e / l) @ vh_
        off = 2.0 ** -11 + 2 * (hd * 2.0 ** -23) * size + 2.0 ** -22 * (s - top).masked_fill(~seen, 0).abs() * 2 + 2.0 ** -18
        t = (e / l * off) @ vh_.abs() + 2.0 ** -25 * (seen.double() @ vh_.abs()) / l
        out[:, h] = torch.where(some[:, None], o, torch.zeros_like(o))
        tol[:, h] = torch.where(some[:, None], 1.05 * t + o.abs() * 2.0 ** -11 + 2.0 ** -25, torch.zeros_like(t))
    return out, tol


def positions_of(pages, table_row, n):
    """The first n positions of a sequence, [n, kv_heads, hd]; pages outside the pool read as zeros."""
    size = pages.shape[1]
    idx = table_row[:-(-n // size)].long()
    ok = (idx >= 0) & (idx < pages.shape[0])
    got = pages[torch.where(ok, idx, torch.zeros_like(idx))] * ok[:, None, None, None]
    return got.flatten(0, 1)[:n]


def assert_close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), (err / tol.clamp_min(1e-30)).nan_to_num(9e9).max().item(),
                           bad.nonzero()[0].tolist())
