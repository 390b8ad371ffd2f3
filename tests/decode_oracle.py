"""Single-token attention in 64 bits from whole sequences, for the tests of the paged cache, with how far a computation that
keeps 32 bits may be off."""
import math

import torch


def taps(x, w, rows):
    """x (H, rows + R - 1, n), w (H, R, S) -> (H, rows, n): sum of w[h, r, t] x[h, j + r, k + t - (S-1)//2], 0 outside."""
    (_, r, s), n = w.shape, x.size(-1)
    left = (s - 1) // 2
    x = torch.nn.functional.pad(x, (left, s - 1 - left))
    return sum(w[:, a, b, None, None] * x[:, a:a + rows, b:b + n] for a in range(r) for b in range(s))


def token(q, k, v, w, scale, pre=None, w2=None, post=None, window=0):
    """The newest row over one sequence: q (H, n, D), k and v (Hkv, n, D), all float64 -> (o (H, D), bound (H, D)).

    bound: every sum of N products in 32 bits is off by at most N g times the sum of the magnitudes, g = 2**-24, and a score that is
    off by d makes its probability off by a factor of 1 + 2 d (its own and the row's sum).  Sums over the keys run along chains of n/8
    at most (eight row groups of a wavefront at least, or a lane for each of 64 keys), then over a few hundred splits and lanes."""
    h, n, d = q.shape
    share = h // k.size(0)
    k, v = k.repeat_interleave(share, 0), v.repeat_interleave(share, 0)
    r, s = w.shape[1:]
    rows = w2.size(1) if w2 is not None else 1
    first = n - (r + rows - 1)
    pos = torch.arange(first, n)
    key = torch.arange(n)
    seen = (key[None] <= pos[:, None]) & (pos[:, None] >= 0) & ((key[None] > pos[:, None] - window) if window else True)
    qr = torch.cat([torch.zeros(h, max(0, -first), d, dtype=q.dtype), q[:, max(0, first):]], 1)
    raw = torch.where(seen, torch.matmul(qr, k.transpose(1, 2)) * scale, 0.0)
    size = torch.where(seen, torch.matmul(qr.abs(), k.abs().transpose(1, 2)) * scale, 0.0)
    sc, big = taps(raw, w, rows), taps(size, w.abs(), rows)
    terms = d + r * s + 8
    if pre is not None:
        sc, big = torch.einsum("oi,ijk->ojk", pre, sc), torch.einsum("oi,ijk->ojk", pre.abs(), big)
        terms += h
    seen = seen[-rows:]
    p = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
    p = torch.where(seen, p, 0.0)      # (rows ahead of the first token see nothing)
    g = 2.0 ** -24
    off = 2 * terms * g * torch.where(seen, big, 0.0).nan_to_num(0.0, 0.0, 0.0).amax()
    pabs, terms = p, n / 4 + 512
    if w2 is not None:
        p, pabs = torch.where(seen[-1:], taps(p, w2, 1), 0.0), taps(p, w2.abs(), 1)
        terms += w2.size(1) * w2.size(2)
    if post is not None:
        p, pabs = torch.einsum("oi,ijk->ojk", post, p), torch.einsum("oi,ijk->ojk", post.abs(), pabs)
        terms += h
    o = torch.matmul(p[:, -1:], v)[:, 0]
    return o, (off + terms * g) * torch.matmul(pabs[:, -1:], v.abs())[:, 0]


def check(got, want, bound, what=""):
    """got: rounded once from 32 bits."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = ((got - want).abs() - (half * (1 + 2 ** -10) * want.abs() + bound + torch.finfo(torch.float16).smallest_normal * 2 ** -10)).nan_to_num(0.0)
    assert off.max() <= 0, f"{what}: {float((got - want).abs().nan_to_num(0.0).max())} off, {float(off.max())} beyond the bound"
