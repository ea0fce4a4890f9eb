"""The int8 path in 64 bits: codes and scales of rows, add + RMS norm before them, products, the gated block.

Test infrastructure only (see ``oracle/__init__.py``).  The reference has no
int8 op; the definitions are those of the op docstrings:

  s = max(f32(amax |x| / 127), 2^-126), q = the integer nearest to x / s, ties to
  even; a row with a value that is not finite: s = NaN, q = 0.
  r' = Out(h + r), x = r' w / sqrt(mean((h + r)^2) + eps), not rounded.
  y = Out((f32(sum_k a b) sb) sa), the sum an integer below 2^31.
  gated: g, u such fp32 values of rows i and d + i, y = Out(act(g) u).

Pins (tests/test_int8.py): codes by integer arithmetic on fractions, products by
Python integers, the activations against torch's.
"""

import math

import torch

MIN_SCALE = 2.0 ** -126


def quant(x):
    """x [T, H], any float type -> (codes int8, scale fp32 [T])."""
    x = x.cpu().double()
    bad = ~torch.isfinite(x).all(1)
    s = (x.abs().amax(1) / 127).float().clamp_min(MIN_SCALE)
    q = torch.round(x / s.double()[:, None])
    q[bad] = 0
    s[bad] = math.nan
    return q.to(torch.int8), s


def add_rms_norm(h, r, w, eps):
    """-> (r' of h's type, the normed rows in 64 bits)."""
    t = h.cpu().double() + r.cpu().double()
    kept = t.float().to(h.dtype)
    return kept, kept.double() * w.cpu().double() / (t.square().mean(1, keepdim=True) + eps).sqrt()


def sums(a, b):
    """Exact integers (K 2^14 < 2^53), as float64."""
    return a.cpu().double() @ b.cpu().double().t()


def scaled(acc, sa, sb):
    """fp32, each operation rounded once."""
    return acc.float() * sb.cpu().float() * sa.cpu().float()[:, None]


def product(a, sa, b, sb, dtype):
    return scaled(sums(a, b), sa, sb).to(dtype)


def act(g, name):
    """(act(g), z) with act(g) = g sigmoid(z), in 64 bits."""
    z = g if name == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    return g * torch.sigmoid(z), z


def gated(a, sa, b, sb, name):
    """(y, bound) in 64 bits: the block's value and how far fp32 arithmetic may take a result from it before
    its one rounding to 16 bits (u = 2^-24; see the terms)."""
    y = sums(a, b) * sb.cpu().double() * sa.cpu().double()[:, None]
    d = y.shape[1] // 2
    g, u = y[:, :d], y[:, d:]
    f, z = act(g, name)
    # g and u: three roundings each (the sum's conversion, two scales).  g reaches the result itself and through
    # z, |g z'| <= 3 |z|, and z acts on sigmoid by |z| (1 - sigmoid): (3 + 9 w) u with w = |z| (1 - sigmoid(z)).  z's own
    # four operations and constants and the product with log2 e: 7 w.  exp2 2, 1 + e, the quotient and the product
    # with u (3 + 1) one each.
    w = z.abs() * torch.sigmoid(-z)
    rel = (16 + 16 * w) * 2.0 ** -24
    # sigmoid below 2^-126 (exp beyond fp32) is 0, and products below fp32's normal range lose bits
    return f * u, (f * u).abs() * rel + g.abs() * u.abs() * 2.0 ** -126 + 2.0 ** -149
