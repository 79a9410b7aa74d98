"""Attention and its gradient from their formulas in float64, and how far float32 sums and 16-bit weights may be off them.

Sizes of errors, for the tests of attention_train and attention_grad. u = 2^-24 is float32's half step, H the operands' (float32:
0, nothing is rounded to fewer bits), T half of the smallest number that the operands' type has, where it is so large that it
counts: a weight below it may vanish (float16 2^-25, of the gradient's weights, which are 32 times as large, 2^-30).
  scores      D products are exact (16 bits) or off by u, and are added one after the other, each sum off by u, twice that
              where the matrix instruction cuts in place of rounding: 2 (D + 4) u scale sum|q k|. An exponent has the scores'
              error, a rounded factor (c = scale log2 e), one rounding of a fused step and one of the power, all of at most u
              times what is added: E = scores + 6 u (|s| + |lse|) + 4 u
  sums        n terms one after the other: 2 (n + 32) u times the sum of their sizes
  out         sum_j p|v| (E + H + E_max + H) + T |v|, the second E for the row's total, which is made from the unrounded
              exponentials, + sums; a quotient by two roundings 3 u; then the result's H
  lse         E_max + 2 (n + 32) u + 4 u (|lse| + |m| + 1)
  gradient    p: E + H, T.  x = g v - delta: 2 (D + 4) u (sum|g v| + sum|g out|) + 2 u |x|.  ds = p x: p dx + |x| p E + 2 u|ds|,
              then H |ds| + T.  dq, dk, dv: these times |k|, |q|, |g|, + sums, 4 u, then the result's H"""

import numpy as np

U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}


def weight_half(d):
    return 0.0 if d == "float32" else HALF[d]


def seen(b, h, sq, sk, causal=False, lengths=None, mask=None):
    s = np.ones((b, h, sq, sk), bool)
    if causal:
        s &= np.arange(sk)[None, :] <= np.arange(sq)[:, None] + (sk - sq)
    if lengths is not None:
        s &= (np.arange(sk)[None, :] < np.asarray(lengths)[:, None])[:, None, None, :]
    if mask is not None:
        s &= mask
    return s


def shared(x, heads):
    return np.repeat(x, heads // x.shape[1], 1)


def without(x, keep):
    return np.where(keep, x, 0.0)


def forward(q, k, v, scale, keep, d="float32"):
    """(out, lse), and how far each may be off."""
    heads, n, dim = q.shape[1], k.shape[2], q.shape[3]
    k, v = shared(k, heads), shared(v, heads)
    used = keep.any((1, 2))[:, None, :, None]  # keys that nobody sees may hold anything
    k, v = without(k, used), without(v, used)
    s = np.where(keep, np.matmul(q, k.swapaxes(2, 3)) * scale, -np.inf)
    m = s.max(3, keepdims=True, initial=-np.inf)
    some = np.isfinite(m)
    e = np.exp(np.where(keep, s, -np.inf) - np.where(some, m, 0.0))
    total = e.sum(3, keepdims=True)
    p = e / np.where(some, total, 1.0)
    lse = np.where(some, np.where(some, m, 0.0) + np.log(np.where(some, total, 1.0)), -np.inf)
    out = np.matmul(p, v)
    size = np.matmul(np.abs(q), np.abs(k).swapaxes(2, 3)) * scale
    flat = np.where(some, lse, 0.0)
    err = without(2 * (dim + 4) * U * size + 6 * U * (np.abs(without(s, keep)) + np.abs(flat)) + 4 * U, keep)
    worst = err.max(3, keepdims=True, initial=0.0)
    h, t = weight_half(d), TINY[d] if d == "float16" else 0.0
    out_err = np.matmul(p * (err + worst + 2 * h + 2 * (n + 32) * U * 2 + 3 * U) + t * keep, np.abs(v))
    lse_err = worst + 2 * (n + 32) * U + 4 * U * (np.abs(flat) + np.abs(np.where(some, m, 0.0)) + 1)
    return (out, lse[..., 0]), (out_err, lse_err[..., 0])


def backward(g, q, k, v, out, lse, scale, keep, d="float32"):
    """(dq, dk, dv) for the given out and lse, and how far each may be off."""
    b, heads, sq, dim = q.shape
    group, kv, n = heads // k.shape[1], k.shape[1], k.shape[2]
    used = keep.any((1, 2))[:, None, :, None]
    k, v = without(shared(k, heads), used), without(shared(v, heads), used)
    s = np.matmul(q, k.swapaxes(2, 3)) * scale
    flat = np.where(np.isfinite(lse), lse, 0.0)[..., None]
    p = np.where(keep, np.exp(np.where(keep, s - flat, 0.0)), 0.0)
    delta = (g * out).sum(3, keepdims=True)
    x = np.matmul(g, v.swapaxes(2, 3)) - delta
    ds = p * x
    size = np.matmul(np.abs(q), np.abs(k).swapaxes(2, 3)) * scale
    e = without(2 * (dim + 4) * U * size + 6 * U * (np.abs(s) + np.abs(flat)) + 4 * U, keep)
    h, t = weight_half(d), 2.0 ** -30 if d == "float16" else 0.0
    x_err = 2 * (dim + 4) * U * (np.matmul(np.abs(g), np.abs(v).swapaxes(2, 3)) + (np.abs(g) * np.abs(out)).sum(3, keepdims=True)) + 2 * U * np.abs(x)
    ds_err = p * x_err * (1 + e) + np.abs(ds) * (e + 2 * U)
    ds_err = ds_err + h * (np.abs(ds) + ds_err) + t * keep
    p_err = p * e + h * p * (1 + e) + t * keep
    # (a lifted weight past the type's largest number is no case here)
    def joined(y):
        return y.reshape(b, kv, group, *y.shape[2:]).sum(2)

    dq = scale * np.matmul(ds, k)
    dk = joined(scale * np.matmul(ds.swapaxes(2, 3), q))
    dv = joined(np.matmul(p.swapaxes(2, 3), g))
    rows, cols = 2 * (n + 32) * U + 4 * U, 2 * (sq * group + 32) * U + 4 * U
    dq_err = scale * np.matmul(ds_err + rows * np.abs(ds), np.abs(k))
    dk_err = joined(scale * np.matmul((ds_err + cols * np.abs(ds)).swapaxes(2, 3), np.abs(q)))
    dv_err = joined(np.matmul((p_err + cols * p).swapaxes(2, 3), np.abs(g)))
    return (dq, dk, dv), (dq_err, dk_err, dv_err)
