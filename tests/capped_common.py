"""Capped attention rows in 64 bits with a bound that small caps cannot hide
behind, and values on which a wrong score shows.

A cap of c keeps every score within +-c, whatever the scores' own rounding is.
With u = 2^-11 (half a step of fp16) an output element is off by at most

  * the capped score: c tanh(s / c) is monotone, so a score off by ds moves it to
    between its values at s - ds and s + ds.  ds = scale (sum |q k| (u + 2^-17)
    + 2^-17 sum |k| + 2^-19 sum |q|): K^ rounded to fp16 once, the fp32 sum of
    128 products (128 * 2^-24), and where a large cap brings Q or K^ below
    fp16's normal range (2^-25 over the factors 2^-8 and 0.0225 they carry).
    The fp32 form of the cap itself: 4.8e-7 c;
  * with e_i = exp(dy_i) - 1 for key i's shift dy_i, weights p_i (1 + d_i), |d_i| <=
    e_i, give sum p_i d_i (v_i - out) / (1 + sum p_i d_i): at most sum p_i e_i
    (|v_i| + |out|) / (1 - E), E = sum p_i e_i;
  * the weight's rounding to fp16, its product with V's scale (or V^), and the
    sum of the weights as rounded or not: 3 u; the fp32 exponent 2^-16;
  * V^ below fp16's normal range: 2^-25 a value (and the same for p d_v, which
    `capped_rows` asserts to stay in that range).
"""
import numpy as np

U = 2.0 ** -11


def _softmax(y, seen):
    y = np.where(seen, y, -np.inf)
    p = np.exp(y - y.max(1, keepdims=True))
    return p / p.sum(1, keepdims=True)


def capped_rows(q, K, V, scale, cap, seen, wrong=None):
    """(out, bound) [rows, 128] of query rows q over K, V [keys, 128]; seen
    [rows, keys], a key at least in each row.  wrong: a function of the scores
    that stands in for them (the bound is the right scores')."""
    s = q @ K.T * scale
    y = cap * np.tanh(s / cap)
    p = _softmax(y, seen)
    aq, ak = np.abs(q), np.abs(K)
    ds = scale * ((aq @ ak.T) * (U + 2.0 ** -17) + 2.0 ** -17 * ak.sum(1)[None] + 2.0 ** -19 * aq.sum(1)[:, None])
    dy = np.maximum(cap * np.tanh((s + ds) / cap) - y, y - cap * np.tanh((s - ds) / cap)) + 4.8e-7 * cap
    e = p * np.expm1(dy)
    E = e.sum(1, keepdims=True)
    assert (E < 0.5).all()
    out, mean = p @ V, p @ np.abs(V)
    amax = np.abs(V).reshape(V.shape[0], 4, 32).max(2).min()
    assert np.exp(-2 * cap) * amax / 128 >= 2.0 ** -14, "p d_v below fp16's normal range"
    moved = e @ np.abs(V)
    bound = (moved + E * np.abs(out) + (3 * U + 2.0 ** -16) * (mean + moved)) / (1 - E) + 2.0 ** -25
    if wrong is not None:
        out = _softmax(cap * np.tanh(wrong(s) / cap), seen) @ V
    return out, bound


def telling_values(q, K, scale, cap, rng):
    """V [keys, 128]: column d follows the capped scores of row d % rows of q, so
    that that row's output depends on them in first order (values 0.25 to 1.25)."""
    t = np.tanh(q @ K.T * scale / cap)
    V = t[np.arange(128) % q.shape[0]].T
    return V + np.where(V < 0, -0.25, 0.25) + rng.uniform(-0.02, 0.02, V.shape)
