"""Scored and tree attention in 64 bits, and how far the kernels may be from it.

The rows' scores are s = scale q.k, then cap tanh(s / cap), or s + slope
(key position - row position); the softmax runs over the keys a row sees.

Bound of an output element, by the roundings on its way (u = 2^-11, half a
step of fp16):
  * K^ = int8 * scale is rounded to fp16 once: a score is off by at most
    ds = u * scale * sum_d |q_d k_d| (a cap only shrinks it: |tanh'| <= 1), and
    a softmax weight relative to the others by 2 ds;
  * a weight is rounded to fp16, its product with V's scale (or V^ = int8 *
    scale) again, and the weights' sum may be that of the rounded ones: 3 u;
  * weights below fp16's range: the largest weight is at least 1 as the kernel
    holds it (its running maximum lags the true one downwards only), so a weight
    that is rounded to a multiple of 2^-24 loses 2^-25 of at least 1, and the
    product with a V scale the same, times at most 127 steps: 2^-25 (|v| + 127)
    a key, over a total weight of at least 1;
  * fp32 arithmetic of the exponent (scores up to 2^7 in log2 units): 2^-16;
  * the output's own rounding, eps / 2.
"""
import numpy as np
import torch

from gpu_common import seq_head_kv, to_np_f32

U = 2.0 ** -11


def row_scores(q, K, scale, pos, cap=0.0, slope=None):
    """q [n, 128], K [keys, 128], pos [n] -> scores [n, keys], all float64."""
    s = q @ K.T * scale
    if cap:
        s = cap * np.tanh(s / cap)
    if slope is not None:
        s = s + slope * (np.arange(K.shape[0])[None] - pos[:, None])
    return s


def seen_keys(sl, nq, j, q_abs=None, causal=True, masks=None):
    """[rows, sl] truth: which keys row j of a sequence sees."""
    key = np.arange(sl)[None]
    if masks is not None:
        node = key - (sl - nq)
        bits = np.array([[(int(m) >> int(max(n, 0))) & 1 if n < 64 else 0 for n in node[0]] for m in masks], bool)
        bits = bits.reshape(len(masks), sl)
        return (node < 0) | (bits & (node <= np.asarray(j)[:, None]))
    if not causal:
        return np.ones((len(j), sl), bool)
    return key <= (sl - nq if q_abs is None else q_abs) + np.asarray(j)[:, None]


def scored_oracle(b, cap=0.0, slopes=None, masks=None, q_abs=None, causal=True, out_eps=0.0, skip=()):
    """(out, bound) float64 [T, Hq, 128] of a workloads.Batch, from the cache as the
    GPU wrote it.  skip: query rows left 0 with an infinite bound."""
    q = to_np_f32(b.query).astype(np.float64)
    G = b.Hq // b.Hkv
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    for s in range(b.num_seqs):
        a, e = int(b.qsl[s]), int(b.qsl[s + 1])
        sl, nq = int(b.seq_lens[s]), e - a
        if nq == 0 or sl <= 0:
            continue
        j = np.arange(nq)
        qa = sl - nq if q_abs is None else int(q_abs[s])
        seen = seen_keys(sl, nq, j, qa, causal, None if masks is None else masks[a:e])
        for h in range(b.Hkv):
            K, V = (x.astype(np.float64) for x in seq_head_kv(b, s, h))
            K, V = np.nan_to_num(K, posinf=0, neginf=0), np.nan_to_num(V, posinf=0, neginf=0)
            for hq in range(h * G, (h + 1) * G):
                x = q[a:e, hq]
                sc = row_scores(x, K, b.scale, qa + j, cap, None if slopes is None else float(slopes[hq]))
                sc = np.where(seen, sc, -np.inf)
                m = sc.max(1, keepdims=True)
                p = np.exp(sc - np.where(np.isfinite(m), m, 0.0))
                l = p.sum(1, keepdims=True)
                p = p / np.where(l > 0, l, 1.0)
                out[a:e, hq] = p @ V
                ds = U * b.scale * (np.abs(x) @ np.abs(K).T * seen).max(1, keepdims=True)
                small = seen.sum(1, keepdims=True) * 2.0 ** -25 * (np.abs(V).max() + 127)
                mean = p @ np.abs(V)
                bound[a:e, hq] = (2 * ds + 3 * U + 2.0 ** -16) * (1 + 2 * ds) * mean + small
    bound += out_eps / 2 * (np.abs(out) + bound)
    for t in skip:
        out[t], bound[t] = 0.0, np.inf
    return out, bound


def check(out, ref, bound):
    o = to_np_f32(out).astype(np.float64)
    fine = np.isfinite(bound)
    assert np.isfinite(o[fine]).all(), "non-finite output"
    off = np.abs(o - ref)
    worst = np.unravel_index(np.argmax(np.where(fine, off - bound, -np.inf)), off.shape)
    assert (off <= bound)[fine].all(), f"off by {off[worst]:.3e} at {worst}, bound {bound[worst]:.3e}"
    norm = np.linalg.norm(ref[fine])
    if norm:  # far below the elements' bound, as the roundings are independent
        assert np.linalg.norm(off[fine]) <= 1e-2 * norm


def eps_of(dt):
    return torch.finfo(dt).eps


def random_tree(rng, n):
    return [-1 if i == 0 or rng.random() < 0.2 else int(rng.integers(0, i)) for i in range(n)]
