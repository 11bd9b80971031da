"""64-bit forms of the batch step's operators (numpy), and the error bounds that their tests use.

u = 2^-24 is half a step of fp32, 2^-8 of bf16 (relative)."""
import numpy as np

import draft_truth as T

U32, U16 = T.U32, T.U16


def quantise(x):
    """Rows [.., D] of f32 (or bf16 values) as the 8-bit cache holds them: int8 entries, f32 scales. numpy's f32 quotients
    are rounded to nearest, as the definition has them."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(-1)
        scale = (top / np.float32(127)).astype(np.float32)
        q = np.clip(np.rint(x / scale[..., None]), -127, 127)
        ok = np.isfinite(x).all(-1)
        q = np.where((ok & (scale > 0))[..., None], q, 0).astype(np.int8)
    return q, np.where(ok, scale, np.float32(np.nan))


def values(q, scale, to=np.float64):
    return q.astype(to) * scale[..., None].astype(to)


def prefix_of(first, b):
    """The prefix of sequence b, or -1."""
    return next((g for g in range(len(first) - 1) if first[g] <= b < first[g + 1]), -1)


def prefix_attention(q, kc, vc, kd, vd, lens, counts, parents, scale, kp, vp, plens, first, gate=None, out=None):
    """draft_truth.tree_attention with prefixes kp, vp [G, pcap, K, D] ahead of the sequences' own rows; kd None: the
    nodes' rows are rows lens[b] + i of the caches. -> (out in float64, sum of |p v|, largest sum of |q k| scale, keys)."""
    B, N = q.shape[:2]
    o = np.zeros(q.shape) if out is None else out.astype(np.float64).copy()
    mag, qk, keys = np.zeros(q.shape), np.zeros(q.shape[:3]), np.ones(B)
    for b in range(B):
        g, n = prefix_of(first, b), lens[b]
        P = plens[g] if g >= 0 else 0
        cat = lambda c, p: np.concatenate([p[g, :P], c[b, :n]])[None] if g >= 0 else c[b:b + 1, :n]  # noqa: E731
        dr = lambda c, d: (c[b:b + 1, n:n + N] if d is None else d[b:b + 1])  # noqa: E731
        own = lambda x: None if x is None else x[b:b + 1]  # noqa: E731
        o[b:b + 1], mag[b:b + 1], qk[b:b + 1] = T.tree_attention(
            q[b:b + 1], cat(kc, kp), cat(vc, vp), dr(kc, kd), dr(vc, vd), [n + P], counts[b:b + 1], parents[b:b + 1], scale,
            gate=own(gate), out=o[b:b + 1])
        keys[b] = n + P + N
    return o, mag, qk, keys


def bound8(q, kmax, vmax, scale, keys, gate=None):
    """What 8-bit rows add to draft_truth.tree_attention_bound: a query's entries to 2^-22 of its row's largest a at
    most, so a score to 2^-22 a sum |k| <= 2^-22 a D kmax, which the output's weights then err by twice (their own and
    the quotient's); probabilities times their row's scale to 2^-22 of the stage's largest, so the output by
    2^-22 of the largest value per key. kmax, vmax: the largest |entry * scale| of keys and values."""
    D = q.shape[-1]
    a = np.abs(q.astype(np.float64)).max(-1, keepdims=True)
    g = 1.0 if gate is None else 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
    return (2.0 * 2.0 ** -22 * a * D * kmax * abs(scale) * vmax + 2.0 ** -22 * np.asarray(keys)[:, None, None, None] * vmax) * g


def sample(x, u, t=1.0, k=0, top_p=1.0, min_p=0.0):
    """One row: (token, p in float64, distance of u and of each threshold from the nearest border that decides them).
    Distances are relative to the whole: a test leaves out what lies within the sums' rounding."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    if not np.isfinite(m):
        return -1, np.zeros(x.shape), 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    if t == 0:
        t, k = 1.0, 1
    near = 1.0
    order = order[:k] if k else order
    w = np.exp((x[order] - m) / t)
    n = len(w)
    if top_p < 1:
        cum = np.cumsum(w)
        n = 1 + int(np.searchsorted(cum, top_p * cum[-1], side="left"))
        near = min(near, np.abs(cum - top_p * cum[-1]).min() / cum[-1])
        n = min(n, len(w))
    n = max(1, min(n, int((w >= min_p).sum())))
    if min_p > 0:
        near = min(near, np.abs(w - min_p).min() if min_p < 1 else 1.0)
    p = np.zeros(len(x))
    p[order[:n]] = w[:n] / w[:n].sum()
    cum = np.cumsum(p)
    tok = int(np.searchsorted(cum, u * cum[-1], side="right"))
    live = cum[p > 0]
    near = min(near, np.abs(live[:-1] - u * cum[-1]).min() if len(live) > 1 else 1.0)
    return tok, p, near
