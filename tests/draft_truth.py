"""64-bit forms of the drafted-token operators (numpy), and the error bounds that their tests use.

u = 2^-24 is half a step of fp32, 2^-8 of bf16 (relative)."""
import math

import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -8


def ancestors(parent, i):
    """Node i and the nodes above it."""
    seen = []
    while i >= 0:
        seen.append(i)
        i = int(parent[i])
    return sorted(seen)


def tree_attention(q, kc, vc, kd, vd, lens, counts, parents, scale, gate=None, out=None):
    """q [B, T, H, D], caches [B, cap, K, D], drafts [B, T, K, D] -> (out [B, T, H, D] in float64, the sum of
    |p v| per output entry, the largest sum of |q k| scale per row). Rows past counts[b] keep `out`."""
    B, T, H, D = q.shape
    K = kc.shape[2]
    R = H // K
    o = np.zeros(q.shape) if out is None else out.astype(np.float64).copy()
    mag, qk = np.zeros(q.shape), np.zeros((B, T, H))
    for b in range(B):
        for i in range(counts[b]):
            at = ancestors(parents[b], i)
            k = np.concatenate([kc[b, :lens[b]], kd[b, at]]).astype(np.float64)
            v = np.concatenate([vc[b, :lens[b]], vd[b, at]]).astype(np.float64)
            for h in range(H):
                kk, vv, x = k[:, h // R], v[:, h // R], q[b, i, h].astype(np.float64)
                s = kk @ x * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                y = p @ vv
                mag[b, i, h] = p @ np.abs(vv)
                qk[b, i, h] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                if gate is not None:
                    g = 1.0 / (1.0 + np.exp(-gate[b, i, h].astype(np.float64)))
                    y = y * g
                    mag[b, i, h] *= g
                o[b, i, h] = y
    return o, mag, qk


def tree_attention_bound(mag, qk, keys, D):
    """How far fp32 sums of exact products may be off. A score's sum of D products on the matrix cores: chains
    whose steps err by at most 64u of what they add and hold (three steps per 32 products at least, every
    step's magnitude at most the whole): 6 D u of sum |q k|. An exponential then errs by that twice (its own
    and the maximum's, the softmax's quotient cancelling neither) and 2^-20 for its argument's scaling and the
    function; the sums over the keys by 6 u a key; the quotient, the gate and the joining of parts by 2^-20."""
    return (2 * 6 * D * U32 * qk[..., None] + 12 * keys * U32 + 2.0 ** -19) * mag + 1e-37


def rope(x, pos, inv, factor, start, rope_dim, pairs, norm=None, eps=1e-6, rotate=True, angle_f32=False):
    """x [s, h, d] -> (rows in float64, the magnitude that their rounding errors scale with)."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * (1.0 + norm.astype(np.float64))
    y, mag = x.copy(), np.abs(x)
    if rotate and rope_dim:
        ang = pos.astype(np.float64)[:, None] * inv
        if angle_f32:
            ang = (pos.astype(np.float32)[:, None] * inv.astype(np.float32)).astype(np.float64)
        c, s = (np.cos(ang) * factor)[:, None], (np.sin(ang) * factor)[:, None]
        e = start + rope_dim
        ia, ib = (slice(start, e, 2), slice(start + 1, e, 2)) if pairs else \
            (slice(start, start + rope_dim // 2), slice(start + rope_dim // 2, e))
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        m = (np.abs(a) + np.abs(b)) * abs(factor)
        mag[..., ia], mag[..., ib] = m, m
    return y, mag


def verify(tokens, parent, counts, p, q, u):
    """(path, n_path, next) as rbt_draft_verify_d's description has them, one sequence after the other."""
    B, T, V = p.shape
    path, n_path, nxt = np.full((B, T), -1, np.int32), np.zeros(B, np.int32), np.full(B, -1, np.int32)
    for b in range(B):
        if counts[b] == 0:
            continue
        cur, way = 0, [0]
        c, S, gone = 0.0, 1.0, []

        def left():
            r = p[b, cur].astype(np.float64)
            if q is not None and c > 0:
                r = r - c * q[b, cur].astype(np.float64)
            r = np.where(r > 0, r, 0.0)
            r[gone] = 0.0
            return r

        for i in range(1, counts[b]):
            x = int(tokens[b, i])
            if parent[b, i] != cur or not 0 <= x < V:
                continue
            qx = 1.0 if q is None else float(q[b, cur, x])
            if float(u[b, i]) * (S * qx) < left()[x]:
                cur, c, S, gone = i, 0.0, 1.0, []
                way.append(i)
            elif q is None:
                S -= left()[x]
                gone.append(x)
            else:
                c += S
                S = left().sum()
        r = left()
        if not r.sum() > 0:
            c, gone, r0 = 0.0, [], p[b, cur].astype(np.float64)
            r = np.where(r0 > 0, r0, 0.0)
        path[b, :len(way)], n_path[b] = way, len(way)
        if r.sum() > 0 and math.isfinite(r.sum()):
            nxt[b] = min(int(np.searchsorted(np.cumsum(r), float(u[b, 0]) * np.cumsum(r)[-1], side="right")),
                         int(np.flatnonzero(r > 0)[-1]))
    return path, n_path, nxt


def random_parents(rng, B, T, shape="tree"):
    """[B, T] int32: "tree" (each node below any earlier one), "chain", "forest" (several roots)."""
    par = np.full((B, T), -1, np.int32)
    for i in range(1, T):
        par[:, i] = i - 1 if shape == "chain" else rng.integers(-1 if shape == "forest" else 0, i, B)
    return par


def _bf16_bits(x):
    """float32 rounded to the nearest bf16, as float32."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7fff + (b >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)


def bf16_parts(x):
    """float32 as the sum of three bf16 rounded to nearest; a first part past the largest bf16 stays that."""
    x = np.asarray(x, np.float32)
    top = np.array(0x7f7f0000, np.uint32).view(np.float32)
    hi = _bf16_bits(np.clip(x, -top, top))
    mid = _bf16_bits(x - hi)
    return hi, mid, _bf16_bits(x - hi - mid)


def six_products(x, y):
    """The products of parts that the matrix cores take for x y, summed in float64: hi hi, hi mid, mid hi, mid mid,
    hi lo and lo hi. With |mid| <= 2^-8 and |lo| <= 2^-17 of the whole, the rest is at most 2^-24 + 2^-34 of it."""
    a, b = (np.asarray(bf16_parts(v), np.float64) for v in (x, y))
    return sum(a[i] * b[j] for i in range(3) for j in range(3) if i + j <= 2)
