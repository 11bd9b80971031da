"""GPU checks of the batch step's operators at their edges: full caches, padding, ranges of settings, odd memory."""
import numpy as np
import pytest

import batch_truth as BT
import draft_truth as T
from test_gpu_batch import _both, _dt, _kv, _reported, _sample_check
from test_gpu_drafts import _i, _np, _t

pytestmark = pytest.mark.gpu


# ---- attention --------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("B,H,K,D,N,cap", [
    (4, 8, 2, 64, 1, 4000),      # many pieces of few rows
    (40, 16, 8, 128, 1, 2000),   # more rows, few pieces
    (4, 8, 2, 256, 3, 4000),
    (2, 40, 1, 192, 2, 4000),    # several row tiles
    (4, 8, 2, 80, 2, 300),       # a head dim off the matrix cores
])
def test_full_cache_without_prefixes(own_ctx, kind, B, H, K, D, N, cap):
    """Nodes' rows in the cache: a sequence whose rows do not fit it is left as it was and reported, whether or not its length
    alone does; the others' bits stay."""
    import torch
    ctx, rng = own_ctx, np.random.default_rng(61)
    cache = _both(_kv(rng, kind, B, cap, K, D), _kv(rng, kind, B, cap, K, D))
    q = _t(rng.standard_normal((B, N, H, D)).astype(np.float32))
    lens = rng.integers(cap // 2, cap - N + 1, B)
    lens[0] = cap - N  # the last that fits

    def run(at):
        out = torch.full_like(q, 3.0)
        ctx.gqa_prefix(q, cache, _i(at), _i([N] * B), D ** -0.5, out, sync=False)
        return out
    good = run(lens)
    ctx.sync()
    assert torch.isfinite(good).all() and (good != 3.0).any(-1).all()
    for full in (cap, cap - N + 1):
        at = lens.copy()
        at[1] = full
        out = run(at)
        _reported(ctx)
        keep = [b for b in range(B) if b != 1]
        assert (out[1] == 3.0).all() and torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("kind", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("D", [64, 256, 80])
@pytest.mark.parametrize("N", [1, 3])
def test_padding_queries(ctx, kind, D, N):
    """Queries and gates of padding nodes and of sequences without nodes, behind a prefix they share with others: whatever
    they hold, the others' bits stay."""
    import torch
    rng = np.random.default_rng(62)
    B, H, K, cap, pcap = 4, 8, 2, 40, 500
    cache, draft, prefix = [_both(_kv(rng, kind, n, c, K, D), _kv(rng, kind, n, c, K, D)) for n, c in ((B, cap), (B, N), (1, pcap))]
    counts = [N, 0, N, max(0, N - 2)]
    q, gate = [_t(rng.standard_normal((B, N, H, D)).astype(np.float32)) for _ in range(2)]
    live = torch.arange(N, device="cuda")[None] < _i(counts)[:, None]

    def run(qq, gg):
        out = torch.full_like(q, 3.0)
        ctx.gqa_prefix(qq, cache, _i([5, 0, 33, 8]), _i(counts), D ** -0.5, out, draft=draft, prefix=prefix, prefix_len=_i([pcap - 1]),
                       prefix_first=_i([0, B]), gate=gg)
        return out
    good = run(q, gate)
    assert torch.isfinite(good).all() and (good[~live] == 3.0).all()
    for bad in (1e7, 1e30, float("inf"), float("nan")):
        qq, gg = q.clone(), gate.clone()
        qq[~live] *= bad
        gg[~live] = bad
        assert torch.equal(run(qq, gg), good), bad


# ---- 8-bit rows -------------------------------------------------------------------------------------
def test_read_back_refuses_sides_over_each_other(ctx):
    """Rows of k and of v that share an entry are refused; sides that lie within each other, between rows, are not."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(63)
    B, Tn, K, D = 2, 5, 3, 64
    cache = (_t(rng.integers(-127, 128, (B, Tn, K, D)).astype(np.int8)), _t(rng.integers(-127, 128, (B, Tn, K, D)).astype(np.int8)),
             _t(rng.random((B, Tn, K)).astype(np.float32)), _t(rng.random((B, Tn, K)).astype(np.float32)))
    want = [BT.values(_np(cache[i]), _np(cache[2 + i]), np.float32) for i in (0, 1)]
    n = B * Tn * K * D
    buf = torch.zeros(4 * n + 512, device="cuda")
    dense = lambda at: buf[at:at + n].view(B, Tn, K, D)  # noqa: E731
    wide = lambda at: buf[at:at + 2 * n].view(B, Tn, 2 * K, D)[:, :, :K]  # noqa: E731
    sides = lambda i: buf[:2 * n].view(K, 2, B, Tn, D)[:, i].permute(1, 2, 0, 3)  # noqa: E731
    rows = lambda at: buf[at:at + 2 * n].view(B, Tn, K, 2 * D)[..., :D]  # noqa: E731
    for k, v in ((dense(0), dense(0)), (dense(0), dense(n - 1)), (dense(1), dense(0)), (dense(n - 4), dense(0)), (wide(0), wide(0)),
                 (wide(0), wide((K - 1) * D)), (wide(0), wide((K + 1) * D)), (wide(0), wide(2 * K * D * 7)), (rows(0), rows(D - 1)),
                 (rows(0), rows(2 * D * (K * Tn * B - 1))), (rows(3 * D + 1), rows(0)), (sides(0), sides(0))):
        for a, b in ((k, v), (v, k)):
            with pytest.raises(R.RbtError, match="overlap"):
                ctx.kv_dequant(cache, a, b)
    for k, v in ((dense(0), dense(n)), (wide(0), wide(K * D)), (wide(0), wide(2 * n)), (rows(0), rows(D)), (rows(0), rows(2 * D * K * Tn * B)),
                 (rows(D), rows(2 * D * 4)), (sides(0), sides(1))):
        for a, b in ((k, v), (v, k)):
            ctx.kv_dequant(cache, a, b)
            assert np.array_equal(_np(a), want[0]) and np.array_equal(_np(b), want[1])
    # one axis of size 1 has no step; rows that no sequence writes count too
    one = lambda at: buf[at:at + n].view(B, Tn, K, D)[:, :1]  # noqa: E731
    ctx.kv_dequant(cache, one(0), one(K * D))
    assert np.array_equal(_np(one(0)), want[0][:, :1]) and np.array_equal(_np(one(K * D)), want[1][:, :1])
    with pytest.raises(R.RbtError, match="overlap"):
        ctx.kv_dequant(cache, dense(0), dense(n - D), n_rows=_i([1, 1]))


# ---- sampling ---------------------------------------------------------------------------------------
def test_draw_at_a_border_of_chunks(ctx):
    """A draw that falls between the sums of a row's chunks as doubles round them: weights are whole numbers of 2^-45, whose
    sums pass 2^53 here. With M = 2^45, the first 8000 entries weigh 4600 M + 16, the next 4000 weigh 2000 M + 32, and all of them
    13200 M + 64; half of that passes 6600 M + 16 and not 6600 M + 48, at the entry of weight 32."""
    import torch
    x = np.full(40000, -np.inf, np.float32)
    x[:4000] = x[4000:4600] = 0.0
    x[8000:10000] = 0.0
    x[12000:18600] = 0.0
    small = lambda w: np.float32(np.log(w * 2.0 ** -45))  # noqa: E731
    for i, w in ((7999, 16), (10000, 32), (20000, 16)):
        x[i] = small(w)
        assert abs(np.exp(np.float64(x[i])) * 2.0 ** 45 - w) < 0.01
    tok = torch.full((1,), -9, dtype=torch.int32, device="cuda")
    ctx.sample(_t(x[None]), _t(np.array([0.5], np.float32)), tok)
    assert int(tok[0]) == 10000


@pytest.mark.parametrize("V", [3000, 40000])
def test_min_p_at_extreme_temperatures(ctx, V):
    """Temperatures below the least normal logit differences and near the largest f32: min-p keeps what the definition does."""
    import torch
    x = np.full((2, V), -1.0, np.float32)
    t, m, u = [1e-35, 1e38], [0.5, 0.001], [0.95, 0.9999]
    x[0, 3], x[0, 7], x[0, 11] = 0.0, -2e-35, -16.3e-30  # the second's weight is e^-2, the third's e^-1630000
    x[1] = -np.inf
    x[1, 5], x[1, 9] = 3e38, -3e38                        # they lie further apart than f32 holds: e^-6
    tok, pr = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, V, device="cuda")
    f = lambda a: _t(np.asarray(a, np.float32))  # noqa: E731
    ctx.sample(_t(x), f(u), tok, temperature=f(t), min_p=f(m), probs=pr)
    for r, want in ((0, 3), (1, 9)):
        one = lambda a: float(np.float32(a[r]))  # noqa: E731
        wt, wp, _ = BT.sample(x[r], one(u), one(t), 0, 1.0, one(m))
        assert wt == want == int(tok[r])
        assert (np.abs(_np(pr)[r] - wp) <= (T.U32 + V * 2.0 ** -45) * wp + 1e-45).all()


@pytest.mark.parametrize("V", [1003, 40003])
def test_probabilities_over_the_logits(ctx, V):
    """probs may be the logits' own dense f32 rows; any other overlap is refused."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(V)
    x = _t((3 * rng.standard_normal((5, V))).astype(np.float32))
    f = lambda a: _t(np.asarray(a, np.float32))  # noqa: E731
    sets = dict(temperature=f([1, 0.7, 0, 2, 1]), top_k=_i([0, 40, 0, 0, 0]), top_p=f([1, 0.9, 1, 0.8, 1]), min_p=f([0, 0, 0, 0, 0.01]))
    u = f(rng.random(5))
    tok, want, pr = (torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros_like(x))
    ctx.sample(x, u, want, probs=pr, **sets)
    y = x.clone()
    ctx.sample(y, u, tok, probs=y, **sets)
    assert torch.equal(tok, want) and torch.equal(y, pr)
    buf = torch.zeros(6 * V + 8, device="cuda")
    wide = buf[:5 * (V + 1)].view(5, V + 1)[:, :V]
    for logits, probs in ((wide, buf[:5 * V].view(5, V)), (buf[:5 * V].view(5, V), buf[4:5 * V + 4].view(5, V)),
                          (buf.view(torch.bfloat16)[:5 * V].view(5, V), buf[:5 * V].view(5, V)),
                          (buf[5 * V - 1:6 * V - 1].view(1, V), buf[4 * V:5 * V].view(1, V))):
        n = logits.shape[0]
        with pytest.raises(R.RbtError, match="overlap"):
            ctx.sample(logits, u[:n], tok[:n], probs=probs)
    wide1 = buf[:V + 1].view(1, V + 1)[:, :V]
    ctx.sample(wide1, u[:1], tok[:1], probs=wide1.view(1, V))  # one row is dense
    ctx.sample(buf[:5 * V].view(5, V)[:1], u[:1], tok[:1], probs=buf[V:2 * V].view(1, V))  # beside it


def test_probabilities_between_the_logits_rows(ctx):
    """Logits far apart in a buffer: probabilities between two of their rows overlap none, one entry on or back they do."""
    import torch
    import rabbit_amd as R
    V = 50
    buf = torch.randn(8 * V, device="cuda")
    x, u, tok = buf.view(2, 4 * V)[:, :V], torch.full((2,), 0.5, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    want = torch.zeros(2, V, device="cuda")
    ctx.sample(x, u, tok, probs=want)
    for at in (V, 2 * V, 5 * V, 6 * V):
        pr = buf[at:at + 2 * V].view(2, V)
        ctx.sample(x, u, tok, probs=pr)
        assert torch.equal(pr, want)
    for at in (0, V - 1, 2 * V + 1, 4 * V, 5 * V - 1):
        with pytest.raises(R.RbtError, match="overlap"):
            ctx.sample(x, u, tok, probs=buf[at:at + 2 * V].view(2, V))


# ---- ranges -----------------------------------------------------------------------------------------
def _attend_check(ctx, kind, H, K, D, lens, counts, N, plens, first, drafted, gated, tree, rng, rows=None, qf=1.0):
    """One call against the 64-bit form, by its bound. rows(rng, *shape): other rows than normal ones."""
    import torch
    B, G, pcap = len(lens), len(plens), max(plens + [0]) + 2
    cap = max(lens) + N
    kv = lambda n, c: [_rows_of(rng, kind, rows, n, c, K, D) for _ in "kv"]  # noqa: E731
    (kc, vc), (kd, vd) = kv(B, cap), kv(B, N)
    kp, vp = kv(G, pcap) if G else ((None, None), (None, None))
    q = (qf * rng.standard_normal((B, N, H, D))).astype(np.float32)
    gate = rng.standard_normal((B, N, H, D)).astype(np.float32) if gated else None
    par = T.random_parents(rng, B, N, tree)
    out, scale = torch.full((B, N, H, D), 3.0, device="cuda"), D ** -0.5
    ctx.gqa_prefix(_t(q), _both(kc, vc), _i(lens), _i(counts), scale, out, draft=_both(kd, vd) if drafted else None,
                   parent=None if tree == "chain" else _i(par), prefix=_both(kp, vp) if G else None, prefix_len=_i(plens) if G else None,
                   prefix_first=_i(first) if G else None, gate=None if gate is None else _t(gate))
    want, mag, qk, keys = BT.prefix_attention(q, kc[1], vc[1], kd[1] if drafted else None, vd[1] if drafted else None, lens, counts, par,
                                              scale, kp[1], vp[1], plens, first, gate=gate, out=np.full(q.shape, 3.0))
    tol = T.tree_attention_bound(mag, qk, keys[:, None, None, None], D)
    if kind == "i8":
        # (a score's error is the query's largest entry times the sum of a key's, which for rows of unequal entries is less
        # than D times the largest: the largest such sum of any key here)
        some = [x for x in ((kc, vc), (kd, vd) if drafted else None, (kp, vp) if G else None) if x]
        ksum = max(np.abs(k[1].astype(np.float64)).sum(-1).max() for k, _ in some)
        vmax = max(np.abs(v[1]).max() for _, v in some)
        tol = tol + BT.bound8(q, ksum / D, vmax, scale, keys, gate)
    live = np.arange(N)[None] < np.array(counts)[:, None]
    got = _np(out)
    assert (got[~live] == 3.0).all()
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol)[live].all(), (err[live].max(), (err / tol)[live].max())
    return np.linalg.norm(err[live]) / np.linalg.norm(want[live])


def _rows_of(rng, kind, rows, *shape):
    if rows is None:
        return _kv(rng, kind, *shape)
    x = rows(rng, *shape).astype(np.float32)
    if kind == "i8":
        q, s = BT.quantise(x)
        return (_t(q), _t(s)), BT.values(q, s)
    return (_t(x),), x


@pytest.mark.parametrize("kind", ["i8", "bf16", "f32"])
@pytest.mark.parametrize("H,K,D,N,lens,counts,plens,first,drafted,tree", [
    (16, 2, 64, 256, [70, 3], [256, 200], [200], [0, 2], True, "chain"),     # a prompt's chunk: the most nodes, eight row tiles
    (8, 2, 128, 130, [0, 40, 65], [130, 33, 64], [129, 5], [0, 1, 3], False, "tree"),
    (12, 1, 192, 40, [100, 31], [40, 17], [], [0], False, "chain"),          # no prefix, the nodes' rows in the cache
    (8, 2, 256, 70, [33, 20], [70, 65], [90], [0, 2], True, "tree"),
    (4, 2, 80, 100, [9, 0], [100, 71], [60], [0, 2], False, "tree"),
])
def test_attend_many_nodes(ctx, kind, H, K, D, N, lens, counts, plens, first, drafted, tree):
    """Chunks of a prompt and large trees: drafted rows over several stages and words of the visibility bits."""
    rel = _attend_check(ctx, kind, H, K, D, lens, counts, N, plens, first, drafted, True, tree, np.random.default_rng(D + N))
    assert rel <= 4e-6  # test_attend's bound of the whole


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("side", ["q", "kv"])
def test_attend_8bit_unequal_channels(ctx, D, side):
    """A channel of the queries, or of the keys and values, 100 times the others: within the bound that the largest entry gives."""
    rng = np.random.default_rng(71)
    f = np.ones(D)
    f[3] = 100.0 if side == "kv" else 0.01
    rows = lambda r, *s: r.standard_normal(s) * f  # noqa: E731
    _attend_check(ctx, "i8", 8, 2, D, [40, 300, 0], [1, 1, 1], 1, [700], [0, 3], False, False, "chain", rng, rows=rows,
                  qf=1.0 / f[3] if side == "kv" else 1.0 / f)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("kf,vf", [(-53, 65), (65, -53), (65, 65), (-53, -53)])
def test_attend_8bit_scales(ctx, D, kf, vf):
    """Scales at both ends of 2^-60 to 2^60, and a little past the upper one: keys' and values' rows times 2^kf and 2^vf (a row's
    largest of 64 or 256 normal numbers lies between 1 and 6, so scales 4.4 to 7 bits below), queries the other way."""
    import torch
    rng = np.random.default_rng(72)
    H, K, cap, pcap = 8, 2, 60, 500
    rows = [[BT.quantise(np.ldexp(rng.standard_normal((n, c, K, D)), f).astype(np.float32)) for f in (kf, vf)] for n, c in ((3, cap), (1, pcap))]
    assert all(2.0 ** -60 <= s.min() and s.max() <= 2.0 ** 60.6 for r in rows for _, s in r)
    t = [tuple(_t(x) for x in (k[0], v[0], k[1], v[1])) for k, v in rows]
    q = np.ldexp(rng.standard_normal((3, 1, H, D)), -kf).astype(np.float32)
    out = torch.zeros(3, 1, H, D, device="cuda")
    lens = [59, 0, 30]
    ctx.gqa_prefix(_t(q), t[0], _i(lens), _i([1] * 3), D ** -0.5, out, prefix=t[1], prefix_len=_i([499]), prefix_first=_i([0, 3]))
    (kc, vc), (kp, vp) = [[BT.values(*x) for x in r] for r in rows]
    want, mag, qk, keys = BT.prefix_attention(q, kc, vc, None, None, lens, [1] * 3, np.full((3, 1), -1), D ** -0.5, kp, vp, [499], [0, 3])
    tol = T.tree_attention_bound(mag, qk, keys[:, None, None, None], D) + BT.bound8(
        q, max(np.abs(kc).max(), np.abs(kp).max()), max(np.abs(vc).max(), np.abs(vp).max()), D ** -0.5, keys)
    err = np.abs(_np(out) - want)
    assert (err <= tol).all()
    assert np.linalg.norm(err) <= 4e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("V", [5000, 70000])
def test_sample_small_min_p(ctx, V):
    """min-p between 0 and e^-21.3, whose bucket is past the last, alone and with the others. What is kept goes by the weights
    themselves (to 2^-48 of each), not by sums: no weight here is within 2^-44 of its min-p."""
    import torch
    rng = np.random.default_rng(V)
    x = (8 * rng.standard_normal((8, V))).astype(np.float32)
    t, m = [1, 1, 1, 0.5, 1, 1, 1, 1], [1e-10, 1e-12, 1e-20, 1e-30, 1e-44, 1e-12, 1e-10, 5e-10]
    k, p, u = [0, 0, 0, 0, 0, 3000, 0, 100], [1, 1, 1, 1, 1, 1, 0.999, 0.9], rng.random(8)
    f = lambda a: _t(np.asarray(a, np.float32))  # noqa: E731
    tok, pr = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.full((8, V), 7.0, device="cuda")
    ctx.sample(_t(x), f(u), tok, temperature=f(t), top_k=_i(k), top_p=f(p), min_p=f(m), probs=pr)
    for r in range(8):
        tok_r, wp, off = _small_min_p_row(x[r], u[r], t[r], k[r], p[r], m[r])
        g = _np(pr)[r].astype(np.float64)
        assert int(tok[r]) == tok_r
        assert (g[wp == 0] == 0).all() and (np.abs(g - wp) <= (T.U32 + 2 * off) * wp + 1e-45).all()


def _small_min_p_row(x, *a):
    """(token, p, the sums' error), the answers being certain."""
    u, t, k, p, m = [float(np.float32(v)) for v in a]
    off = len(x) * 2.0 ** -46 + 2.0 ** -48
    w = np.exp((x.astype(np.float64) - x.max()) / t)
    assert (np.abs(w - m) > 2.0 ** -44 * m).all()
    tok, wp, _ = BT.sample(x, u, t, int(k), p, m)
    assert BT.sample(x, u, t, int(k), p, 0.0)[2] > 2 * off or p == 1.0
    assert np.abs(np.cumsum(wp)[wp > 0] - u).min() > 2 * off
    return tok, wp, off


@pytest.mark.parametrize("V", [20000, 131072])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sample_masked_and_flat_rows(ctx, V, dtype):
    """Rows masked to fewer tokens than top-k, by -inf, the type's lowest value and NaN; rows without spikes, whose thresholds lie
    among thousands of entries."""
    import torch
    rng = np.random.default_rng(V)
    x = np.full((6, V), -np.inf, np.float32)
    x[1] = float(torch.finfo(_dt(dtype)).min)
    x[2] = np.nan
    for r in range(3):
        x[r, rng.choice(V, 20, replace=False)] = rng.standard_normal(20)
    x[3:] = rng.standard_normal((3, V))
    x[4] *= 2.5
    u = rng.random(6)
    for k, p, m, t in ((50, 1.0, 0.0, 1.0), (50, 0.9, 0.01, 0.8), (0, 0.9, 0.0, 1.0), (21, 0.5, 0.0, 2.0)):
        _sample_check(ctx, x, u, dtype, [t] * 6, [k] * 6, [p] * 6, [m] * 6)
