"""GPU checks of the batch step's operators together, as a serving loop has them: written to 8 bits, attended to behind
shared prefixes, sampled from, verified and committed, eagerly and captured; and of their longer and odder calls."""
import numpy as np
import pytest

import batch_truth as BT
import draft_truth as T
from test_gpu_batch import _both, _dt, _kv, _reported, _sample_check
from test_gpu_drafts import _bf, _i, _np, _t

pytestmark = pytest.mark.gpu


class _Loop:
    """One layer's decode step of B users, N nodes each, behind prefixes in an 8-bit cache: buffers and calls."""

    def __init__(self, rng, B, N, H, K, D, V, cap, plens, first):
        import torch
        self.B, self.N, self.H, self.K, self.D, self.V, self.cap = B, N, H, K, D, V, cap
        z = lambda *s, dt="float32": torch.zeros(*s, dtype=_dt(dt), device="cuda")  # noqa: E731
        cache = lambda n, rows: (z(n, rows, K, D, dt="int8"), z(n, rows, K, D, dt="int8"), z(n, rows, K), z(n, rows, K))  # noqa: E731
        self.x, self.out = z(B, N, H + 2 * K, D), z(B, N, H, D)
        self.cache, self.draft = cache(B, cap), cache(B, N)
        self.prefix = cache(len(plens), max(plens) + 2)
        self.plens, self.first = _i(plens), _i(first)
        self.len, self.len2, self.n, self.parent = _i([0] * B), _i([0] * B), _i([N] * B), _i(np.tile(np.arange(-1, N - 1), (B, 1)))
        self.w = _t((rng.standard_normal((H * D, V)) * 2 / (H * D) ** 0.5).astype(np.float32))
        self.logits, self.probs = z(B * N, V), z(B, N, V)
        self.u, self.uv = z(B * N), z(B, N)
        self.t, self.k = _t(np.full(B * N, 0.8, np.float32)), _i([12] * (B * N))
        self.p, self.m = _t(np.full(B * N, 0.95, np.float32)), _t(np.full(B * N, 0.001, np.float32))
        self.drawn, self.tok = z(B * N, dt="int32"), z(B, N, dt="int32")
        self.path, self.n_path, self.next = z(B, N, dt="int32"), z(B, dt="int32"), z(B, dt="int32")

    def attend(self, ctx, q, sync=True):
        k, v = self.x[:, :, self.H:self.H + self.K], self.x[:, :, self.H + self.K:]
        ctx.kv_quant(k, v, self.draft, n_rows=self.n, sync=sync)
        ctx.gqa_prefix(q, self.cache, self.len, self.n, self.D ** -0.5, self.out, draft=self.draft, parent=self.parent,
                       prefix=self.prefix, prefix_len=self.plens, prefix_first=self.first, sync=sync)

    def choose(self, ctx, sync=True):
        ctx.sample(self.logits, self.u, self.drawn, self.t, self.k, self.p, self.m, probs=self.probs.view(self.B * self.N, -1), sync=sync)
        ctx.draft_verify(self.tok, self.parent, self.n, self.probs, self.uv, self.path, self.n_path, self.next, sync=sync)
        c, d = [[t] for t in self.cache], [[t] for t in self.draft]
        ctx.kv_commit(c[0], c[1], d[0], d[1], self.path, self.n_path, self.len, self.len2, sync=sync)
        c, d = [[t.unsqueeze(-1)] for t in self.cache], [[t.unsqueeze(-1)] for t in self.draft]
        ctx.kv_commit(c[2], c[3], d[2], d[3], self.path, self.n_path, self.len, self.len2, sync=sync)

    def run(self, ctx):
        import torch
        self.attend(ctx, self.x[:, :, :self.H].contiguous())
        torch.mm(self.out.view(self.B * self.N, -1), self.w, out=self.logits)
        self.choose(ctx)

    def fill(self, rng, rep):
        B, N = self.B, self.N
        self.x.copy_(_t(rng.standard_normal(tuple(self.x.shape)).astype(np.float32)))
        self.n.copy_(_i([N] + [int(c) for c in rng.integers(0, N + 1, B - 1)]))
        self.parent.copy_(_i(T.random_parents(rng, B, N, ("tree", "chain")[rep % 2])))
        self.u.copy_(_t((rng.integers(0, 2 ** 24, B * N) / 2.0 ** 24).astype(np.float32)))
        self.uv.copy_(_t((rng.integers(0, 2 ** 24, (B, N)) / 2.0 ** 24).astype(np.float32)))
        self.tok.copy_(_i(rng.integers(0, self.V, (B, N))))
        if rep:  # some drafts are what the target has drawn, so that paths of several nodes stand
            self.tok[:, 1:] = self.drawn.view(B, N)[:, :-1]
        plens = self.plens.cpu().numpy().copy()
        plens[0] = int(rng.integers(1, self.prefix[0].shape[1] + 1))
        self.plens.copy_(_i(plens))

    STATE = ("cache", "len2", "out", "probs", "drawn", "path", "n_path", "next", "draft")

    def state(self):
        return [t.clone() for n in self.STATE for t in (getattr(self, n) if isinstance(getattr(self, n), tuple) else (getattr(self, n),))]

    def put(self, st):
        it = iter(st)
        for n in self.STATE:
            for t in (getattr(self, n) if isinstance(getattr(self, n), tuple) else (getattr(self, n),)):
                t.copy_(next(it))


def _loop(ctx, rng, B=5, N=4, H=16, K=2, D=64, V=300, cap=60, plens=(130, 40), first=(0, 3, 4)):
    s = _Loop(rng, B, N, H, K, D, V, cap, list(plens), list(first))
    rows = rng.standard_normal((2, len(plens), s.prefix[0].shape[1], K, D)).astype(np.float32)
    ctx.kv_quant(_t(rows[0]), _t(rows[1]), s.prefix)
    return s


def test_step_against_64_bits(own_ctx):
    """Four steps of a batch: each operator's result from what the one before it left, against the 64-bit forms."""
    ctx, rng = own_ctx, np.random.default_rng(21)
    s = _loop(ctx, rng)
    B, N, H, K, D = s.B, s.N, s.H, s.K, s.D
    for rep in range(4):
        s.fill(rng, rep)
        before, lens, counts, par = [_np(t).copy() for t in s.cache], _np(s.len).copy(), _np(s.n), _np(s.parent)
        s.out.fill_(3.0)
        s.run(ctx)
        x = _np(s.x)
        qd, sd = BT.quantise(x[:, :, H:])
        draft = [_np(t) for t in s.draft]
        live = np.arange(N)[None] < counts[:, None]
        for i, lo in ((0, 0), (1, K)):
            assert np.array_equal(draft[i][live], qd[:, :, lo:lo + K][live])
            assert np.array_equal(draft[2 + i][live], sd[:, :, lo:lo + K][live])
        val = [BT.values(r[i], r[2 + i]) for r in (before, draft, [_np(t) for t in s.prefix]) for i in (0, 1)]
        want, mag, qk, keys = BT.prefix_attention(x[:, :, :H], *val[:4], lens, counts, par, D ** -0.5, *val[4:], _np(s.plens).tolist(),
                                                  _np(s.first).tolist(), out=np.full((B, N, H, D), 3.0))
        tol = T.tree_attention_bound(mag, qk, keys[:, None, None, None], D) + BT.bound8(
            x[:, :, :H], max(np.abs(t).max() for t in val[::2]), max(np.abs(t).max() for t in val[1::2]), D ** -0.5, keys)
        got = _np(s.out)
        assert (np.abs(got - want) <= tol)[live].all() and (got[~live] == 3.0).all()
        lg, pr, drawn = _np(s.logits), _np(s.probs).reshape(B * N, -1), _np(s.drawn)
        f = lambda v: float(np.float32(v))  # noqa: E731
        for r in np.flatnonzero(live.ravel()):
            tok, p, near = BT.sample(lg[r], float(_np(s.u)[r]), f(0.8), 12, f(0.95), f(0.001))
            off = s.V * 2.0 ** -46 + 2.0 ** -48
            assert near > 2 * off and drawn[r] == tok and (np.abs(pr[r] - p) <= (T.U32 + 2 * off) * p + 1e-45).all()
        path, m, after = _np(s.path), _np(s.n_path), [_np(t) for t in s.cache]
        assert np.array_equal(_np(s.len2), lens + m)
        for b in range(B):
            for c, bf, d in zip(after, before, draft):
                w = bf[b].copy()
                w[lens[b]:lens[b] + m[b]] = d[b, path[b, :m[b]]]
                assert np.array_equal(c[b], w)
        s.len.copy_(s.len2)
        assert int(s.len.max()) <= s.cap - N
    assert int(s.len.sum()) > 8


def test_step_captured(own_ctx):
    """The whole step in a graph, replayed with eager steps between: other rows, trees, lengths and prefix lengths each time. A
    graph of another size shares the context's scratch."""
    import torch
    from helpers import HipGraph
    ctx, rng = own_ctx, np.random.default_rng(22)
    loops = [_loop(ctx, rng), _loop(ctx, rng, B=40, N=1, H=8, K=2, D=128, V=33000, plens=(400,), first=(0, 39))]
    graphs = []
    for s in loops:
        s.fill(rng, 0)
        s.run(ctx)
    for s in loops:
        g, q = HipGraph(ctx.stream), torch.zeros(s.B, s.N, s.H, s.D, device="cuda")
        torch.cuda.synchronize()
        g.begin()
        s.attend(ctx, q, sync=False)
        s.choose(ctx, sync=False)
        g.end()
        graphs.append((g, q))
    for rep in range(1, 4):
        for s, (g, q) in zip(loops, graphs):
            s.fill(rng, rep)
            s.len.copy_(_i(rng.integers(0, s.cap - s.N + 1, s.B)))
            torch.cuda.synchronize()
            st = s.state()
            s.run(ctx)
            torch.cuda.synchronize()
            q.copy_(s.x[:, :, :s.H])
            eager = s.state()
            s.put(st)  # (the logits stay: their product is the library's and not in the graph)
            torch.cuda.synchronize()
            g.launch()
            ctx.sync()
            assert all(torch.equal(a, b) for a, b in zip(s.state(), eager)), rep


# ---- attention: longer prefixes, more of them, and the calls that equal others -------------------------------------
LONG = [
    # kind, heads, kv, hd, B, N, prefix lengths, first: several pieces, row tiles and stages
    ("bf16", 32, 2, 256, 9, 1, [1700], [0, 9]),
    ("i8", 32, 2, 256, 9, 1, [1700], [0, 9]),
    ("f32", 32, 2, 256, 9, 1, [1700], [0, 9]),
    ("bf16", 32, 2, 128, 20, 3, [900, 1333], [0, 13, 20]),
    ("i8", 32, 2, 128, 20, 3, [900, 1333], [0, 13, 20]),
    ("f32", 32, 2, 128, 20, 3, [900, 1333], [0, 13, 20]),
    ("i8", 24, 1, 192, 6, 2, [1025], [0, 6]),
    ("bf16", 24, 1, 192, 6, 2, [1025], [0, 6]),
    ("f32", 8, 1, 64, 40, 1, [2000], [1, 39]),
    ("i8", 8, 1, 64, 40, 1, [2000], [1, 39]),
    ("bf16", 8, 8, 64, 90, 1, [3 * g for g in range(90)], list(range(91))),  # a prefix for each
    ("i8", 8, 4, 64, 90, 1, [3 * g for g in range(90)], list(range(91))),
    ("i8", 40, 1, 256, 2, 1, [300], [0, 2]),   # 40 query heads of a KV head: three row tiles of a sequence alone
    ("bf16", 40, 1, 128, 2, 4, [300], [0, 2]),
]


@pytest.mark.parametrize("kind,H,K,D,B,N,plens,first", LONG)
@pytest.mark.parametrize("hint", [False, True])
def test_attend_long(ctx, kind, H, K, D, B, N, plens, first, hint):
    """hint: lengths past max_len and max_prefix, which only choose the split."""
    import torch
    rng = np.random.default_rng(H * D + B)
    G, pcap, cap = len(plens), max(plens) + 5, 150
    kc, vc, kd, vd = [_kv(rng, kind, B, n, K, D) for n in (cap, cap, N, N)]
    kp, vp = _kv(rng, kind, G, pcap, K, D), _kv(rng, kind, G, pcap, K, D)
    q = rng.standard_normal((B, N, H, D)).astype(np.float32)
    lens, counts = rng.integers(0, cap + 1, B).tolist(), rng.integers(0, N + 1, B).tolist()
    lens[0], counts[0] = cap, N
    par = T.random_parents(rng, B, N, "tree")
    out, scale = torch.full((B, N, H, D), 3.0, device="cuda"), D ** -0.5
    ctx.gqa_prefix(_t(q), _both(kc, vc), _i(lens), _i(counts), scale, out, draft=_both(kd, vd), parent=_i(par), prefix=_both(kp, vp),
                   prefix_len=_i(plens), prefix_first=_i(first), max_len=7 if hint else 0, max_prefix=60 if hint else 0)
    want, mag, qk, keys = BT.prefix_attention(q, kc[1], vc[1], kd[1], vd[1], lens, counts, par, scale, kp[1], vp[1], plens, first,
                                              out=np.full(q.shape, 3.0))
    tol = T.tree_attention_bound(mag, qk, keys[:, None, None, None], D)
    if kind == "i8":
        tol = tol + BT.bound8(q, max(np.abs(x[1]).max() for x in (kc, kd, kp)), max(np.abs(x[1]).max() for x in (vc, vd, vp)), scale, keys)
    live = np.arange(N)[None] < np.array(counts)[:, None]
    got = _np(out)
    assert (got[~live] == 3.0).all()
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol)[live].all(), (err[live].max(), (err / tol)[live].max())
    assert np.linalg.norm(err[live]) <= 4e-6 * np.linalg.norm(want[live])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D,H,K,N", [(64, 8, 2, 1), (128, 20, 4, 5), (256, 64, 4, 1), (80, 6, 2, 3)])
def test_attend_without_prefixes_is_the_tree_call(ctx, kind, D, H, K, N):
    """No prefixes, rows of the nodes beside the cache: the bits of rbt_gqa_tree_d."""
    import torch
    rng = np.random.default_rng(D)
    B, cap = 3, 500
    kc, vc, kd, vd = [_kv(rng, kind, B, n, K, D)[0][0] for n in (cap, cap, N, N)]
    q, par = _t(rng.standard_normal((B, N, H, D)).astype(np.float32)), _i(T.random_parents(rng, B, N, "tree"))
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    ctx.gqa_tree(q, kc, vc, kd, vd, _i([500, 0, 77]), _i([N, N, 1]), par, 0.1, a)
    ctx.gqa_prefix(q, (kc, vc), _i([500, 0, 77]), _i([N, N, 1]), 0.1, b, draft=(kd, vd), parent=par)
    assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 256, 80])
def test_attend_8bit_scores(ctx, D):
    """Queries of zeros, of NaN and huge ones, attn_scale 0 and below 0, rows of scale 0: what the definition gives."""
    import torch
    rng = np.random.default_rng(31)
    B, H, K, cap = 4, 8, 2, 200
    kc, vc = _kv(rng, "i8", B, cap, K, D), _kv(rng, "i8", B, cap, K, D)
    kp, vp = _kv(rng, "i8", 1, 300, K, D), _kv(rng, "i8", 1, 300, K, D)
    q = rng.standard_normal((B, 1, H, D)).astype(np.float32)
    q[0] = 0.0
    q[1, 0, 3, 5] = np.nan
    q[2] *= np.float32(1e30)
    lens, plens, first = [150, 0, 199, 30], [280], [0, 4]

    def run(scale, qq=q, kt=kc):
        out = torch.full((B, 1, H, D), 3.0, device="cuda")
        ctx.gqa_prefix(_t(qq), _both(kt, vc), _i(lens), _i([1] * B), scale, out, prefix=_both(kp, vp), prefix_len=_i(plens),
                       prefix_first=_i(first))
        return _np(out).astype(np.float64)

    def want(scale, qq=q):
        w, mag, qk, keys = BT.prefix_attention(np.nan_to_num(qq), kc[1], vc[1], None, None, lens, [1] * B, np.full((B, 1), -1), scale,
                                               kp[1], vp[1], plens, first)
        tol = T.tree_attention_bound(mag, qk, keys[:, None, None, None], D) + BT.bound8(
            np.nan_to_num(qq), max(np.abs(x[1]).max() for x in (kc, kp)), max(np.abs(x[1]).max() for x in (vc, vp)), scale, keys)
        return w, tol

    for scale in (0.1, -0.1, 0.0):
        got = run(scale)
        w, tol = want(scale)
        ok = [0, 3] + ([2] if scale == 0 else [])
        assert (np.abs(got - w) <= tol)[ok].all()
        assert np.isnan(got[1, 0, 3]).all()
        others = [h for h in range(H) if h != 3]
        assert (np.abs(got[1, 0, others] - w[1, 0, others]) <= tol[1, 0, others]).all()
        if scale:  # one key stands: scores lie 1e28 and more apart, and its value is what comes out
            # the weight 1 times the row's scale to 2^-22 in digits, a product, a quotient and a sum in fp32
            assert np.abs(got[2] - w[2]).max() <= (2.0 ** -22 + 4 * T.U32) * max(np.abs(x[1]).max() for x in (vc, vp))


def test_two_contexts_at_once(own_ctx):
    """Two contexts at once from two threads, each with scratch of its own: both give what one alone does."""
    import threading
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(41)
    kind, B, H, K, D = "i8", 6, 16, 2, 128
    rows = [_both(_kv(rng, kind, n, c, K, D), _kv(rng, kind, n, c, K, D)) for n, c in ((B, 64), (1, 700))]
    q, x = _t(rng.standard_normal((B, 1, H, D)).astype(np.float32)), _t(rng.standard_normal((B, 50000)).astype(np.float32) * 3)
    u = _t(rng.random(B, dtype=np.float32))

    def step(c, out, tok):
        c.gqa_prefix(q, rows[0], _i([40] * B), _i([1] * B), 0.1, out, prefix=rows[1], prefix_len=_i([699]), prefix_first=_i([0, B]))
        c.sample(x, u, tok, top_p=_t(np.full(B, 0.9, np.float32)))
    res = [(torch.zeros_like(q), torch.zeros(B, dtype=torch.int32, device="cuda")) for _ in range(3)]
    step(own_ctx, *res[0])
    other = R.Context(0)

    def many(c, r):
        for _ in range(20):
            step(c, *r)
    ts = [threading.Thread(target=many, args=a) for a in ((own_ctx, res[1]), (other, res[2]))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    other.close()
    for out, tok in res[1:]:
        assert torch.equal(out, res[0][0]) and torch.equal(tok, res[0][1])


# ---- sampling: long rows ---------------------------------------------------------------------------------------
SETS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.01), (0.0, 0, 1.0, 0.0),
        (1.0, 1, 1.0, 0.0), (3.0, 700, 0.5, 0.0), (0.05, 30, 0.99, 0.0), (1.0, 20000, 0.999, 0.0), (1.0, 513, 1.0, 0.0),
        (1.0, 0, 0.0, 0.0), (2.0, 0, 0.7, 1e-3), (1.0, 512, 1.0, 0.0), (1.0, 0, 1.0, 1.0)]


@pytest.mark.parametrize("V,stride", [(32769, 0), (100003, 100003), (131072, 131081), (70000, 70001)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sample_long(ctx, V, stride, dtype):
    rng = np.random.default_rng(V)
    n = len(SETS)
    x = (2.5 * rng.standard_normal((n, V))).astype(np.float32)
    x[:, rng.integers(0, V, 3)] += 8
    x[3, rng.integers(0, V, 1000)] = np.nan
    x[4, V // 2:] = -np.inf
    t, k, p, m = zip(*SETS)
    _sample_check(ctx, x, rng.random(n), dtype, t, k, p, m, stride=stride or None)


@pytest.mark.parametrize("V", [9000, 40001, 131072])
def test_sample_long_ties(ctx, V):
    """Thousands of equal logits at every border: the lowest indices stand."""
    low = float(np.finfo(np.float32).min)
    x = np.full((5, V), low, np.float32)
    x[0] = 0.25
    x[1, V // 3:] = 1.5                   # a long tail of the lowest value
    x[2, ::2], x[2, 1::2] = 0.0, -0.0
    x[3, 1::3] = -7.0                     # the largest, thousands of times
    x[4] = -np.inf
    x[4, V - 5000:] = 2.0
    u = [0.31, 0.77, 0.5003, 0.61, 0.99]
    for k, p, m in ((0, 1.0, 0.0), (10, 1.0, 0.0), (0, 0.3331, 0.0), (2500, 0.5003, 0.0), (700, 1.0, 0.5), (0, 0.77, 1.0)):
        _sample_check(ctx, x, u, t=[0.9] * 5, k=[k] * 5, p=[p] * 5, m=[m] * 5)


@pytest.mark.parametrize("V,n", [(33000, 300), (2500, 700)])
def test_sample_many_rows(ctx, V, n):
    """More rows than the chip takes at once give what a few of them do, bit for bit."""
    import torch
    rng = np.random.default_rng(n)
    x = _t((3 * rng.standard_normal((n, V))).astype(np.float32))
    sets = [SETS[i % len(SETS)] for i in range(n)]
    t, k, p, m = [np.array(a) for a in zip(*sets)]
    f = lambda a: _t(np.asarray(a, np.float32))  # noqa: E731
    u = f(rng.integers(0, 2 ** 24, n) / 2.0 ** 24)

    def run(lo, hi):
        tok, pr = torch.full((hi - lo,), -9, dtype=torch.int32, device="cuda"), torch.zeros(hi - lo, V, device="cuda")
        ctx.sample(x[lo:hi], u[lo:hi], tok, f(t[lo:hi]), _i(k[lo:hi]), f(p[lo:hi]), f(m[lo:hi]), probs=pr)
        return tok, pr
    tok, pr = run(0, n)
    for lo, hi in ((0, 1), (1, 20), (20, 33), (n - 7, n)):
        a, b = run(lo, hi)
        assert torch.equal(a, tok[lo:hi]) and torch.equal(b, pr[lo:hi])
    for r in range(0, n, 29):
        one = lambda a: float(np.float32(a[r]))  # noqa: E731
        want, wp, near = BT.sample(_np(x)[r], float(u[r]), one(t), int(k[r]), one(p), one(m))
        off = V * 2.0 ** -46 + 2.0 ** -48
        assert near > 2 * off and int(tok[r]) == want
        assert (np.abs(_np(pr)[r] - wp) <= (T.U32 + 2 * off) * wp + 1e-45).all()


@pytest.mark.parametrize("V,n,probs", [(500, 3, True), (60000, 4, True), (131072, 2, False)])
def test_sample_captured(own_ctx, V, n, probs):
    """Replays over new logits and settings, with eager calls of other sizes between them, equal the eager call; bad settings are
    reported by the sync after their replay alone."""
    import torch
    from helpers import HipGraph
    ctx, rng = own_ctx, np.random.default_rng(V)
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    x, u, t, p, m, k = z(n, V), z(n), z(n), z(n), z(n), _i([0] * n)
    tok, pr = torch.zeros(n, dtype=torch.int32, device="cuda"), z(n, V) if probs else None
    other = _t(rng.standard_normal((7, 90000)).astype(np.float32))
    call = lambda tk, q, sync=True: ctx.sample(x, u, tk, t, k, p, m, probs=q, sync=sync)  # noqa: E731

    def fill(rep):
        x.copy_(_t((3 * rng.standard_normal((n, V))).astype(np.float32)))
        u.copy_(_t((rng.integers(0, 2 ** 24, n) / 2.0 ** 24).astype(np.float32)))
        for b, col in zip((t, k, p, m), zip(*[SETS[(rep * n + i) % len(SETS)] for i in range(n)])):
            b.copy_(_t(np.asarray(col, np.float32)) if b is not k else _i(col))
    fill(0)
    call(tok, pr)
    ctx.sample(other, z(7), torch.zeros(7, dtype=torch.int32, device="cuda"))
    g = HipGraph(ctx.stream)
    torch.cuda.synchronize()
    g.begin()
    call(tok, pr, sync=False)
    g.end()
    for rep in range(1, 6):
        fill(rep)
        if rep == 3:
            t[0] = -1.0
        torch.cuda.synchronize()
        g.launch()
        if rep == 3:
            _reported(ctx)
        else:
            ctx.sync()
        ctx.sample(other, z(7), torch.zeros(7, dtype=torch.int32, device="cuda"))
        w, wp = torch.zeros_like(tok), z(n, V) if probs else None
        call(w, wp, sync=False)
        if rep == 3:
            _reported(ctx)
            assert int(tok[0]) == -1
        else:
            ctx.sync()
        assert torch.equal(tok, w) and (pr is None or torch.equal(pr, wp)), rep


def test_sample_odd_addresses(ctx):
    """Rows that begin at any entry: views one to seven entries into a buffer, probabilities at any f32."""
    import torch
    rng = np.random.default_rng(51)
    for V in (1003, 40003):
        for off in (1, 2, 3, 5, 7):
            for dt in ("float32", "bfloat16"):
                base = _t((2 * rng.standard_normal(off + 3 * (V + 1))).astype(np.float32), _dt(dt))
                x = base[off:].view(3, V + 1)[:, :V]
                pr = torch.zeros(off + 3 * V, device="cuda")[off:].view(3, V)
                tok = torch.zeros(3, dtype=torch.int32, device="cuda")
                u = _t(rng.random(3, dtype=np.float32))
                ctx.sample(x, u, tok, top_p=_t(np.full(3, 0.9, np.float32)), probs=pr)
                y, tk, py = x.contiguous(), torch.zeros_like(tok), torch.zeros(3, V, device="cuda")
                ctx.sample(y, u, tk, top_p=_t(np.full(3, 0.9, np.float32)), probs=py)
                assert torch.equal(tok, tk) and torch.equal(pr, py)


def test_empty_batches(ctx):
    import torch
    e = lambda *s, dt="float32": torch.zeros(*s, dtype=_dt(dt), device="cuda")  # noqa: E731
    c8 = (e(0, 5, 2, 64, dt="int8"), e(0, 5, 2, 64, dt="int8"), e(0, 5, 2), e(0, 5, 2))
    ctx.kv_quant(e(0, 1, 2, 64), e(0, 1, 2, 64), c8)
    ctx.gqa_prefix(e(0, 1, 4, 64), c8, e(0, dt="int32"), e(0, dt="int32"), 0.1, e(0, 1, 4, 64))
    ctx.sample(e(0, 50), e(0), e(0, dt="int32"))
