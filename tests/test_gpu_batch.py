"""GPU checks of the batch step's operators (rbt_kv_quant_d, rbt_kv_dequant_d, rbt_gqa_prefix_d, rbt_sample_d) against
their 64-bit forms (batch_truth.py), each by the bound derived there, and of a decode step made of them."""
import numpy as np
import pytest

import batch_truth as BT
import draft_truth as T
from test_gpu_drafts import _bf, _i, _np, _t

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return getattr(torch, name)


def _reported(ctx):
    """The next rbt_sync reports numbers that did not fit; the one after it is clean."""
    import rabbit_amd as R
    with pytest.raises(R.RbtError) as e:
        ctx.sync()
    assert e.value.status == R.abi.RBT_E_INVALID and "batch step" in str(e.value)
    ctx.sync()


# ---- 8-bit rows ------------------------------------------------------------------------------------
def _cache8(B, cap, K, D):
    import torch
    return (torch.full((B, cap, K, D), 99, dtype=torch.int8, device="cuda"), torch.full((B, cap, K, D), 98, dtype=torch.int8, device="cuda"),
            torch.full((B, cap, K), 9.0, device="cuda"), torch.full((B, cap, K), 8.0, device="cuda"))


@pytest.mark.parametrize("B,Tn,K,D,cap,dtype,wide,counts,lens", [
    (1, 1, 4, 256, 8, "float32", False, None, [3]),              # the new token of one user
    (1, 1, 4, 256, 1, "bfloat16", False, None, None),            # a cache of one row
    (3, 5, 4, 256, 11, "bfloat16", True, [5, 0, 2], [6, 11, 0]),  # views of q, k, v rows, an empty sequence, full ones
    (2, 70, 2, 64, 70, "float32", True, [70, 69], [0, 1]),
    (2, 3, 1, 33, 5, "float32", False, [3, 1], [2, 4]),          # odd heads: entry by entry
    (2, 3, 3, 80, 5, "bfloat16", True, [3, 1], [0, 0]),
    (1, 4, 2, 7, 6, "bfloat16", False, None, [2]),
    (1, 2, 1, 1, 2, "float32", False, None, None),               # one entry: +-127 or 0
    (1, 2, 2, 512, 3, "float32", False, None, [1]),
    (1, 2, 2, 520, 3, "bfloat16", False, None, [1]),             # past the lanes' eights
    (1, 3, 1, 1024, 3, "float32", False, None, None),
    (5, 33, 8, 128, 64, "bfloat16", False, [33, 32, 1, 0, 17], [31, 0, 63, 64, 20]),
])
def test_quant(ctx, B, Tn, K, D, cap, dtype, wide, counts, lens):
    """Entries and scales are those of the definition, bit for bit; no other row is touched; and the rows read back."""
    import torch
    rng = np.random.default_rng(B * 1000 + Tn + D)
    x = (rng.standard_normal((B, Tn, (6 if wide else 2) * K, D)) * np.exp(3 * rng.standard_normal((B, Tn, 1, 1)))).astype(np.float32)
    if D > 1:
        x[0, 0, -1] = 0.0                     # a row of zeros
        x[0, -1, -1, 0] = 3e38
        x[-1, -1, -2 * K] *= np.float32(1e-42)  # subnormal scales
    src = _t(x, _dt(dtype))
    kk, vv = src[:, :, -2 * K:-K], src[:, :, -K:]
    n = counts or [Tn] * B
    at = lens or [0] * B
    cache = _cache8(B, cap, K, D)
    ctx.kv_quant(kk, vv, cache, length=None if lens is None else _i(lens), n_rows=None if counts is None else _i(counts))
    got = [_np(t) for t in cache]
    out = [torch.full((B, Tn, K, D), 5.0, dtype=_dt(d), device="cuda") for d in ("float32", "bfloat16") for _ in "kv"]
    ctx.kv_dequant(cache, out[0], out[1], length=None if lens is None else _i(lens), n_rows=None if counts is None else _i(counts))
    ctx.kv_dequant(cache, out[2], out[3], length=None if lens is None else _i(lens), n_rows=None if counts is None else _i(counts))
    for side, rows in enumerate((kk, vv)):
        q, s = BT.quantise(_np(rows))
        wq, ws = np.full((B, cap, K, D), 99 - side, np.int8), np.full((B, cap, K), 9.0 - side, np.float32)
        for b in range(B):
            wq[b, at[b]:at[b] + n[b]], ws[b, at[b]:at[b] + n[b]] = q[b, :n[b]], s[b, :n[b]]
        assert np.array_equal(got[2 + side], ws) and np.array_equal(got[side], wq)
        want = BT.values(q, s, np.float32)
        for d, o in (("float32", out[side]), ("bfloat16", out[2 + side])):
            w = want if d == "float32" else _bf(want)
            for b in range(B):
                assert np.array_equal(_np(o)[b, :n[b]], w[b, :n[b]]) and (_np(o)[b, n[b]:] == 5.0).all()


def test_quant_halves(ctx):
    """Quotients at halves and one step beside them, scales on both sides of every rule, bit for bit."""
    rng = np.random.default_rng(11)
    R, K, D = 290, 2, 256
    a = np.ldexp(1 + rng.random((1, R, K, 1)), (np.arange(R) - 145).reshape(1, R, 1, 1) * 4 // 5).astype(np.float32)
    x = (a / np.float32(127)).astype(np.float64) * (rng.integers(-127, 127, (1, R, K, D)) + 0.5)
    x = x.astype(np.float32)
    x[..., 1::3] = np.nextafter(x[..., 1::3], np.float32(np.inf))
    x[..., 2::3] = np.nextafter(x[..., 2::3], np.float32(-np.inf))
    x = np.clip(x, -a, a)
    x[..., :1] = a
    cache = _cache8(1, R, K, D)
    ctx.kv_quant(_t(x), _t(-x), cache)
    q, s = BT.quantise(x)
    assert np.array_equal(_np(cache[0]), q) and np.array_equal(_np(cache[2]), s)
    assert np.array_equal(_np(cache[1]), -q) and np.array_equal(_np(cache[3]), s)


def test_quant_special_values(ctx):
    """A row with a non-finite entry reads back as NaN, whole; its neighbours do not notice."""
    import torch
    rng = np.random.default_rng(5)
    for D in (64, 33):
        x = rng.standard_normal((1, 4, 3, D)).astype(np.float32)
        x[0, 0, 1, 5], x[0, 2, 0, D - 1], x[0, 3, 2, 0] = np.nan, np.inf, -np.inf
        cache = _cache8(1, 4, 3, D)
        ctx.kv_quant(_t(x), _t(-x), cache)
        k, v = torch.zeros(1, 4, 3, D, device="cuda"), torch.zeros(1, 4, 3, D, device="cuda")
        ctx.kv_dequant(cache, k, v)
        bad = ~np.isfinite(x).all(-1)
        q, s = BT.quantise(x)
        assert np.array_equal(_np(cache[0]), q) and np.array_equal(_np(cache[2]), s, equal_nan=True)
        assert np.isnan(_np(k)[bad]).all() and np.isfinite(_np(k)[~bad]).all()
        assert np.array_equal(_np(v), -_np(k), equal_nan=True)


def test_quant_strided_results_and_bad_sequences(ctx):
    """Results into a view whose heads lie apart; sequences that do not fit are left alone and reported."""
    import torch
    rng = np.random.default_rng(6)
    B, Tn, K, D, cap = 4, 3, 2, 64, 8
    x = _t(rng.standard_normal((B, Tn, K, D)).astype(np.float32))
    lens, counts = [6, 0, -1, 5], [3, 4, 1, 3]  # past the cap; more than max_rows; negative; fits
    cache = _cache8(B, cap, K, D)
    ctx.kv_quant(x, x, cache, length=_i(lens), n_rows=_i(counts), sync=False)
    _reported(ctx)
    q, s = BT.quantise(_np(x))
    got = _np(cache[0])
    assert (got[:3] == 99).all() and np.array_equal(got[3, 5:], q[3]) and (got[3, :5] == 99).all()
    both = torch.full((K, 2, B, Tn, D), 5.0, device="cuda")
    k, v = [both[:, i].permute(1, 2, 0, 3) for i in (0, 1)]
    ctx.kv_dequant(cache, k, v, length=_i(lens), n_rows=_i(counts), sync=False)
    _reported(ctx)
    assert (_np(k)[:3] == 5.0).all() and np.array_equal(_np(k)[3], BT.values(q, s, np.float32)[3])
    assert np.array_equal(_np(v), _np(k))


def test_quant_captured(ctx):
    """A captured write follows the lengths, and equals the eager one at every replay."""
    import torch
    rng = np.random.default_rng(7)
    B, K, D, cap = 3, 4, 128, 9
    x, ln = _t(rng.standard_normal((B, 1, K, D)).astype(np.float32)), _i([0, 3, 5])
    cache, want = _cache8(B, cap, K, D), _cache8(B, cap, K, D)
    stream = ctx.torch_stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        ctx.kv_quant(x, x, cache, length=ln, sync=False)
    for step in range(3):
        new = rng.standard_normal((B, 1, K, D)).astype(np.float32)
        x.copy_(_t(new))
        ln.copy_(_i([step, 3 + step, 5 + step]))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ctx.kv_quant(x, x, want, length=ln)
        assert all(torch.equal(a, b) for a, b in zip(cache, want))


def test_commit_moves_8bit_rows(ctx):
    """rbt_kv_commit_d over int8 rows of odd sizes, and their scales as rows of head_dim 1."""
    import torch
    rng = np.random.default_rng(8)
    for K, D in ((2, 64), (1, 33), (3, 7)):
        B, N, cap = 2, 4, 9
        caches = [torch.zeros((B, cap, K, D), dtype=torch.int8, device="cuda") for _ in "kv"]
        drafts = [_t(rng.integers(-127, 128, (B, N, K, D)).astype(np.int8)) for _ in "kv"]
        sc = [torch.zeros(B, cap, K, device="cuda") for _ in "kv"]
        sd = [_t(rng.random((B, N, K)).astype(np.float32)) for _ in "kv"]
        path, m, ln, lo = _i([[0, 2, 3, -1], [0, -1, -1, -1]]), _i([3, 1]), _i([4, 8]), _i([0, 0])
        ctx.kv_commit([caches[0]], [caches[1]], [drafts[0]], [drafts[1]], path, m, ln, lo)
        ctx.kv_commit([sc[0][..., None]], [sc[1][..., None]], [sd[0][..., None]], [sd[1][..., None]], path, m, ln, lo)
        for c, d in zip(caches + sc, drafts + sd):
            want = np.zeros_like(_np(c))
            want[0, 4:7], want[1, 8] = _np(d)[0, [0, 2, 3]], _np(d)[1, 0]
            assert np.array_equal(_np(c), want)
        assert _np(lo).tolist() == [7, 9]


# ---- attention over shared prefixes ------------------------------------------------------------------
def _kv(rng, kind, *shape):
    """Rows of a cache as (tensors, the values they stand for)."""
    x = rng.standard_normal(shape).astype(np.float32)
    if kind == "i8":
        q, s = BT.quantise(x)
        return (_t(q), _t(s)), BT.values(q, s)
    if kind == "bf16":
        return (_t(x, _dt("bfloat16")),), _bf(x)
    return (_t(x),), x


def _both(k, v):
    """(k, v[, k_scale, v_scale]) tensors of two sides."""
    return tuple(t for pair in zip(k[0], v[0]) for t in pair)


ATTEND = [
    # kind, heads, kv, hd, B, N, prefix lengths, first, own lens, counts, kind of tree, gate, draft
    ("bf16", 64, 4, 256, 3, 1, [130], [0, 3], [5, 0, 70], [1, 1, 1], "chain", True, True),
    ("i8", 64, 4, 256, 3, 1, [130], [0, 3], [5, 0, 70], [1, 1, 1], "chain", True, True),
    ("f32", 64, 4, 256, 3, 1, [130], [0, 3], [5, 0, 70], [1, 1, 1], "chain", True, True),
    ("i8", 64, 4, 256, 2, 1, [], [0], [300, 1], [1, 1], "chain", True, False),       # no prefix, rows in the cache
    ("bf16", 20, 4, 128, 5, 3, [65, 1, 0], [0, 2, 3, 4], [9, 0, 64, 3, 2], [3, 1, 2, 3, 0], "tree", False, True),
    ("i8", 20, 4, 128, 5, 3, [65, 1, 0], [0, 2, 3, 4], [9, 0, 64, 3, 2], [3, 1, 2, 3, 0], "tree", False, True),
    ("f32", 20, 4, 128, 5, 3, [65, 1, 0], [0, 2, 3, 4], [9, 0, 64, 3, 2], [3, 1, 2, 3, 0], "tree", False, True),
    ("i8", 12, 12, 64, 4, 2, [200, 77], [1, 2, 4], [0, 33, 128, 129], [2, 2, 1, 2], "chain", True, False),
    ("bf16", 16, 2, 64, 33, 1, [257], [0, 33], [1] * 33, [1] * 33, "chain", False, True),
    ("i8", 16, 2, 64, 33, 1, [257], [0, 33], [1] * 33, [1] * 33, "chain", False, True),
    ("i8", 48, 3, 192, 6, 4, [140, 33], [0, 5, 6], [3, 2, 1, 0, 65, 66], [4, 4, 4, 4, 4, 4], "tree", True, True),
    ("f32", 48, 3, 192, 6, 4, [140, 33], [0, 5, 6], [3, 2, 1, 0, 65, 66], [4, 4, 4, 4, 4, 4], "tree", True, True),
    ("bf16", 6, 2, 80, 3, 5, [50], [0, 2], [4, 20, 7], [5, 2, 1], "tree", True, True),  # head dims off the matrix cores
    ("i8", 6, 2, 80, 3, 5, [50], [0, 2], [4, 20, 7], [5, 2, 1], "tree", True, False),
    ("f32", 3, 3, 33, 2, 2, [9, 8], [0, 0, 2], [1, 0], [2, 1], "chain", False, False),   # an empty group
    ("i8", 4, 1, 512, 2, 1, [40], [0, 2], [3, 4], [1, 1], "chain", False, True),
]


@pytest.mark.parametrize("kind,H,K,D,B,N,plens,first,lens,counts,tree,gated,drafted", ATTEND)
def test_attend(ctx, kind, H, K, D, B, N, plens, first, lens, counts, tree, gated, drafted):
    import torch
    rng = np.random.default_rng(H + D + B + N)
    cap, G, pcap = max(lens) + N + 1, len(plens), max(plens + [0]) + 3
    kc, vc = _kv(rng, kind, B, cap, K, D), _kv(rng, kind, B, cap, K, D)
    kd, vd = _kv(rng, kind, B, N, K, D), _kv(rng, kind, B, N, K, D)
    kp, vp = (_kv(rng, kind, G, pcap, K, D), _kv(rng, kind, G, pcap, K, D)) if G else ((None, None), (None, None))
    q = rng.standard_normal((B, N, H, D)).astype(np.float32)
    gate = rng.standard_normal((B, N, H, D)).astype(np.float32) if gated else None
    par = T.random_parents(rng, B, N, tree)
    out = torch.full((B, N, H, D), 3.0, device="cuda")
    scale = D ** -0.5
    ctx.gqa_prefix(_t(q), _both(kc, vc), _i(lens), _i(counts), scale, out, draft=_both(kd, vd) if drafted else None,
                   parent=None if tree == "chain" else _i(par), prefix=_both(kp, vp) if G else None,
                   prefix_len=_i(plens) if G else None, prefix_first=_i(first) if G else None,
                   gate=None if gate is None else _t(gate))
    want, mag, qk, keys = BT.prefix_attention(q, kc[1], vc[1], kd[1] if drafted else None, vd[1] if drafted else None, lens,
                                              counts, par, scale, kp[1], vp[1], plens, first, gate=gate,
                                              out=np.full(q.shape, 3.0))
    tol = T.tree_attention_bound(mag, qk, keys[:, None, None, None], D)
    if kind == "i8":
        top = lambda *xs: max(np.abs(x).max() for x in xs if x is not None)  # noqa: E731
        tol = tol + BT.bound8(q, top(kc[1], kd[1], kp[1]), top(vc[1], vd[1], vp[1]), scale, keys, gate)
    live = np.arange(N)[None] < np.array(counts)[:, None]
    got = _np(out)
    assert (got[~live] == 3.0).all()
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol)[live].all(), (err[live].max(), (err / tol)[live].max())
    # As a whole: a query's entry is off by 2^-23 / sqrt 3 of the row's largest (at most 5 of its rms) as rounding errors
    # are, a score by that times |k| scale (near 1 here), 3.5e-7; a weight by sqrt 2 of it, probabilities and fp32 sums by
    # no more: under 1e-6 of the output, times 4
    assert np.linalg.norm(err[live]) <= 4e-6 * np.linalg.norm(want[live])


def _small(rng, kind="bf16", B=4, N=1, K=2, H=8, D=64, cap=40, G=2, pcap=70):
    q = _t(rng.standard_normal((B, N, H, D)).astype(np.float32))
    rows = [_both(_kv(rng, kind, n, c, K, D), _kv(rng, kind, n, c, K, D)) for n, c in ((B, cap), (B, N), (G, pcap))]
    return q, rows


@pytest.mark.parametrize("kind", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("D", [64, 80])
def test_attend_bad_numbers(ctx, kind, D):
    """Lengths, counts, prefixes and parents outside their ranges: the sequences concerned are left as they were and
    reported; nothing else changes."""
    import torch
    rng = np.random.default_rng(9)
    q, (cache, draft, prefix) = _small(rng, kind, D=D)
    call = lambda lens, counts, plens, first, **kw: ctx.gqa_prefix(  # noqa: E731
        q, cache, _i(lens), _i(counts), 0.125, kw["out"], draft=kw.get("draft", draft), prefix=prefix, prefix_len=_i(plens),
        prefix_first=_i(first), parent=kw.get("parent"), sync=False)
    good = torch.full_like(q, 3.0)
    call([5, 6, 7, 8], [1, 1, 1, 1], [70, 30], [0, 2, 3], out=good)
    ctx.sync()
    for lens, counts, plens, first, skipped, kw in [
            ([41, 6, 7, 8], [1, 1, 1, 1], [70, 30], [0, 2, 3], [0], {}), ([5, -1, 7, 8], [1, 1, 1, 1], [70, 30], [0, 2, 3], [1], {}),
            ([5, 6, 7, 8], [1, 1, 2, -1], [70, 30], [0, 2, 3], [2, 3], {}), ([5, 6, 7, 8], [1, 1, 1, 1], [71, 30], [0, 2, 3], [0, 1], {}),
            ([5, 6, 7, 8], [1, 1, 1, 1], [70, -5], [0, 2, 3], [2], {}), ([5, 6, 7, 8], [1, 1, 1, 1], [70, 30], [0, 2, 5], [0, 1, 2, 3], {}),
            ([5, 6, 7, 8], [1, 1, 1, 1], [70, 30], [2, 1, 3], [0, 1, 2, 3], {}),
            ([5, 6, 7, 8], [1, 1, 1, 1], [70, 30], [-1, 2, 3], [0, 1, 2, 3], {}),
            ([5, 6, 7, 8], [1, 1, 1, 1], [70, 30], [0, 2, 3], [], dict(parent=_i([[-1], [0], [-1], [7]])))]:
        out = torch.full_like(q, 3.0)
        call(lens, counts, plens, first, out=out, **kw)
        _reported(ctx)
        keep = [b for b in range(4) if b not in skipped]
        assert (out[skipped] == 3.0).all() and torch.equal(out[keep], good[keep]), (lens, counts, plens, first)
    out = torch.full_like(q, 3.0)
    call([5, 6, 40, 39], [1, 1, 1, 1], [70, 30], [0, 2, 3], out=out, draft=None)  # the node's row is past the cache
    _reported(ctx)
    assert (out[2] == 3.0).all() and torch.isfinite(out).all() and (out[3] != 3.0).any()


@pytest.mark.parametrize("kind", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("D", [64, 256, 80])
def test_attend_what_is_not_seen(ctx, kind, D):
    """Rows past the lengths, other users' prefixes, padding nodes and nodes on other branches hold NaN or infinities: no output
    notices. A NaN value in a prefix reaches the users of that prefix alone."""
    import torch
    rng = np.random.default_rng(10)
    q, (cache, draft, prefix) = _small(rng, kind, N=3, D=D)
    par = _i([[-1, 0, 0]] * 4)
    lens, counts, plens, first = [5, 0, 33, 8], [3, 2, 3, 1], [33, 64], [0, 2, 3]
    def run(c, d, p):
        out = torch.full_like(q, 3.0)
        ctx.gqa_prefix(q, c, _i(lens), _i(counts), 0.125, out, draft=d, parent=par, prefix=p, prefix_len=_i(plens), prefix_first=_i(first))
        return out
    good = run(cache, draft, prefix)
    bad = [[t.clone() for t in r] for r in (cache, draft, prefix)]
    which = (2, 3) if kind == "i8" else (0, 1)  # 8-bit rows: their scales
    for i, val in zip(which, (float("nan"), float("inf")) if kind != "i8" else (float("nan"), float("nan"))):
        for b in range(4):
            bad[0][i][b, lens[b]:] = val
            bad[1][i][b, counts[b]:] = val
        for g in range(2):
            bad[2][i][g, plens[g]:] = val
    got = run(*bad)
    assert torch.equal(got, good)
    bad[1][which[0]][0, 2] = float("nan")  # node 2 of sequence 0: nodes 0 and 1 do not see it
    bad[1][which[1]][2, 1] = float("nan")  # node 1 of sequence 2: nodes 0 and 2
    got = run(*bad)
    assert torch.equal(got[0, :2], good[0, :2]) and torch.equal(got[2, [0, 2]], good[2, [0, 2]]) and torch.equal(got[[1, 3]], good[[1, 3]])
    assert torch.isnan(got[0, 2]).all() and torch.isnan(got[2, 1]).all()
    bad[2][which[1]][1, 63] = float("nan")  # the last row of prefix 1: sequence 2 alone
    got = run(*bad)
    assert torch.isnan(got[2]).all() and torch.equal(got[[1, 3]], good[[1, 3]]) and torch.equal(got[0, :2], good[0, :2])


# ---- sampling --------------------------------------------------------------------------------------------
def _sample_check(ctx, x, u, dtype="float32", t=None, k=None, p=None, m=None, probs=True, stride=None):
    """Tokens and probabilities against the 64-bit form. A probability is rounded once; the sum of the weights is off by
    half a unit of 2^-45 per entry, of a whole of at least 1, and an exponential by 2^-48. A row whose thresholds lie within
    that of a border has no certain answer (none does here)."""
    import torch
    n, V = x.shape
    xt = torch.zeros(n, stride or V, dtype=_dt(dtype), device="cuda")
    xt[:, :V] = _t(x, _dt(dtype))
    if stride and stride > V:
        xt[:, V:] = 1e9
    xt = xt[:, :V]
    tok = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    pr = torch.full((n, V), 7.0, device="cuda") if probs else None
    f = lambda a: None if a is None else _t(np.asarray(a, np.float32))  # noqa: E731
    ctx.sample(xt, f(u), tok, temperature=f(t), top_k=None if k is None else _i(k), top_p=f(p), min_p=f(m), probs=pr)
    got, xv = _np(tok), _np(xt)
    for r in range(n):
        one = lambda a, d: d if a is None else float(np.float32(a[r]))  # noqa: E731
        want, wp, near = BT.sample(xv[r], float(np.float32(u[r])), one(t, 1.0), 0 if k is None else k[r], one(p, 1.0), one(m, 0.0))
        off = V * 2.0 ** -46 + 2.0 ** -48
        if (x_live := xv[r][wp > 0]).size and (x_live == x_live[0]).all():
            off = 2.0 ** -50  # weights that are all 1: their sums are whole numbers, only u times the whole is rounded
        assert near > 2 * off, (r, near)
        assert got[r] == want, (r, got[r], want)
        if probs:
            g = _np(pr)[r].astype(np.float64)
            assert np.array_equal(g > 0, wp.astype(np.float32) > 0) or np.abs(g - wp)[(g > 0) != (wp.astype(np.float32) > 0)].max() < 1e-44
            assert (np.abs(g - wp) <= (T.U32 + 2 * off) * wp + 1e-45).all()
    return got


@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4097, 32000, 50257])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sample(ctx, V, dtype):
    """Rows with settings of their own: none, each filter alone, all together, greedy, high and low temperatures."""
    rng = np.random.default_rng(V)
    sets = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.01), (0.0, 0, 1.0, 0.0),
            (1.0, 1, 1.0, 0.0), (5.0, 700, 0.5, 0.0), (0.05, 30, 0.99, 0.0), (1.0, V, 0.999, 0.0), (1.0, V + 5, 1.0, 1.0), (1.0, 0, 0.0, 0.0),
            (2.0, 0, 0.7, 1e-6)]
    n = len(sets)
    x = (2.5 * rng.standard_normal((n, V))).astype(np.float32)
    x[:, rng.integers(0, V, 3)] += 8
    t, k, p, m = zip(*sets)
    u = rng.random(n)
    _sample_check(ctx, x, u, dtype, t, k, p, m, stride=V + 3 if V % 2 else None)
    _sample_check(ctx, x[:3], rng.random(3), dtype, probs=False)


def test_sample_ties_and_masks(ctx):
    """Equal logits: the lower index first, at every border; banned tokens by -inf and by the type's lowest value; one token
    left; all equal."""
    low = float(np.finfo(np.float32).min)
    V = 3001
    x = np.full((8, V), -np.inf, np.float32)
    x[0] = 0.25                                    # all equal: the first k, the first share
    x[1] = np.repeat(np.arange(V // 3 + 1), 3)[:V] % 7
    x[2, 17] = -3.0                                # one token
    x[3, [5, 9, 2000]] = [1.0, 1.0, 1.0]
    x[4] = low
    x[4, 100:110] = 2.0
    x[5] = 0.0
    x[6, ::2], x[6, 1::2] = 0.0, -0.0              # zeros of both signs are equal
    x[7] = low
    u = [0.31, 0.77, 0.5, 0.61, 0.99, 0.123, 0.9999, 0.001]
    for k, p in ((0, 1.0), (10, 1.0), (0, 0.3331), (700, 0.5003), (2, 0.9)):
        got = _sample_check(ctx, x, u, t=[0.9] * 8, k=[k] * 8, p=[p] * 8)
        assert got[2] == 17 and got[3] in (5, 9, 2000)
    g = _sample_check(ctx, x, u, t=[0.0] * 8)
    assert g.tolist() == [0, int(np.argmax(x[1])), 17, 5, 100, 0, 0, 0]


def test_sample_borders(ctx):
    """u at 0 and at the largest number below 1: the first and the last token with any probability."""
    x = np.array([[-np.inf, 2.0, 1.0, -np.inf, 0.0, -np.inf]] * 2, np.float32)
    import torch
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")
    ctx.sample(_t(x), _t(np.array([0.0, 1.0 - 2.0 ** -24], np.float32)), tok)
    assert _np(tok).tolist() == [1, 4]


def test_sample_refused_rows(ctx):
    """Rows that nothing can be drawn from give -1 and zeros; settings out of range do so too and are reported."""
    import torch
    V = 130
    x = np.zeros((12, V), np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 7] = np.inf
    x[3, 5] = np.nan  # a NaN among others is passed over
    t, k, p, m, u = [1.0] * 12, [0] * 12, [1.0] * 12, [0.0] * 12, [0.5] * 12
    def run():
        tok, pr = torch.full((12,), 5, dtype=torch.int32, device="cuda"), torch.full((12, V), 7.0, device="cuda")
        f = lambda a: _t(np.asarray(a, np.float32))  # noqa: E731
        ctx.sample(_t(x), f(u), tok, temperature=f(t), top_k=_i(k), top_p=f(p), min_p=f(m), probs=pr, sync=False)
        return tok, pr
    tok, pr = run()
    ctx.sync()
    assert _np(tok)[:3].tolist() == [-1, -1, -1] and (_np(pr)[:3] == 0).all() and _np(pr)[3, 5] == 0
    assert (_np(tok)[3:] >= 0).all()
    t[4], t[5], k[6], p[7], p[8], m[9], u[10], u[11] = -1.0, np.nan, -3, 1.5, np.nan, -0.1, 1.0, np.nan
    tok, pr = run()
    _reported(ctx)
    assert (_np(tok)[4:] == -1).all() and (_np(pr)[4:] == 0).all() and _np(tok)[3] >= 0


def test_sample_draws_follow_the_probabilities(ctx):
    """Over a grid of u every token comes up in its share, to one point of the grid."""
    import torch
    rng = np.random.default_rng(3)
    n, V = 4096, 50
    row = rng.standard_normal(V).astype(np.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tok = torch.zeros(n, dtype=torch.int32, device="cuda")
    full = lambda v: _t(np.full(n, v, np.float32))  # noqa: E731
    ctx.sample(_t(np.tile(row, (n, 1))), _t(u), tok, top_p=full(0.8))
    _, p, _ = BT.sample(row, 0.5, top_p=float(np.float32(0.8)))
    assert np.abs(np.bincount(_np(tok), minlength=V) - n * p).max() <= 1.0
