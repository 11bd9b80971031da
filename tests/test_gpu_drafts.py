"""GPU checks of the drafted-token operators (rbt_rope_d, rbt_tree_positions_d, rbt_gqa_tree_d,
rbt_draft_verify_d, rbt_kv_commit_d) against their 64-bit forms (draft_truth.py), each by the bound derived
there, and of a decode step made of them against rbt_gqa_step_d."""
import numpy as np
import pytest

import draft_truth as T
from helpers import rel_l2

pytestmark = pytest.mark.gpu


def _t(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _i(a):
    return _t(np.asarray(a, np.int32))


def _bf(a):
    """numpy float32 rounded to bf16 and back."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16).float().numpy()


def _np(t):
    return t.float().cpu().numpy() if str(t.dtype) == "torch.bfloat16" else t.cpu().numpy()


# ---- rotary positions ------------------------------------------------------------------------------
def _rope_check(got, want, mag, b16, live):
    # norm: the root's and the weight's roundings, four; rotation: cos, sin, two products, one sum, and the
    # product with the factor: eight half steps of the magnitude in all; then one rounding to bf16
    tol = 8 * T.U32 * mag + (T.U16 * (np.abs(want) + 8 * T.U32 * mag) if b16 else 0.0) + 1e-38
    bad = np.abs(got.astype(np.float64) - want) > tol
    assert not bad[live].any(), (np.argwhere(bad)[:5], np.abs(got - want)[live].max())


@pytest.mark.parametrize("s,heads,kv,hd,start,rd,pairs,norm,src16,dst16", [
    (1, 64, 4, 256, 0, 64, False, True, False, True),      # Qwen 3.8's decode token
    (5, 20, 4, 128, 0, 128, False, True, False, False),
    (37, 5, 1, 192, 128, 64, True, False, False, True),    # the last third, interleaved
    (3, 3, 2, 80, 0, 40, False, True, True, True),
    (3, 3, 2, 80, 40, 40, True, True, True, False),
    (2, 2, 1, 7, 1, 6, False, True, False, True),          # odd head, odd start
    (2, 2, 1, 7, 1, 6, True, True, True, False),
    (4, 2, 1, 1024, 0, 1024, False, True, False, False),
    (4, 2, 1, 1024, 24, 1000, True, True, True, True),
    (4, 3, 2, 260, 2, 258, False, False, False, False),
    (3, 2, 2, 64, 16, 6, False, True, False, False),       # three pairs: no whole quads
    (300, 4, 2, 64, 0, 32, False, False, True, True),
    (2, 3, 1, 64, 0, 0, False, True, False, True),         # norms alone
])
def test_rope(ctx, s, heads, kv, hd, start, rd, pairs, norm, src16, dst16):
    """q, k and v in one call from strided rows, a quarter of the positions negative (their rows stay)."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(hd + rd + s)
    inv, _ = R.rope_freqs(rd, 1e4)
    pos = rng.integers(0, 1 << 20, s)
    pos[1::4] = -1
    tt, dt = (torch.bfloat16 if f else torch.float32 for f in (src16, dst16))
    x = [rng.standard_normal((s, h, 2, hd)).astype(np.float32) for h in (heads, kv, kv)]
    w = [(0.2 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2)] + [None]
    src = [_t(v, tt) for v in x]
    dst = [torch.full((s, h, hd), 7.0, dtype=dt, device="cuda") for h in (heads, kv, kv)]
    parts = [R.rope_part(a[:, :, 0], d, norm=None if ww is None else _t(ww), rotate=i < 2)
             for i, (a, d, ww) in enumerate(zip(src, dst, w))]
    keep = [_t(ww) if ww is not None else None for ww in w]  # the tensors the parts point to
    for p, k in zip(parts, keep):
        p.norm = None if k is None else k.data_ptr()
    ctx.rope(parts, _i(pos), hd, _t(inv) if rd else None, rope_dim=rd, rope_start=start,
             layout=R.ROPE_INTERLEAVED if pairs else R.ROPE_HALF, factor=1.25)
    live = pos >= 0
    for i in range(3):
        want, mag = T.rope(_np(src[i])[:, :, 0], pos, inv, 1.25, start, rd, pairs, w[i], rotate=i < 2)
        got = _np(dst[i])
        _rope_check(got, want, mag, dst16, live)
        assert (got[~live] == 7.0).all()


@pytest.mark.parametrize("hd,dtype", [(256, "float32"), (96, "bfloat16"), (33, "float32")])
def test_rope_in_place_and_far(ctx, hd, dtype):
    """In place over heads that lie [head, token], at positions up to 2^31 - 1: the angles keep 64 bits."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(hd)
    rd = hd // 4 * 2
    inv, f = R.rope_freqs(rd, 1e6, kind=R.ROPE_YARN, factor=32.0, orig_ctx=32768)
    pos = np.array([0, 1, 393215, 1 << 22, (1 << 31) - 1])
    x = _t(rng.standard_normal((6, 5, hd)).astype(np.float32), getattr(torch, dtype))
    before = _np(x).transpose(1, 0, 2)
    view = x.permute(1, 0, 2)
    ctx.rope([R.rope_part(view, view)], _i(pos), hd, _t(inv), factor=f)
    want, mag = T.rope(before, pos, inv, f, 0, rd, False)
    _rope_check(_np(x).transpose(1, 0, 2), want, mag, dtype == "bfloat16", np.ones(5, bool))


def test_rope_special_values(ctx):
    """NaN and infinities stay in their pair (without a norm) and their row (with one)."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 63] = np.nan, np.inf, -np.inf
    src, w = _t(x), _t(np.zeros(64, np.float32))
    inv = _t(R.rope_freqs(32, 1e4)[0])
    for norm in (None, w):
        out = torch.zeros_like(src)
        ctx.rope([R.rope_part(src, out, norm=norm)], _i([1, 2, 3]), 64, inv)
        finite = np.isfinite(_np(out))
        hit = np.zeros_like(finite)
        if norm is None:
            hit[0, 0, [3, 19]], hit[1, 1, 40], hit[2, 0, 63] = True, True, True
        else:
            hit[0, 0], hit[1, 1, 40], hit[2, 0, 63] = True, True, True  # inf: the others become 0
        assert np.array_equal(~finite, hit)


def test_rope_matches_the_step(ctx):
    """With angles rounded as rbt_gqa_step_d rounds them, the rotated key is the one that it pushes."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(4)
    H, K, D, rd = 8, 2, 256, 64
    inv, _ = R.rope_freqs(rd, 1e7, as_f32=True)
    kn = _t((0.1 * rng.standard_normal(D)).astype(np.float32))
    for pos in (0, 5, 30001):
        k = _t(rng.standard_normal((1, K, D)).astype(np.float32))
        out = torch.zeros_like(k)
        kc = torch.zeros(pos + 1, K, D, device="cuda")
        ctx.gqa_step(H, K, D, rd, 1e7, 0.0625, 1e-6, kn, kn, kc, torch.zeros_like(kc), pos + 1, pos,
                     torch.zeros(H, 2, D, device="cuda"), k, k, torch.zeros(H, D, device="cuda"))
        ctx.rope([R.rope_part(k, out, norm=kn)], _i([pos]), D, _t(inv), angle_f32=True)
        assert torch.allclose(out[0], kc[pos], rtol=2e-7, atol=1e-7)  # the sums of squares round apart, if at all


# ---- positions -------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,N,shape", [(1, 1, "tree"), (5, 64, "tree"), (3, 256, "chain"), (4, 255, "forest")])
def test_tree_positions(ctx, B, N, shape):
    import torch
    rng = np.random.default_rng(N)
    par, lens = T.random_parents(rng, B, N, shape), rng.integers(0, 1 << 20, B)
    n = rng.integers(0, N + 1, B)
    n[0] = N
    pos = torch.full((B, N), -7, dtype=torch.int32, device="cuda")
    ctx.tree_positions(_i(par), _i(n), _i(lens), pos)
    want = np.array([[lens[b] + len(T.ancestors(par[b], i)) - 1 if i < n[b] else -1 for i in range(N)] for b in range(B)])
    assert np.array_equal(_np(pos), want)


def test_bad_numbers_are_reported_once(ctx):
    """Counts, lengths and parents outside their range: nothing of such a sequence is written, the others are
    whole, and the next synchronisation says so."""
    import torch
    import rabbit_amd as R
    rng = np.random.default_rng(0)
    B, N, H, K, D, cap = 5, 4, 4, 2, 64, 30
    par = T.random_parents(rng, B, N)
    n, lens = [4, 5, 4, -1, 4], [30, 3, 31, 3, -1]
    pos = torch.full((B, N), 9, dtype=torch.int32, device="cuda")
    ctx.tree_positions(_i(par), _i([4, 5, 4, -1, 4]), _i([30, 3, 0, 3, -1]), pos, sync=False)
    with pytest.raises(R.RbtError) as e:
        ctx.sync()
    assert e.value.status == R.abi.RBT_E_INVALID
    ctx.sync()  # reported once
    assert (_np(pos)[[1, 3, 4]] == -1).all() and (_np(pos)[[0, 2]] >= 0).all()
    q, kc, vc, kd, vd = (rng.standard_normal(sh).astype(np.float32) for sh in
                         ((B, N, H, D), (B, cap, K, D), (B, cap, K, D), (B, N, K, D), (B, N, K, D)))
    out = torch.full((B, N, H, D), 5.0, device="cuda")
    ctx.gqa_tree(_t(q), _t(kc), _t(vc), _t(kd), _t(vd), _i(lens), _i(n), _i(par), 0.125, out, sync=False)
    with pytest.raises(R.RbtError):
        ctx.sync()
    assert (_np(out)[1:] == 5.0).all()
    want, mag, qk = T.tree_attention(q[:1], kc[:1], vc[:1], kd[:1], vd[:1], [30], [4], par[:1], 0.125)
    assert (np.abs(_np(out)[:1] - want) <= T.tree_attention_bound(mag, qk, cap + N, D)).all()
    bad = par[:1].copy()
    bad[0, 2] = 2  # its own parent
    ctx.gqa_tree(_t(q[:1]), _t(kc[:1]), _t(vc[:1]), _t(kd[:1]), _t(vd[:1]), _i([30]), _i([4]), _i(bad), 0.125, out[:1], sync=False)
    with pytest.raises(R.RbtError):
        ctx.sync()
    path, n_path, nxt = (torch.full(sh, 9, dtype=torch.int32, device="cuda") for sh in ((1, 4), (1,), (1,)))
    p = torch.full((1, 4, 10), 0.1, device="cuda")
    for tok, cnt, pr in (([0, 10, 2, 3], 4, par[:1]), ([0, 1, -1, 3], 4, par[:1]), ([0, 1, 2, 3], 5, par[:1]), ([0, 1, 2, 3], 4, bad)):
        ctx.draft_verify(_i([tok]), _i(pr), _i([cnt]), p, _t(np.full((1, 4), 0.99, np.float32)), path, n_path, nxt, sync=False)
        with pytest.raises(R.RbtError):
            ctx.sync()
        assert _np(nxt)[0] == (-1 if cnt == 5 else 9)
    cache = [torch.zeros(1, 8, 1, 8, device="cuda") for _ in range(2)]
    draft = [torch.ones(1, 4, 1, 8, device="cuda") for _ in range(2)]
    lo = torch.full((1,), 99, dtype=torch.int32, device="cuda")
    for path, cnt, ln in (([0, 1, 2, 3], 4, 5), ([0, 4, -1, -1], 2, 0), ([0, -1, -1, -1], 2, 0), ([0, 1, 2, 3], 5, 0), ([0] * 4, 1, 9)):
        ctx.kv_commit(cache[:1], cache[1:], draft[:1], draft[1:], _i([path]), _i([cnt]), _i([ln]), lo, sync=False)
        with pytest.raises(R.RbtError):
            ctx.sync()
        assert _np(lo)[0] == ln and not cache[0].any() and not cache[1].any()


# ---- tree attention --------------------------------------------------------------------------------
def _attend(ctx, B, N, H, K, D, lens, counts, shape="tree", kv16=False, gate=None, seed=0, scale=None, max_len=0, cap=None, edit=None, rel=1e-5):
    """One call against the 64-bit form: the derived bound entry by entry, and 1e-5 relative L2 per row."""
    import torch
    rng = np.random.default_rng(seed + N + D + max(lens))
    cap = max(lens) + 3 if cap is None else cap
    scale = D ** -0.5 if scale is None else scale
    par = T.random_parents(rng, B, N, shape)
    q = rng.standard_normal((B, N, H, D)).astype(np.float32)
    kc, vc = (rng.standard_normal((B, cap, K, D)).astype(np.float32) for _ in range(2))
    kd, vd = (rng.standard_normal((B, N, K, D)).astype(np.float32) for _ in range(2))
    if kv16:
        kc, vc, kd, vd = (_bf(x) for x in (kc, vc, kd, vd))
    for b in range(B):  # rows that nothing may read
        kc[b, lens[b]:] = vc[b, lens[b]:] = np.nan
        kd[b, counts[b]:] = vd[b, counts[b]:] = np.nan
        q[b, counts[b]:] = np.nan
    if edit:
        edit(q, kc, vc, kd, vd, par)
    dt = torch.bfloat16 if kv16 else torch.float32
    g = gt = None
    if gate:
        qg = rng.standard_normal((B, N, H, 2, D)).astype(np.float32)
        g = qg[..., 1, :]
        gt = _t(qg)[..., 1, :]
    out = torch.full((B, N, H, D), 3.0, device="cuda")
    ctx.gqa_tree(_t(q), _t(kc, dt), _t(vc, dt), _t(kd, dt), _t(vd, dt), _i(lens), _i(counts), _i(par), scale, out, gate=gt,
                 max_len=max_len)
    want, mag, qk = T.tree_attention(q, kc, vc, kd, vd, lens, counts, par, scale, g, np.full(q.shape, 3.0))
    got = _np(out).astype(np.float64)
    worst = 0.0
    for b in range(B):
        c = counts[b]
        assert (got[b, c:] == 3.0).all()
        if c:
            tol = T.tree_attention_bound(mag[b, :c], qk[b, :c], lens[b] + c, D)
            off = np.abs(got[b, :c] - want[b, :c])
            assert np.isfinite(got[b, :c]).all() and (off <= tol).all(), (b, off.max(), (off / tol).max())
            worst = max(worst, np.max(np.linalg.norm(off, axis=-1) / np.linalg.norm(want[b, :c], axis=-1)))
    assert worst < rel, worst
    return got


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("H,K,D", [(64, 4, 256), (20, 4, 128), (3, 3, 64), (16, 1, 192), (34, 2, 64), (6, 2, 80), (2, 1, 1), (4, 2, 320)])
def test_tree_attention_shapes(ctx, H, K, D, kv16):
    """Head layouts from one query head per KV head to seventeen, head dims on and off the tiles; three
    sequences, one without a cache, one without nodes."""
    _attend(ctx, 3, 5, H, K, D, [130, 0, 77], [5, 4, 0], kv16=kv16)


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("N,shape", [(1, "tree"), (2, "chain"), (4, "tree"), (9, "forest"), (33, "tree"), (64, "chain"), (65, "tree"),
                                     (130, "forest"), (256, "chain"), (256, "tree")])
def test_tree_attention_nodes(ctx, N, shape, kv16):
    _attend(ctx, 1, N, 4, 2, 64, [70], [N], shape=shape, kv16=kv16, gate=True)


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("L", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2049, 5000])
def test_tree_attention_lengths(ctx, L, kv16):
    """Lengths around every tile and split."""
    _attend(ctx, 2, 3, 8, 2, 128, [L, L // 2], [3, 2], kv16=kv16)


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("H,K,D,N", [(16, 1, 64, 33), (16, 1, 256, 20), (48, 3, 192, 9), (8, 1, 128, 70), (1, 1, 64, 256)])
def test_tree_attention_ragged(ctx, H, K, D, N, kv16):
    """Row tiles over several workgroups and waves without rows: counts from none to all, several pieces of the
    cache beside none."""
    _attend(ctx, 4, N, H, K, D, [700, 90, 0, 1300], [N, N // 2 + 1, 1, 0], kv16=kv16, gate=True)


@pytest.mark.parametrize("kv16,N", [(False, 1), (True, 1), (False, 6), (True, 20)])
def test_tree_attention_qwen(ctx, kv16, N):
    """Qwen 3.8's heads with the gate inside q_proj's rows; max_len below and at the lengths."""
    got = [_attend(ctx, 2, N, 64, 4, 256, [700, 333], [N, N], kv16=kv16, gate=True, max_len=m, cap=800) for m in (0, 1, 700)]
    for g in got[1:]:
        assert rel_l2(g, got[0]) < 2e-6


@pytest.mark.parametrize("D,H", [(64, 4), (80, 4), (64, 32), (256, 32), (128, 2)])
@pytest.mark.parametrize("kv16", [False, True])
def test_tree_attention_masked_values(ctx, D, H, kv16):
    """NaN, infinities and the largest values in nodes that others do not see; a node that sees one has it."""
    import torch
    rng = np.random.default_rng(3)
    N, K, L = 12, 2, 40
    big = float(np.finfo(np.float32).max) if not kv16 else 3.0e38

    def edit(q, kc, vc, kd, vd, par):
        par[0, :] = [-1, 0, 0, 0, 1, 2, 3, 4, 5, 6, 7, 8]
        kd[0, 1], vd[0, 2], kd[0, 3], vd[0, 3] = np.nan, np.inf, -np.inf, np.nan
        vd[0, 4], kd[0, 5] = np.nan, big

    for b16 in (kv16,):
        q = rng.standard_normal((1, N, H, D)).astype(np.float32)
        kc, vc = (_bf(rng.standard_normal((1, L, K, D))) for _ in range(2))
        kd, vd = (_bf(rng.standard_normal((1, N, K, D))) for _ in range(2))
        par = np.zeros((1, N), np.int32)
        clean = (kd.copy(), vd.copy())
        edit(q, kc, vc, kd, vd, par)
        dt = torch.bfloat16 if b16 else torch.float32
        out = torch.zeros(1, N, H, D, device="cuda")
        ctx.gqa_tree(_t(q), _t(kc, dt), _t(vc, dt), _t(kd, dt), _t(vd, dt), _i([L]), _i([N]), _i(par), D ** -0.5, out)
        want, mag, qk = T.tree_attention(q, kc, vc, *clean, [L], [N], par, D ** -0.5)
        got = _np(out)
        dirty = {1, 2, 3, 4, 5}
        for i in range(N):
            seen = set(T.ancestors(par[0], i))
            if not seen & dirty:
                assert (np.abs(got[0, i] - want[0, i]) <= T.tree_attention_bound(mag[0, i], qk[0, i], L + N, D)).all(), i
            if seen & {1, 4}:  # NaN keys or values on the way
                assert np.isnan(got[0, i]).all(), i


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("B,N,H,K,D,lens,counts,cap", [
    (9, 12, 32, 4, 64, [4100, 0, 63, 2049, 1, 4096, 700, 64, 4099], [12, 12, 0, 5, 1, 12, 7, 12, 3], 4100),
    (8, 40, 16, 1, 256, [3400, 100, 3333, 0, 65, 2000, 1500, 3399], [40, 17, 39, 40, 1, 0, 25, 9], 3400),
    (6, 12, 16, 1, 64, [3, 0, 70, 1, 5, 2], [12, 3, 12, 1, 9, 12], 12000),
    (6, 12, 16, 1, 192, [11999, 0, 70, 1, 5, 2], [12, 3, 12, 1, 9, 12], 12000),
    (70, 6, 8, 1, 128, [37 * i % 1900 for i in range(70)], [i % 7 for i in range(70)], 1900),
    (64, 6, 8, 1, 128, [1900] + [0] * 63, [6] * 64, 1900)])
def test_tree_attention_batches(ctx, B, N, H, K, D, lens, counts, cap, kv16):
    """Larger batches: lengths from none to all, several row tiles, caches far longer than what they hold, more
    than a wave of sequences, one long sequence among empty ones."""
    _attend(ctx, B, N, H, K, D, lens, counts, kv16=kv16, gate=True, cap=cap)


@pytest.mark.parametrize("kv16", [False, True])
def test_tree_attention_many_short(ctx, kv16):
    """Many short sequences; non-finite values of one stay out of the others' rows."""
    import torch
    B, N, H, K, D, cap = 300, 12, 32, 8, 64, 200
    rng = np.random.default_rng(17)
    lens, counts = rng.integers(0, cap + 1, B), rng.integers(0, N + 1, B)
    _attend(ctx, B, N, H, K, D, lens.tolist(), counts.tolist(), kv16=kv16, cap=cap)
    dt = torch.bfloat16 if kv16 else torch.float32
    q = rng.standard_normal((B, N, H, D)).astype(np.float32)
    kc, vc = (_bf(rng.standard_normal((B, cap, K, D))) for _ in range(2))
    kd, vd = (_bf(rng.standard_normal((B, N, K, D))) for _ in range(2))
    par = np.tile(np.array([[-1] + [0] * (N - 1)], np.int32), (B, 1))  # node 1 is seen by itself only
    outs = []
    for bad in (False, True):
        if bad:
            vd[::2, 1] = np.inf
        out = torch.zeros(B, N, H, D, device="cuda")
        ctx.gqa_tree(_t(q), _t(kc, dt), _t(vc, dt), _t(kd, dt), _t(vd, dt), _i(lens), _i(counts), _i(par), 0.125, out)
        outs.append(_np(out))
    keep = np.ones((B, N), bool)
    keep[::2, 1] = False
    assert np.array_equal(outs[0][keep], outs[1][keep])
    hit = [b for b in range(0, B, 2) if counts[b] > 1]
    assert not np.isfinite(outs[1][hit, 1]).any()


def test_tree_attention_extreme_scores(ctx):
    """Scores past a hundred, all equal ones, and a scale of 0 and below it."""
    def scaled(f):
        def edit(q, *rest):
            q *= f
        return edit
    _attend(ctx, 1, 3, 4, 2, 64, [300], [3], scale=0.0)
    _attend(ctx, 1, 3, 4, 2, 64, [300], [3], scale=-0.125)
    _attend(ctx, 1, 3, 4, 2, 64, [300], [3], edit=scaled(0.0))
    _attend(ctx, 1, 3, 4, 2, 64, [300], [3], edit=scaled(30.0), kv16=True, rel=1e-4)  # sum |q k| near 150: a few u of it


def test_tree_attention_long(ctx):
    """A long cache split over many workgroups, short beside it."""
    _attend(ctx, 2, 2, 4, 1, 64, [40000, 3], [2, 2], kv16=True)


def test_tree_attention_far_offsets(ctx):
    """The last of the sequences lies past 2^32 bytes and 2^31 entries of the caches."""
    import torch
    B, N, H, K, D, cap = 3, 2, 4, 4, 256, 900000
    rng = np.random.default_rng(8)
    kc = torch.empty(B, cap, K, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    L = 50
    kc[2, :L], vc[2, :L] = _t(rng.standard_normal((L, K, D)).astype(np.float32), kc.dtype), \
        _t(rng.standard_normal((L, K, D)).astype(np.float32), kc.dtype)
    q, kd, vd = rng.standard_normal((B, N, H, D)).astype(np.float32), _bf(rng.standard_normal((B, N, K, D))), \
        _bf(rng.standard_normal((B, N, K, D)))
    par = np.array([[-1, 0]] * B, np.int32)
    out = torch.zeros(B, N, H, D, device="cuda")
    ctx.gqa_tree(_t(q), kc, vc, _t(kd, kc.dtype), _t(vd, kc.dtype), _i([0, 0, L]), _i([0, 0, N]), _i(par), 0.0625, out, max_len=64)
    want, mag, qk = T.tree_attention(q[2:], _np(kc[2:, :L]), _np(vc[2:, :L]), kd[2:], vd[2:], [L], [N], par[2:], 0.0625)
    assert (np.abs(_np(out)[2:] - want) <= T.tree_attention_bound(mag, qk, L + N, D)).all()
    # and the move of the rows to the last places of the same caches
    lo = torch.zeros(B, dtype=torch.int32, device="cuda")
    ctx.kv_commit([kc], [vc], [_t(kd, kc.dtype)], [_t(vd, kc.dtype)], _i([[0, 1]] * B), _i([0, 0, 2]), _i([0, 0, cap - 2]), lo)
    assert np.array_equal(_np(kc[2, cap - 2:]), kd[2]) and np.array_equal(_np(vc[2, cap - 2:]), vd[2])
    assert _np(lo).tolist() == [0, 0, cap]


# ---- verification ----------------------------------------------------------------------------------
def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _verify(ctx, tok, par, n, p, q, u, max_children=0):
    import torch
    B, N = tok.shape
    path, n_path, nxt = (torch.full(sh, -9, dtype=torch.int32, device="cuda") for sh in ((B, N), (B,), (B,)))
    ctx.draft_verify(_i(tok), _i(par), _i(n), _t(p), _t(u), path, n_path, nxt, q=None if q is None else _t(q), max_children=max_children)
    want = T.verify(tok, par, n, p, q, u)
    for name, g, w in zip(("path", "n_path", "next"), (path, n_path, nxt), want):
        assert np.array_equal(_np(g), w), (name, np.argwhere(_np(g) != w)[:4], _np(g)[_np(g) != w][:4], w[_np(g) != w][:4])
    return want


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("B,N,V,shape,children", [
    (1, 1, 1, "tree", 0), (2, 1, 1000, "chain", 1), (3, 5, 7, "tree", 0), (8, 16, 1003, "tree", 0), (4, 33, 4096, "tree", 2),
    (2, 256, 517, "tree", 0), (2, 256, 64, "chain", 1), (5, 9, 50001, "forest", 0), (3, 6, 131075, "chain", 0), (40, 8, 300, "tree", 3)])
def test_verify(ctx, B, N, V, shape, children, drawn):
    """Trees of drafts from a distribution near the target's; ragged counts, odd vocabularies."""
    rng = np.random.default_rng(B * 1000 + N + V)
    logits = rng.standard_normal((B, N, V)) * 3
    p, q = _softmax(logits), _softmax(logits + rng.standard_normal((B, N, V)))
    par = T.random_parents(rng, B, N, shape)
    n = rng.integers(0, N + 1, B)
    n[0] = N
    tok = np.zeros((B, N), np.int32)
    for b in range(B):
        for i in range(1, N):
            r = q[b, max(par[b, i], 0)].astype(np.float64)
            tok[b, i] = rng.choice(V, p=r / r.sum())
    u = rng.random((B, N), dtype=np.float32)
    path, n_path, _ = _verify(ctx, tok, par, n, p, q if drawn else None, u, children)
    assert n_path.max() <= N


def test_verify_children_past_the_hint(ctx):
    """max_children changes only how the work is launched: a tree of many children called a chain."""
    rng = np.random.default_rng(3)
    B, N, V = 3, 40, 9000
    p, q = (_softmax(rng.standard_normal((B, N, V)) * 3) for _ in range(2))
    par = np.where(np.arange(N) == 0, -1, 0)[None].repeat(B, 0).astype(np.int32)
    tok = rng.integers(0, V, (B, N)).astype(np.int32)
    u = (0.5 + 0.5 * rng.random((B, N))).astype(np.float32).clip(0, np.float32(1 - 2.0 ** -24))
    for hint in (1, 2, 0, 1 << 40):
        _verify(ctx, tok, par, [N] * B, p, q, u, hint)


def test_verify_borders(ctx):
    """Given numbers at the ends of their range, rows with zeros, repeated siblings, an empty residual."""
    V = 1500
    rng = np.random.default_rng(5)
    p = _softmax(rng.standard_normal((6, 4, V)) * 3)
    q = _softmax(rng.standard_normal((6, 4, V)) * 3)
    par = np.array([[-1, 0, 0, 0]] * 6, np.int32)
    tok = rng.integers(0, V, (6, 4)).astype(np.int32)
    u = rng.random((6, 4), dtype=np.float32)
    u[0], u[1] = 0.0, np.float32(1.0) - np.float32(2.0 ** -24)
    p[2, 0, : V // 2], p[2, 0, -5:] = 0.0, 0.0
    tok[3, 1:] = tok[3, 1]                       # the same token three times
    q[4] = p[4]                                  # the residual is empty: every child stands but for u = 1 - 2^-24
    p[5, 0] = 0.0
    p[5, 0, 77] = 1.0                            # one certain token
    for qq in (q, None):
        for n in ([4] * 6, [1] * 6):
            _verify(ctx, tok, par, n, p, qq, u)
    z = p.copy()
    z[0], z[1, 0], z[2, 0, 3], z[3, 0, 9] = 0.0, np.nan, np.inf, -1.0
    want = _verify(ctx, tok, par, [1] * 6, z, None, u)
    assert want[2][0] == -1 and want[2][1] == -1 and want[2][2] == -1 and want[2][3] >= 0


def test_verify_keeps_the_targets_distribution(ctx):
    """Over many sequences the first token after node 0 is distributed as p, whatever the drafts: the largest
    deviation of the counts is within five standard deviations."""
    V, B = 6, 1024
    rng = np.random.default_rng(11)
    p, q = np.array([.3, .05, .25, .1, .2, .1]), np.array([.1, .4, .1, .2, .1, .1])
    counts = np.zeros(V)
    for rep in range(8):
        tok = np.zeros((B, 4), np.int32)
        tok[:, 1:] = rng.choice(V, (B, 3), p=q)
        par = np.array([[-1, 0, 0, 0]] * B, np.int32)
        u = rng.random((B, 4), dtype=np.float32)
        P, Q = (np.broadcast_to(x.astype(np.float32), (B, 4, V)) for x in (p, q))
        path, n_path, nxt = _verify(ctx, tok, par, np.full(B, 4), P, Q, u)
        first = np.where(n_path > 1, np.take_along_axis(tok, np.maximum(path[:, 1:2], 0), 1)[:, 0], nxt)
        counts += np.bincount(first, minlength=V)
    n = 8 * B
    assert (np.abs(counts - n * p) < 5 * np.sqrt(n * p * (1 - p))).all(), counts / n


# ---- commit ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("L,K,D,dtype,off", [(1, 4, 256, "bfloat16", 0), (3, 2, 64, "float32", 0), (2, 1, 3, "bfloat16", 0),
                                             (2, 3, 5, "float32", 0), (2, 2, 8, "bfloat16", 1), (70, 1, 16, "bfloat16", 0), (0, 1, 8, "float32", 0)])
def test_commit(ctx, L, K, D, dtype, off):
    """Rows of any width and alignment, more layers than one launch takes, no layers; full caches and empty paths."""
    import torch
    rng = np.random.default_rng(L + D)
    B, N, cap = 4, 9, 20
    dt = getattr(torch, dtype)

    def buf(*shape):
        n = int(np.prod(shape))
        return torch.randn(n + off, device="cuda").to(dt)[off:].view(*shape)

    caches = [[buf(B, cap, K, D) for _ in range(L)] for _ in range(2)]
    drafts = [[buf(B, N, K, D) for _ in range(L)] for _ in range(2)]
    before = [[t.clone() for t in side] for side in caches]
    lens, cnt = [0, 11, 20, 7], [9, 9, 0, 4]
    path = np.full((B, N), -1, np.int32)
    for b in range(B):
        path[b, :cnt[b]] = np.sort(rng.choice(N, cnt[b], replace=False))
    lo = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    ctx.kv_commit(*caches, *drafts, _i(path), _i(cnt), _i(lens), lo)
    assert _np(lo).tolist() == [a + c for a, c in zip(lens, cnt)]
    for side in range(2):
        for l in range(L):
            for b in range(B):
                before[side][l][b, lens[b]:lens[b] + cnt[b]] = drafts[side][l][b, torch.from_numpy(path[b, :cnt[b]].astype(np.int64)).cuda()]
            assert torch.equal(caches[side][l], before[side][l])


# ---- together --------------------------------------------------------------------------------------
class _Step:
    """A decode step of one attention layer and the verification, on buffers of its own."""

    def __init__(self, R, B, N, H, K, D, rd, cap, kv, V, angle_f32=True):
        import torch
        self.R, self.B, self.N, self.H, self.K, self.D = R, B, N, H, K, D
        rng = np.random.default_rng(17)
        z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.inv = _t(R.rope_freqs(rd, 1e7, as_f32=angle_f32)[0])
        self.angle_f32 = angle_f32
        self.qn, self.kn = (_t((0.1 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
        self.qg, self.k, self.v = z(B, N, H, 2, D), z(B, N, K, D), z(B, N, K, D)
        self.q, self.out = z(B, N, H, D), z(B, N, H, D)
        self.kd, self.vd, self.kc, self.vc = z(B, N, K, D, dtype=kv), z(B, N, K, D, dtype=kv), z(B, cap, K, D, dtype=kv), z(B, cap, K, D, dtype=kv)
        self.len, self.len2, self.n = (z(B, dtype=torch.int32) for _ in range(3))
        self.parent, self.pos, self.tok, self.path = (z(B, N, dtype=torch.int32) for _ in range(4))
        self.n_path, self.next = z(B, dtype=torch.int32), z(B, dtype=torch.int32)
        self.p, self.pq, self.u = z(B, N, V), z(B, N, V), z(B, N)
        s, rows = B * N, lambda t: t.view(B * N, *t.shape[2:])  # noqa: E731
        self.parts = [R.rope_part(rows(self.qg)[:, :, 0], rows(self.q), norm=self.qn),
                      R.rope_part(rows(self.k), rows(self.kd), norm=self.kn), R.rope_part(rows(self.v), rows(self.vd), rotate=False)]

    def run(self, ctx, sync=True, verify=True):
        ctx.tree_positions(self.parent, self.n, self.len, self.pos, sync=sync)
        ctx.rope(self.parts, self.pos, self.D, self.inv, angle_f32=self.angle_f32, sync=sync)
        ctx.gqa_tree(self.q, self.kc, self.vc, self.kd, self.vd, self.len, self.n, self.parent, self.D ** -0.5, self.out,
                     gate=self.qg[..., 1, :], sync=sync)
        if verify:
            ctx.draft_verify(self.tok, self.parent, self.n, self.p, self.u, self.path, self.n_path, self.next, q=self.pq, sync=sync)
        ctx.kv_commit([self.kc], [self.vc], [self.kd], [self.vd], self.path, self.n_path, self.len, self.len2, sync=sync)


def test_decode_steps_match_the_one_token_step(ctx):
    """Plain decoding of two sequences and then a tree, over Qwen 3.8's heads: outputs and caches as
    rbt_gqa_step_d gives them token by token along every path of the tree."""
    import torch
    import rabbit_amd as R
    H, K, D, rd, cap, N = 64, 4, 256, 64, 40, 7
    st = _Step(R, 2, N, H, K, D, rd, cap, torch.float32, 11)
    g = torch.Generator(device="cuda").manual_seed(1)
    ref = [(torch.zeros(cap, K, D, device="cuda"), torch.zeros(cap, K, D, device="cuda")) for _ in range(2)]

    def step(b, pos, i, caches):
        out = torch.zeros(H, D, device="cuda")
        ctx.gqa_step(H, K, D, rd, 1e7, D ** -0.5, 1e-6, st.qn, st.kn, *caches, cap, pos, st.qg[b, i].contiguous(),
                     st.k[b, i].contiguous(), st.v[b, i].contiguous(), out)
        return out

    def fill():
        for t in (st.qg, st.k, st.v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))

    st.n.fill_(1)
    st.parent.fill_(-1)
    st.path.fill_(-1)
    st.path[:, 0] = 0
    st.n_path.fill_(1)
    for pos in range(9):  # plain decoding: one node per sequence
        fill()
        st.run(ctx, verify=False)
        for b in range(2):
            want = step(b, pos, 0, ref[b])
            assert rel_l2(_np(st.out[b, 0]), _np(want)) < 1e-5
        st.len.copy_(st.len2)
    fill()
    par = np.array([[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, 2, 3, 4, 5]], np.int32)
    st.parent.copy_(_i(par))
    st.n.fill_(N)
    st.path.copy_(_i([[0, 2, 5, 6, -1, -1, -1], [0, 1, 2, -1, -1, -1, -1]]))
    st.n_path.copy_(_i([4, 3]))
    st.run(ctx, verify=False)
    for b in range(2):
        for i in range(N):
            way = T.ancestors(par[b], i)
            caches = tuple(t.clone() for t in ref[b])
            for j, node in enumerate(way):
                want = step(b, 9 + j, node, caches)
            assert rel_l2(_np(st.out[b, i]), _np(want)) < 1e-5, (b, i)
            if way == _np(st.path[b])[:len(way)].tolist() and len(way) == int(st.n_path[b]):
                for got, w in zip((st.kc[b], st.vc[b]), caches):  # the committed rows are the path's
                    assert rel_l2(_np(got[:9 + len(way)]), _np(w[:9 + len(way)])) < 1e-6
    assert _np(st.len2).tolist() == [13, 12]


@pytest.mark.parametrize("kv", ["float32", "bfloat16"])
def test_captured_step_replays(own_ctx, kv):
    """A whole step in a HIP graph: replays over new inputs, lengths and trees equal the eager step, with eager
    work between them; a second graph of another size shares the context's scratch."""
    import torch
    import rabbit_amd as R
    from helpers import HipGraph
    ctx = own_ctx
    B, N, V = 3, 12, 700
    st = [_Step(R, B, n, 16, 2, 128, 64, 300, getattr(torch, kv), V, angle_f32=False) for n in (N, 3)]
    rng = np.random.default_rng(2)

    def fill(s, n, rep):
        for t in (s.qg, s.k, s.v, s.kc, s.vc):
            t.copy_(_t(rng.standard_normal(tuple(t.shape)).astype(np.float32)))
        s.len.copy_(_i(rng.integers(0, 300 - n, B)))
        s.n.copy_(_i([n, rng.integers(0, n + 1), rng.integers(1, n + 1)]))
        s.parent.copy_(_i(T.random_parents(rng, B, n, ("tree", "chain", "tree")[rep % 3])))
        s.tok.copy_(_i(rng.integers(0, 20, (B, n))))
        lg = rng.standard_normal((B, n, V)).astype(np.float32)
        lg[..., :20] += 6
        s.p.copy_(_t(_softmax(lg)))
        s.pq.copy_(_t(_softmax(lg + 0.5 * rng.standard_normal(lg.shape))))
        s.u.copy_(_t(rng.random((B, n), dtype=np.float32)))

    names = ("out", "path", "n_path", "next", "len2", "kc", "vc", "pos")
    graphs = []
    for s, n in zip(st, (N, 3)):
        fill(s, n, 0)
        s.run(ctx)
        gr = HipGraph(ctx.stream)
        gr.begin()
        s.run(ctx, sync=False)
        gr.end()
        graphs.append(gr)
    for rep in range(4):
        for s, n, gr in zip(st, (N, 3), graphs):
            fill(s, n, rep)
            torch.cuda.synchronize()
            state = {k: getattr(s, k).clone() for k in names}
            gr.launch()
            ctx.sync()
            got = {k: getattr(s, k).clone() for k in names}
            for k in names:
                getattr(s, k).copy_(state[k])
            s.run(ctx)  # eager work between the replays
            for k in names:
                assert torch.equal(got[k], getattr(s, k)), (rep, n, k)


@pytest.mark.parametrize("D,H,N", [(64, 8, 3), (128, 16, 5), (192, 8, 2)])
def test_captured_before_any_call_of_its_kind(own_ctx, D, H, N):
    """The first call of a shape stands in a capture (its split is chosen there); scratch is there from a larger one."""
    import torch
    from helpers import HipGraph
    ctx, B, K, cap = own_ctx, 12, 2, 900
    g = torch.Generator(device="cuda").manual_seed(D)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    big = [r(8, 40, 32, 256), r(8, 1000, 2, 256), r(8, 1000, 2, 256), r(8, 40, 2, 256), r(8, 40, 2, 256)]
    ctx.gqa_tree(*big, _i([1000] * 8), _i([40] * 8), _i(np.tile(np.arange(-1, 39), (8, 1))), 0.1, torch.empty_like(big[0]))
    q, kc, vc, kd, vd = r(B, N, H, D), r(B, cap, K, D), r(B, cap, K, D), r(B, N, K, D), r(B, N, K, D)
    par, n = _i(np.tile(np.arange(-1, N - 1), (B, 1))), _i([N] * B)
    ln, out = _i([0] * B), torch.zeros_like(q)
    torch.cuda.synchronize()
    gr = HipGraph(ctx.stream)
    gr.begin()
    ctx.gqa_tree(q, kc, vc, kd, vd, ln, n, par, 0.1, out, sync=False)
    gr.end()
    for rep in range(3):
        ln.copy_(_i([(rep * 311 + 97 * b) % (cap + 1) for b in range(B)]))
        out.zero_()
        torch.cuda.synchronize()
        gr.launch()
        ctx.sync()
        want = torch.zeros_like(q)
        ctx.gqa_tree(q, kc, vc, kd, vd, ln, n, par, 0.1, want)
        assert torch.equal(out, want), rep


def test_results_do_not_change_from_run_to_run(ctx):
    """The same call twice gives the same bits."""
    import torch
    import rabbit_amd as R
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, kc, vc, kd, vd = r(2, 9, 32, 128), r(2, 3000, 4, 128), r(2, 3000, 4, 128), r(2, 9, 4, 128), r(2, 9, 4, 128)
    par = _i(T.random_parents(np.random.default_rng(0), 2, 9))
    outs = []
    for _ in range(3):
        out = torch.zeros_like(q)
        ctx.gqa_tree(q, kc, vc, kd, vd, _i([2999, 1777]), _i([9, 8]), par, 0.1, out)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- products of split f32 rows ----------------------------------------------------------------------
def _one_row(ctx, B, N, H, K, D, cap, q, kc, vc, kd, vd, scale):
    """One committed row, and nodes that see it and themselves; every head and node has the same numbers, given by
    their first entries. -> (out [D], the 64-bit form's)."""
    import torch
    full = lambda head, *sh: np.broadcast_to(np.pad(np.asarray(head, np.float32), (0, D - len(head))), (*sh, D)).copy()  # noqa: E731
    a = [full(q, B, N, H), full(kc, B, cap, K), full(vc, B, cap, K), full(kd, B, N, K), full(vd, B, N, K)]
    par = np.full((B, N), -1, np.int32)
    out = torch.zeros(B, N, H, D, device="cuda")
    ctx.gqa_tree(*(_t(x) for x in a), _i([1] * B), _i([N] * B), _i(par), scale, out)
    got = _np(out).astype(np.float64)
    assert (got == got[0, 0, 0]).all()
    want, _, _ = T.tree_attention(a[0][:1, :1, :K], *(x[:1, :1] for x in a[1:]), [1], [1], par[:1, :1], scale)
    return got[0, 0, 0], want[0, 0, 0]


# 48 rows of one KV head (three row tiles) by eight waves, and in a batch with room for 600 rows by four
SPLIT = [(1, 1, 48, 1, 64, 1), (1, 4, 48, 4, 192, 9), (2, 1, 48, 1, 256, 1), (16, 4, 96, 8, 64, 600), (16, 4, 96, 8, 128, 600)]
LONG = np.array(0x3f80ffff, np.uint32).view(np.float32)  # 1 + 2^-7 - 2^-23
LN2 = np.float32(np.log(2.0))                            # times log2(e) in f32 it rounds to 1: scores are exact powers of two


@pytest.mark.parametrize("B,N,H,K,D,cap", SPLIT)
def test_split_keys_products(ctx, B, N, H, K, D, cap):
    """The product of two long mantissas against its fp32 rounding times a power of two (all parts kept, their sum exact).
    Their difference of scores, near 2^14 in powers of two, is off by the last addition (2u at most, whichever way it
    rounds) and by the products left out (for these two numbers 2^-38); the output's slope over it is ln 2 / 4."""
    t = np.float32(2.0 ** 14)
    got, want = _one_row(ctx, B, N, H, K, D, cap, [LONG, LONG * LONG], [LONG * t], [1.0], [0.0, t], [0.0], LN2)
    assert abs(got[0] - want[0]) <= np.log(2) / 4 * 2.1 * T.U32 * float(t) * 1.02 + 2.0 ** -22, (got[0], want[0])
    got, want = _one_row(ctx, B, N, H, K, D, cap, [-LONG, LONG * LONG], [LONG * t], [1.0], [0.0, -t], [0.0], LN2)
    assert abs(got[0] - want[0]) <= np.log(2) / 4 * 2.1 * T.U32 * float(t) * 1.02 + 2.0 ** -22, (got[0], want[0])


@pytest.mark.parametrize("B,N,H,K,D,cap", SPLIT)
def test_split_values_products(ctx, B, N, H, K, D, cap):
    """A probability with a long middle and last part times 1 and times a long mantissa: their quotient is that mantissa but
    for the last addition (2u at most), two divisions (u each) and the products left out (2^-38)."""
    s = np.float32(np.log2(0.5 * (1.0 + 2.0 ** -7 - 2.0 ** -21)))
    got, _ = _one_row(ctx, B, N, H, K, D, cap, [1.0], [s], [1.0, LONG, -LONG], [0.0], [0.0], LN2)
    for g, w in ((got[1], float(LONG)), (got[2], -float(LONG))):
        assert abs(g / got[0] / w - 1.0) <= 4.1 * T.U32, (g / got[0] / w - 1.0) / T.U32


def test_split_rows_of_the_largest_numbers(ctx):
    """Finite numbers that would round to an infinite bf16 keep their products."""
    top = np.float32(np.finfo(np.float32).max)
    got, want = _one_row(ctx, 1, 1, 48, 1, 64, 1, [2.0 ** -126, 0.0], [top], [top, -top], [0.0, top], [0.0], 1.0)
    assert np.isfinite(got).all() and (np.abs(got[:2] / want[:2] - 1.0) <= 2.0 ** -19).all()
    got, want = _one_row(ctx, 1, 1, 48, 1, 64, 1, [top], [2.0 ** -126], [1.0], [0.0], [0.0], 1.0)
    assert abs(got[0] - want[0]) <= 2.0 ** -20


# ---- non-finite keys and values that are seen ----------------------------------------------------------
# one to 24 row tiles of a KV head, one sequence and batches; caches of several pieces (the last: one)
SEEN = [(1, 12, 4, 2, 64, 5000), (1, 24, 32, 2, 256, 3000), (1, 9, 4, 2, 192, 4000), (16, 12, 32, 8, 64, 1500),
        (16, 12, 32, 4, 128, 1500), (2, 12, 4, 2, 80, 300), (2, 12, 8, 2, 128, 40)]


def _seen_case(B, N, H, K, D, L, kv16, rng):
    q = rng.standard_normal((B, N, H, D)).astype(np.float32)
    kc, vc = (_bf(rng.standard_normal((B, L, K, D))) for _ in range(2))
    kd, vd = (_bf(rng.standard_normal((B, N, K, D))) for _ in range(2))
    par = np.broadcast_to(np.array([-1, 0, 0, 0, 0, 0, 2, 3, 4, 0] + [0] * (N - 10) if N > 9 else [-1, 0, 0, 0, 0, 0, 2, 3, 4]), (B, N))
    return q, kc, vc, kd, vd, par.astype(np.int32).copy()


def _seen_call(ctx, q, kc, vc, kd, vd, par, kv16):
    import torch
    B, N, _, D = q.shape
    dt = torch.bfloat16 if kv16 else torch.float32
    out = torch.zeros(q.shape, device="cuda")
    ctx.gqa_tree(_t(q), _t(kc, dt), _t(vc, dt), _t(kd, dt), _t(vd, dt), _i([kc.shape[1]] * B), _i([N] * B), _i(par), D ** -0.5, out)
    return _np(out)


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("B,N,H,K,D,L", SEEN)
def test_seen_values_reach_their_entries(ctx, B, N, H, K, D, L, kv16):
    """A non-finite value makes its entry of the nodes that see it non-finite and nothing else; a NaN key all entries."""
    q, kc, vc, kd, vd, par = _seen_case(B, N, H, K, D, L, kv16, np.random.default_rng(D + L))
    vals = [x.copy() for x in (vc, kd, vd)]
    R, hit = H // K, np.zeros(q.shape, bool)
    sees = np.array([[j in T.ancestors(par[0], i) for j in range(N)] for i in range(N)])

    def put(where, j, entry, value, heads=slice(None)):
        where[:, j, heads, entry] = value
        rows = slice(None) if where is vals[0] else sees[:, j]
        h = [x for x in range(H) if x // R in range(K)[heads]]
        e = slice(None) if where is vals[1] else entry
        hit[np.ix_(range(B), np.arange(N)[rows], h, np.arange(D)[e] if isinstance(e, slice) else [e])] = True

    put(vals[0], L // 3, 9, np.inf, slice(1, 2))       # committed, seen by every node of one KV head
    put(vals[0], L - 1, D - 1, np.nan, slice(0, 1))
    put(vals[2], 2, 3, np.inf)
    put(vals[2], 3, 17, np.nan)
    put(vals[2], 4, 40, -np.inf)
    put(vals[2], 1, 5, np.inf)                          # a leaf
    put(vals[1], 5, 8, np.nan)                          # a NaN key
    got = _seen_call(ctx, q, kc, vals[0], vals[1], vals[2], par, kv16)
    want, mag, qk = T.tree_attention(q, kc, vc, kd, vd, [L] * B, [N] * B, par, D ** -0.5)
    ok = np.abs(got - want) <= T.tree_attention_bound(mag, qk, L + N, D)
    assert not np.isfinite(got[hit]).any(), np.argwhere(hit & np.isfinite(got))[:5]
    assert ok[~hit].all(), np.argwhere(~hit & ~ok)[:5]


@pytest.mark.parametrize("kv16", [False, True])
@pytest.mark.parametrize("B,N,H,K,D,L", SEEN)
def test_seen_infinite_keys(ctx, B, N, H, K, D, L, kv16):
    """An infinite key has no weight where its score is -inf, or makes the output non-finite; nodes that do not see it have
    theirs."""
    q, kc, vc, kd, vd, par = _seen_case(B, N, H, K, D, L, kv16, np.random.default_rng(D + L + 1))
    want, mag, qk = T.tree_attention(q, kc, vc, kd, vd, [L] * B, [N] * B, par, D ** -0.5)
    gone, mag2, qk2 = T.tree_attention(q, np.delete(kc, L // 2, 1), np.delete(vc, L // 2, 1), kd, vd, [L - 1] * B, [N] * B, par, D ** -0.5)
    bad = kd.copy()
    bad[:, 2, :, 11] = np.inf
    sees = np.array([2 in T.ancestors(par[0], i) for i in range(N)])
    got = _seen_call(ctx, q, kc, vc, bad, vd, par, kv16)
    assert (np.abs(got - want) <= T.tree_attention_bound(mag, qk, L + N, D))[:, ~sees].all()
    assert not np.isfinite(got[:, sees][q[:, sees][..., 11] > 0]).any()  # score inf
    bad = kc.copy()
    bad[:, L // 2, :, 11] = -np.inf
    got = _seen_call(ctx, q, bad, vc, kd, vd, par, kv16)
    rows = np.isfinite(got).all(-1)
    assert not np.isfinite(got[~rows]).any() and not rows[q[..., 11] < 0].any()
    assert (np.abs(got - gone) <= T.tree_attention_bound(mag2, qk2, L + N, D))[rows].all()


def test_positions_up_to_the_largest(ctx):
    """Positions up to 2^31 - 1; a sequence whose nodes could pass it is skipped and reported, not wrapped around."""
    import torch
    import rabbit_amd as R
    top = (1 << 31) - 1
    par = _i([[-1, 0, 1]] * 4)
    pos = torch.full((4, 3), 9, dtype=torch.int32, device="cuda")
    ctx.tree_positions(par, _i([3, 1, 0, 2]), _i([top - 2, top, top, 5]), pos)
    assert _np(pos).tolist() == [[top - 2, top - 1, top], [top, -1, -1], [-1] * 3, [5, 6, -1]]
    ctx.tree_positions(par, _i([3, 2, 3, 2]), _i([top - 1, top, 4, 5]), pos, sync=False)
    with pytest.raises(R.RbtError):
        ctx.sync()
    assert _np(pos).tolist() == [[-1] * 3, [-1] * 3, [4, 5, 6], [5, 6, -1]]


@pytest.mark.parametrize("N,V,children", [(2, 5000, 0), (2, 70001, 0), (12, 70001, 0), (12, 40000, 11), (200, 20000, 0)])
def test_verify_rejections(ctx, N, V, children):
    """One child, and more rejections at one node than the call has launches: each residual is the last one's, and the draw is
    from what the last leaves."""
    rng = np.random.default_rng(N + V)
    B = 3
    p, q = (_softmax(rng.standard_normal((B, N, V)) * 2) for _ in range(2))
    par = np.where(np.arange(N) == 0, -1, 0)[None].repeat(B, 0).astype(np.int32)
    tok = np.stack([rng.choice(V, N, p=q[b, 0].astype(np.float64) / q[b, 0].astype(np.float64).sum()) for b in range(B)])
    u = rng.random((B, N), dtype=np.float32)
    u[:2, 1:] = np.float32(1.0) - np.float32(2.0 ** -24)  # rejected unless the residual passes q
    p[1, 0, tok[1, 1:]] = 0.0                              # none can stand
    path, n_path, _ = _verify(ctx, tok.astype(np.int32), par, [N] * B, p, q, u, children)
    assert n_path[1] == 1
