"""CPU checks of the drafted-token entry points: rotary frequency tables against their formulas, and every
refusal of arguments (they are checked before the context, so a call without one reaches them)."""
import ctypes as C
import math

import numpy as np
import pytest

from rabbit_amd import abi
from rabbit_amd.abi import RBT_E_INVALID, RBT_E_UNSUPPORTED


def test_plain_frequencies(rbt_lib):
    import rabbit_amd as R
    inv, f = R.rope_freqs(64, 1e7)
    np.testing.assert_allclose(inv, 1e7 ** (-np.arange(0, 64, 2) / 64), rtol=1e-14)
    assert f == 1.0
    inv, f = R.rope_freqs(64, 1e6, kind=R.ROPE_LINEAR, factor=4.0)
    np.testing.assert_allclose(inv, 1e6 ** (-np.arange(0, 64, 2) / 64) / 4.0, rtol=1e-14)
    assert f == 1.0
    assert R.rope_freqs(0, 1e4)[0].size == 0
    inv, _ = R.rope_freqs(64, 1e7, as_f32=True)  # as rbt_gqa_step_d rounds them
    e = (np.float32(-2.0) * np.arange(32, dtype=np.float32)) / np.float32(64)
    want = np.array([np.float32(math.pow(1e7, float(x))) for x in e])
    assert np.array_equal(inv, want.astype(np.float64))


def test_base_frequencies(rbt_lib):
    """The slowest pair is interpolated by the factor and the fastest kept."""
    import rabbit_amd as R
    plain = R.rope_freqs(128, 1e4)[0]
    inv, _ = R.rope_freqs(128, 1e4, kind=R.ROPE_BASE, factor=8.0)
    np.testing.assert_allclose(inv, (1e4 * 8.0 ** (128 / 126)) ** (-np.arange(0, 128, 2) / 128), rtol=1e-13)
    np.testing.assert_allclose(plain[[0, -1]] / inv[[0, -1]], [1.0, 8.0], rtol=1e-12)


def test_yarn_frequencies(rbt_lib):
    import rabbit_amd as R
    d, theta, s, ctx, bf, bs = 64, 1e4, 16.0, 4096, 32.0, 1.0
    inv, f = R.rope_freqs(d, theta, kind=R.ROPE_YARN, factor=s, orig_ctx=ctx, beta_fast=bf, beta_slow=bs)
    plain = theta ** (-np.arange(0, d, 2) / d)
    # pair j turns ctx * plain[j] / 2 pi times over the context: at least beta_fast turns keep their frequency,
    # at most beta_slow divide by s (the ramp's ends are rounded outwards to whole pairs)
    j = [d * math.log(ctx / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (bf, bs)]
    lo, hi = math.floor(j[0]), math.ceil(j[1])
    for k in range(d // 2):
        r = min(max((k - lo) / (hi - lo), 0.0), 1.0)
        assert inv[k] == pytest.approx(plain[k] * (1 - r) + plain[k] / s * r, rel=1e-13), k
    turns = ctx * plain / (2 * math.pi)
    assert np.allclose(inv[:lo + 1], plain[:lo + 1], rtol=1e-14) and (turns[:lo] >= bf).all()
    assert np.allclose(inv[hi:], plain[hi:] / s, rtol=1e-14) and (turns[hi:] <= bs).all()
    assert f == pytest.approx(0.1 * math.log(s) + 1.0, rel=1e-7)
    assert R.rope_freqs(d, theta, kind=R.ROPE_YARN, factor=s, orig_ctx=ctx, attn_factor=0.5)[1] == 0.5


def test_wavelength_frequencies(rbt_lib):
    import rabbit_amd as R
    d, theta, s, ctx, lo, hi = 128, 5e5, 8.0, 8192, 1.0, 4.0
    inv, f = R.rope_freqs(d, theta, kind=R.ROPE_WAVELENGTH, factor=s, orig_ctx=ctx, low_freq=lo, high_freq=hi)
    for k, w in enumerate(theta ** (-np.arange(0, d, 2) / d)):
        wave = 2 * math.pi / w
        mix = (ctx / wave - lo) / (hi - lo)
        want = w if wave < ctx / hi else w / s if wave > ctx / lo else (1 - mix) * w / s + mix * w
        assert inv[k] == pytest.approx(want, rel=1e-12), k
    assert f == 1.0


@pytest.mark.parametrize("kw", [dict(rope_dim=3), dict(rope_dim=2048), dict(theta=0.0), dict(theta=float("nan")), dict(kind=9),
                                dict(kind=1, factor=0.5), dict(kind=1, factor=float("inf")), dict(kind=2, factor=2.0, rope_dim=2),
                                dict(kind=3, factor=2.0), dict(kind=3, factor=2.0, orig_ctx=64, beta_fast=1.0, beta_slow=2.0),
                                dict(kind=4, factor=2.0, orig_ctx=64, low_freq=4.0, high_freq=4.0), dict(attn_factor=-1.0)])
def test_frequency_refusals(rbt_lib, kw):
    import rabbit_amd as R
    kw = {"rope_dim": 64, "theta": 1e4, **kw}
    with pytest.raises(R.RbtError) as e:
        R.rope_freqs(kw.pop("rope_dim"), kw.pop("theta"), **kw)
    assert e.value.status == RBT_E_INVALID


def _message(lib):
    return (lib.rbt_last_error(None) or b"").decode()


A = 1 << 20  # an address that is aligned; nothing reads it in a call that is refused


def _refused(lib, rc, status, text):
    assert rc == status and text in _message(lib), (rc, _message(lib))


def _part(**kw):
    d = dict(src=A, dst=2 * A, src_dtype=0, dst_dtype=0, n_heads=2, src_token_stride=128, src_head_stride=64,
             dst_token_stride=128, dst_head_stride=64, norm=None, rotate=1)
    d.update(kw)
    return abi.RbtRopePart(**d)


@pytest.mark.parametrize("desc,part,status,text", [
    (dict(layout=2), {}, RBT_E_INVALID, "layout"), (dict(head_dim=0), {}, RBT_E_UNSUPPORTED, "head_dim"),
    (dict(head_dim=1025), {}, RBT_E_UNSUPPORTED, "head_dim"), (dict(rope_dim=15), {}, RBT_E_INVALID, "rotated"),
    (dict(rope_start=60), {}, RBT_E_INVALID, "rotated"), (dict(rope_dim=66), {}, RBT_E_INVALID, "rotated"),
    (dict(factor=float("inf")), {}, RBT_E_INVALID, "factor"), (dict(eps=-1.0), {}, RBT_E_INVALID, "eps"),
    (dict(inv_freq=None), {}, RBT_E_INVALID, "inv_freq"), ({}, dict(src=None), RBT_E_INVALID, "null src"),
    ({}, dict(dst=None), RBT_E_INVALID, "null src"), ({}, dict(src_dtype=2), RBT_E_INVALID, "types"),
    ({}, dict(n_heads=0), RBT_E_INVALID, "heads"), ({}, dict(src=A + 2), RBT_E_INVALID, "aligned"),
    ({}, dict(dst=A + 1, dst_dtype=1), RBT_E_INVALID, "aligned"), ({}, dict(dst_head_stride=63), RBT_E_INVALID, "overlap"),
    ({}, dict(dst_token_stride=127), RBT_E_INVALID, "overlap"), ({}, dict(dst_token_stride=0), RBT_E_INVALID, "overlap"),
    ({}, dict(src_token_stride=1 << 41), RBT_E_INVALID, "stride")])
def test_rope_refusals(rbt_lib, desc, part, status, text):
    d = dict(layout=0, head_dim=64, rope_start=0, rope_dim=16, inv_freq=A, factor=1.0, angle_f32=0, eps=1e-6)
    d.update(desc)
    call = lambda dd, pp, n=1, pos=A, s=3: rbt_lib.rbt_rope_d(None, C.byref(dd), C.byref(pp), n, pos, s)  # noqa: E731
    _refused(rbt_lib, call(abi.RbtRopeDesc(**d), _part(**part)), status, text)


def test_rope_accepts(rbt_lib):
    """Calls that are right reach the check of the context: rows by heads or by tokens, sources that repeat."""
    d = abi.RbtRopeDesc(0, 64, 0, 16, A, 1.0, 0, 1e-6)
    for p in (_part(), _part(dst_token_stride=64, dst_head_stride=192), _part(src_token_stride=0, src_head_stride=0),
              _part(dst_dtype=1, dst=A + 2), _part(n_heads=1, dst_head_stride=0, dst_token_stride=64)):
        _refused(rbt_lib, rbt_lib.rbt_rope_d(None, C.byref(d), C.byref(p), 1, A, 3), RBT_E_INVALID, "null context")
    p = _part()
    _refused(rbt_lib, rbt_lib.rbt_rope_d(None, C.byref(d), C.byref(p), 1, None, 3), RBT_E_INVALID, "positions")
    _refused(rbt_lib, rbt_lib.rbt_rope_d(None, C.byref(d), C.byref(p), 9, A, 3), RBT_E_INVALID, "tensors")
    _refused(rbt_lib, rbt_lib.rbt_rope_d(None, None, C.byref(p), 1, A, 3), RBT_E_INVALID, "null descriptor")
    _refused(rbt_lib, rbt_lib.rbt_rope_d(None, C.byref(d), C.byref(p), 1, A, 1 << 24), RBT_E_UNSUPPORTED, "tokens")


@pytest.mark.parametrize("desc,args,status,text", [
    (dict(n_heads=6), {}, RBT_E_INVALID, "shape"), (dict(n_kv_heads=0), {}, RBT_E_INVALID, "shape"),
    (dict(n_heads=0), {}, RBT_E_INVALID, "shape"), (dict(head_dim=0), {}, RBT_E_UNSUPPORTED, "head_dim"),
    (dict(head_dim=1088), {}, RBT_E_UNSUPPORTED, "head_dim"), (dict(kv_dtype=3), {}, RBT_E_INVALID, "type"),
    (dict(attn_scale=float("nan")), {}, RBT_E_INVALID, "attn_scale"), (dict(attn_scale=3e38), {}, RBT_E_INVALID, "attn_scale"), (dict(cap=0), {}, RBT_E_INVALID, "rows"),
    (dict(max_len=101), {}, RBT_E_INVALID, "max_len"), (dict(gate_head_stride=1 << 41), dict(gate=A), RBT_E_INVALID, "stride"),
    ({}, dict(T=0), RBT_E_INVALID, "step"), ({}, dict(T=257), RBT_E_UNSUPPORTED, "nodes"), ({}, dict(B=65536), RBT_E_INVALID, "step"),
    ({}, dict(q=None), RBT_E_INVALID, "null"), ({}, dict(kd=None), RBT_E_INVALID, "null"), ({}, dict(out=None), RBT_E_INVALID, "null"),
    ({}, dict(parent=None), RBT_E_INVALID, "null"), ({}, dict(kc=A + 8), RBT_E_INVALID, "aligned"),
    ({}, dict(q=A + 4), RBT_E_INVALID, "aligned"), ({}, {}, RBT_E_INVALID, "null context")])
def test_gqa_tree_refusals(rbt_lib, desc, args, status, text):
    d = dict(n_heads=8, n_kv_heads=4, head_dim=64, attn_scale=0.125, kv_dtype=0, cap=100, max_len=0, gate_token_stride=0,
             gate_head_stride=0)
    d.update(desc)
    a = dict(B=2, T=3, q=A, kc=A, vc=A, kd=A, vd=A, len=A, n=A, parent=A, gate=None, out=A)
    a.update(args)
    _refused(rbt_lib, rbt_lib.rbt_gqa_tree_d(None, C.byref(abi.RbtGqaTreeDesc(**d)), *a.values()), status, text)


@pytest.mark.parametrize("args,status,text", [
    (dict(T=300), RBT_E_UNSUPPORTED, "nodes"), (dict(T=0), RBT_E_INVALID, "step"), (dict(B=1025), RBT_E_UNSUPPORTED, "sequences"),
    (dict(V=0), RBT_E_INVALID, "vocabulary"), (dict(p=None), RBT_E_INVALID, "null"), (dict(u=None), RBT_E_INVALID, "null"),
    (dict(next=None), RBT_E_INVALID, "null"), (dict(q=A + 2), RBT_E_INVALID, "aligned"), ({}, RBT_E_INVALID, "null context")])
def test_verify_refusals(rbt_lib, args, status, text):
    a = dict(B=2, T=3, V=50, children=0, tokens=A, parent=A, n=A, p=A, q=None, u=A, path=A, n_path=A, next=A)
    a.update(args)
    _refused(rbt_lib, rbt_lib.rbt_draft_verify_d(None, *a.values()), status, text)


@pytest.mark.parametrize("desc,args,status,text", [
    (dict(kv_dtype=2), {}, RBT_E_INVALID, "type"), (dict(n_kv_heads=0), {}, RBT_E_INVALID, "caches"),
    (dict(cap=0), {}, RBT_E_INVALID, "caches"), ({}, dict(T=257), RBT_E_UNSUPPORTED, "nodes"),
    ({}, dict(len_out=A), RBT_E_INVALID, "len_out"), ({}, dict(path=None), RBT_E_INVALID, "null"),
    ({}, dict(layer=None), RBT_E_INVALID, "layer 1"), ({}, dict(layer=A + 1), RBT_E_INVALID, "layer 1"),
    ({}, {}, RBT_E_INVALID, "null context")])
def test_commit_refusals(rbt_lib, desc, args, status, text):
    d = dict(n_layers=2, n_kv_heads=4, head_dim=64, kv_dtype=0, cap=100)
    d.update(desc)
    a = dict(T=3, path=A, n_path=A, len=A, len_out=2 * A)
    layer = args.pop("layer", A) if "layer" in args else A
    a.update(args)
    ptr = (C.c_void_p * 2)(A, layer)
    _refused(rbt_lib, rbt_lib.rbt_kv_commit_d(None, C.byref(abi.RbtKvCommitDesc(**d)), 2, a.pop("T"), ptr, ptr, ptr, ptr,
                                              *a.values()), status, text)


def test_positions_refusals(rbt_lib):
    _refused(rbt_lib, rbt_lib.rbt_tree_positions_d(None, 2, 257, A, A, A, A), RBT_E_UNSUPPORTED, "nodes")
    _refused(rbt_lib, rbt_lib.rbt_tree_positions_d(None, 2, 3, A, None, A, A), RBT_E_INVALID, "null tree buffer")
    _refused(rbt_lib, rbt_lib.rbt_tree_positions_d(None, 2, 3, A, A, A, A), RBT_E_INVALID, "null context")


def test_truth_forms_agree_with_closed_cases():
    """The 64-bit forms that the GPU tests compare with: a residual by hand, and a chain that is plain attention."""
    import draft_truth as T
    p = np.array([[[0.5, 0.25, 0.25, 0.0]] * 3], np.float32)
    q = np.array([[[0.25, 0.5, 0.0, 0.25]] * 3], np.float32)
    par, n = np.array([[-1, 0, 0]], np.int32), [3]
    u = np.array([[0.4, 0.51, 0.9]], np.float32)
    # token 1: 0.51 * 0.5 >= 0.25, rejected; the residual is [0.25, 0, 0.25, 0], its mass 0.5; token 0: the residual's
    # probability 0.5 over q's 0.25 is above 0.9, so it stands; then the draw from p after node 2
    path, m, x = T.verify(np.array([[0, 1, 0]]), par, n, p, q, u)
    assert path.tolist() == [[0, 2, -1]] and m.tolist() == [2] and x.tolist() == [0]
    # without q: token 1 rejected (0.51 >= 0.25), the rest's mass 0.75; token 2: 0.9 * 0.75 >= 0.25, rejected; left [0.5, 0, 0, 0]
    path, m, x = T.verify(np.array([[0, 1, 2]]), par, n, p, None, u)
    assert path.tolist() == [[0, -1, -1]] and x.tolist() == [0]
    rng = np.random.default_rng(0)
    qq, k, v = rng.standard_normal((1, 3, 2, 4)), rng.standard_normal((1, 8, 1, 4)), rng.standard_normal((1, 8, 1, 4))
    o, _, _ = T.tree_attention(qq, k[:, :5], v[:, :5], k[:, 5:], v[:, 5:], [5], [3], T.random_parents(rng, 1, 3, "chain"), 0.5)
    for i in range(3):
        s = np.exp(qq[0, i] @ k[0, :6 + i, 0].T * 0.5)
        assert np.allclose(o[0, i], s / s.sum(-1, keepdims=True) @ v[0, :6 + i, 0])


def test_bf16_parts_of_f32_products():
    """An fp32 number is its three parts; a product of two by six of the parts' nine products is off by 2^-24 (1 + 2^-6) of
    it at most, at the mantissas whose parts are longest and at the largest numbers too, and as much to either side."""
    import draft_truth as T
    rng = np.random.default_rng(0)
    man, few = rng.integers(0, 1 << 23, (2, 1 << 20)), rng.integers(0, 1 << 7, (2, 1 << 17)) << 16
    man[:, :1 << 16] = few[:, :1 << 16] | 0xffff        # parts by truncation are longest here
    man[:, 1 << 16:1 << 17] = few[:, 1 << 16:] | 0x7f80  # and rounded ones here
    for ex in (127, 17, 254):  # (below 2^-110 the last part is finer than bf16's subnormals)
        x, y = (((e << 23) | m).astype(np.uint32).view(np.float32) for e, m in zip((ex, 127), man))
        for v in (x, y):
            hi, mid, lo = (np.asarray(p, np.float64) for p in T.bf16_parts(v))
            v = v.astype(np.float64)
            assert np.array_equal(hi + mid + lo, v) and np.isfinite(hi).all()
            # (the factors: numbers past the largest bf16, whose first part is not the nearest)
            assert (np.abs(mid) <= 2.0 ** -8 * (1 + 2.0 ** -16) * v).all()
            assert (np.abs(lo) <= 2.0 ** -17 * (1 + 2.0 ** -7) * v).all()
        exact = x.astype(np.float64) * y.astype(np.float64)
        off = (T.six_products(x, y) - exact) / exact
        assert np.abs(off).max() <= T.U32 * (1 + 2.0 ** -6)
        assert abs(off.mean()) < 0.02 * T.U32


class _Tensor:
    """What the Python calls ask a device tensor, without a device."""

    is_cuda = True

    def __init__(self, *shape, dtype="float32", stride=None):
        self.shape, self.dtype = shape, "torch." + dtype
        self.strides = stride or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return self.strides[i]

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return A


def _no_gpu(lib):
    """A Context whose calls reach the library's checks and are refused there for want of a context."""
    import rabbit_amd as R
    c = R.Context.__new__(R.Context)
    c.lib, c.h, c._keep = lib, None, []
    return c


def test_rope_call_fits_its_parts(rbt_lib):
    """pos and head_dim agree with the tensors of every part; parts hold the tensors they point to."""
    import gc
    import weakref
    import rabbit_amd as R
    ctx, inv = _no_gpu(rbt_lib), _Tensor(16, dtype="float64")
    part = lambda s, hd: R.rope_part(_Tensor(s, 2, hd), _Tensor(s, 2, hd), norm=_Tensor(hd))  # noqa: E731
    pos = lambda *sh: _Tensor(*sh, dtype="int32")  # noqa: E731
    for parts, p, hd in (([part(5, 64)], pos(6), 64), ([part(5, 64)], pos(4), 64), ([part(5, 64), part(4, 64)], pos(5), 64),
                         ([part(5, 64)], pos(5), 128), ([part(5, 64)], pos(5), 32), ([part(5, 64), part(5, 32)], pos(5), 64)):
        with pytest.raises(ValueError):
            ctx.rope(parts, p, hd, inv, sync=False)
    with pytest.raises(TypeError):  # nothing is known of a bare struct's rows
        ctx.rope([_part()], pos(3), 64, inv, sync=False)
    for p in (pos(6), pos(2, 3)):  # right calls reach the library
        with pytest.raises(R.RbtError, match="null context"):
            ctx.rope([part(6, 64), part(6, 64)], p, 64, inv, sync=False)
    ts = [_Tensor(3, 2, 64), _Tensor(3, 2, 64), _Tensor(64)]
    p, refs = R.rope_part(ts[0], ts[1], norm=ts[2]), [weakref.ref(t) for t in ts]
    del ts
    gc.collect()
    assert all(r() is not None for r in refs)
    assert p.src == p.norm == A


def _attend_args(B, N, H, K, D, gate):
    i32 = lambda *sh: _Tensor(*sh, dtype="int32")  # noqa: E731
    return (_Tensor(B, N, H, D), _Tensor(B, 9, K, D), _Tensor(B, 9, K, D), _Tensor(B, N, K, D), _Tensor(B, N, K, D), i32(B),
            i32(B), i32(B, N), 0.125, _Tensor(B, N, H, D), gate)


@pytest.mark.parametrize("B,N,stride,ok", [
    (3, 1, (1024, 512, 128, 1), True),   # the first node's gates of q_proj rows with two nodes
    (3, 1, (512, 7, 128, 1), True),      # one node: the step from node to node is nobody's
    (1, 4, (7, 512, 128, 1), True),      # one sequence
    (3, 4, (2048, 512, 128, 1), True), (3, 4, (4096, 512, 128, 1), False), (3, 1, (512, 512, 128, 2), False)])
def test_gate_views(rbt_lib, B, N, stride, ok):
    """Gates inside wider rows: every view that two strides describe, no other."""
    import rabbit_amd as R
    ctx = _no_gpu(rbt_lib)
    with pytest.raises(R.RbtError if ok else ValueError, match="null context" if ok else "gate"):
        ctx.gqa_tree(*_attend_args(B, N, 4, 2, 64, _Tensor(B, N, 4, 64, stride=stride)), sync=False)


@pytest.mark.parametrize("B,args", [
    (2, dict(n_path=2 * A, path=3 * A, len=4 * A, len_out=2 * A)), (2, dict(n_path=2 * A, path=3 * A, len=4 * A, len_out=3 * A)),
    (2, dict(n_path=2 * A, path=3 * A, len=4 * A, len_out=3 * A + 20)), (2, dict(n_path=2 * A, path=3 * A, len=4 * A, len_out=4 * A - 4)),
    (2, dict(n_path=2 * A, path=3 * A, len=4 * A, len_out=4 * A + 4))])
def test_commit_refuses_lengths_over_its_inputs(rbt_lib, B, args):
    """len_out is written while other workgroups, and the launches of further layers, still read path, n_path and len."""
    d = abi.RbtKvCommitDesc(2, 4, 64, 0, 100)
    ptr = (C.c_void_p * 2)(A, A)
    call = lambda a: rbt_lib.rbt_kv_commit_d(None, C.byref(d), B, 3, ptr, ptr, ptr, ptr, a["path"], a["n_path"], a["len"],  # noqa: E731
                                             a["len_out"])
    _refused(rbt_lib, call(args), RBT_E_INVALID, "len_out")
    for free in (3 * A + 24, 3 * A - 8, 2 * A + 8, 4 * A + 8, 5 * A):  # beside them
        _refused(rbt_lib, call({**args, "len_out": free}), RBT_E_INVALID, "null context")
