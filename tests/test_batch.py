"""CPU checks of the batch step's entry points: every refusal of arguments (they are checked before the context, so a
call without one reaches them), and the 64-bit forms that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import batch_truth as BT
from rabbit_amd import abi
from rabbit_amd.abi import RBT_E_INVALID, RBT_E_UNSUPPORTED
from test_drafts import A, _no_gpu, _refused, _Tensor


def _rows(**kw):
    return abi.RbtKvRows(**{**dict(k=A, v=A, k_scale=A, v_scale=A), **kw})


@pytest.mark.parametrize("read", [False, True])
@pytest.mark.parametrize("desc,args,status,text", [
    (dict(n_kv_heads=0), {}, RBT_E_INVALID, "kv heads"), (dict(head_dim=0), {}, RBT_E_UNSUPPORTED, "head_dim"),
    (dict(head_dim=1025), {}, RBT_E_UNSUPPORTED, "head_dim"), (dict(cap=0), {}, RBT_E_INVALID, "rows"),
    (dict(cap=1 << 31), {}, RBT_E_INVALID, "rows"), (dict(dtype=2), {}, RBT_E_INVALID, "type"), (dict(dtype=8), {}, RBT_E_INVALID, "type"),
    (dict(row_stride=1 << 41), {}, RBT_E_INVALID, "stride"), ({}, dict(T=101), RBT_E_INVALID, "rows"), ({}, dict(B=65536), RBT_E_INVALID, "sequences"),
    ({}, dict(k=None), RBT_E_INVALID, "null"), ({}, dict(v=None), RBT_E_INVALID, "null"), ({}, dict(k=A + 2), RBT_E_INVALID, "aligned"),
    ({}, dict(len=A + 2), RBT_E_INVALID, "aligned"), ({}, dict(rows=None), RBT_E_INVALID, "null"),
    ({}, dict(rows=_rows(k=None)), RBT_E_INVALID, "null"), ({}, dict(rows=_rows(v_scale=None)), RBT_E_INVALID, "null"),
    ({}, dict(rows=_rows(k_scale=A + 1)), RBT_E_INVALID, "aligned"), ({}, {}, RBT_E_INVALID, "null context"),
    ({}, dict(T=0, k=None), RBT_E_INVALID, "null context"), ({}, dict(len=None, n=None), RBT_E_INVALID, "null context")])
def test_quant_refusals(rbt_lib, desc, args, status, text, read):
    d = dict(n_kv_heads=4, head_dim=64, cap=100, dtype=0, seq_stride=3 * 256, row_stride=256, head_stride=64)
    d.update(desc)
    a = dict(B=2, T=3, k=A, v=A, len=A, n=A, rows=_rows())
    a.update(args)
    rows = None if a["rows"] is None else C.byref(a["rows"])
    d = C.byref(abi.RbtKvQuantDesc(**d))
    rc = rbt_lib.rbt_kv_dequant_d(None, d, a["B"], a["T"], rows, a["len"], a["n"], a["k"], a["v"]) if read else \
        rbt_lib.rbt_kv_quant_d(None, d, a["B"], a["T"], a["k"], a["v"], a["len"], a["n"], rows)
    _refused(rbt_lib, rc, status, text)


@pytest.mark.parametrize("strides,ok", [((768, 256, 64), True), ((767, 256, 64), False), ((768, 255, 64), False), ((768, 256, 63), False),
                                        ((64, 128, 3 * 128), True), ((64, 128, 3 * 128 - 1), False), ((0, 256, 64), False)])
def test_read_back_refuses_overlapping_rows(rbt_lib, strides, ok):
    """Results may lie in any order of their axes, not over each other. Sources may repeat."""
    d = abi.RbtKvQuantDesc(4, 64, 100, 0, *strides)
    rows = _rows()
    _refused(rbt_lib, rbt_lib.rbt_kv_dequant_d(None, C.byref(d), 2, 3, C.byref(rows), A, A, A, A), RBT_E_INVALID,
             "null context" if ok else "overlap")
    _refused(rbt_lib, rbt_lib.rbt_kv_quant_d(None, C.byref(d), 2, 3, A, A, A, A, C.byref(rows)), RBT_E_INVALID, "null context")


@pytest.mark.parametrize("desc,args,status,text", [
    (dict(n_heads=6), {}, RBT_E_INVALID, "shape"), (dict(n_kv_heads=0), {}, RBT_E_INVALID, "shape"),
    (dict(head_dim=0), {}, RBT_E_UNSUPPORTED, "head_dim"), (dict(head_dim=1025), {}, RBT_E_UNSUPPORTED, "head_dim"),
    (dict(kv_dtype=2), {}, RBT_E_INVALID, "type"), (dict(attn_scale=float("inf")), {}, RBT_E_INVALID, "attn_scale"),
    (dict(cap=0), {}, RBT_E_INVALID, "rows"), (dict(max_len=101), {}, RBT_E_INVALID, "max_len"),
    (dict(prefix_cap=0), {}, RBT_E_INVALID, "prefixes"), (dict(max_prefix=51), {}, RBT_E_INVALID, "max_prefix"),
    (dict(gate_token_stride=1 << 41), dict(gate=A), RBT_E_INVALID, "stride"), ({}, dict(T=0), RBT_E_INVALID, "step"),
    ({}, dict(T=257), RBT_E_UNSUPPORTED, "nodes"), ({}, dict(B=65536), RBT_E_INVALID, "step"), ({}, dict(G=1025), RBT_E_UNSUPPORTED, "prefixes"),
    ({}, dict(B=65535, T=9), RBT_E_UNSUPPORTED, "too many"), ({}, dict(q=None), RBT_E_INVALID, "null"), ({}, dict(out=None), RBT_E_INVALID, "null"),
    ({}, dict(len=None), RBT_E_INVALID, "null"), ({}, dict(n=None), RBT_E_INVALID, "null"), ({}, dict(plen=None), RBT_E_INVALID, "null"),
    ({}, dict(first=None), RBT_E_INVALID, "null"), ({}, dict(q=A + 4), RBT_E_INVALID, "aligned"), ({}, dict(gate=A + 2), RBT_E_INVALID, "aligned"),
    ({}, dict(cache=None), RBT_E_INVALID, "null cache"), ({}, dict(prefix=None), RBT_E_INVALID, "null prefix"),
    ({}, dict(draft=_rows(v=None)), RBT_E_INVALID, "null draft"), ({}, dict(prefix=_rows(k=A + 8)), RBT_E_INVALID, "prefix rows must"),
    (dict(kv_dtype=8), dict(cache=_rows(k_scale=None)), RBT_E_INVALID, "null cache"),
    (dict(kv_dtype=8), dict(draft=_rows(k_scale=A + 2)), RBT_E_INVALID, "draft scales"), ({}, {}, RBT_E_INVALID, "null context"),
    ({}, dict(parent=None, draft=None, gate=None), RBT_E_INVALID, "null context"),
    (dict(prefix_cap=0), dict(G=0, plen=None, first=None, prefix=None), RBT_E_INVALID, "null context"),
    ({}, dict(cache=_rows(k_scale=None, v_scale=A + 1)), RBT_E_INVALID, "null context")])
def test_prefix_refusals(rbt_lib, desc, args, status, text):
    d = dict(n_heads=8, n_kv_heads=4, head_dim=64, attn_scale=0.125, kv_dtype=0, cap=100, max_len=0, prefix_cap=50, max_prefix=0,
             gate_token_stride=0, gate_head_stride=0)
    d.update(desc)
    a = dict(B=2, T=3, G=2, q=A, prefix=_rows(), cache=_rows(), draft=_rows(), plen=A, first=A, len=A, n=A, parent=A, gate=None, out=A)
    a.update(args)
    for r in ("prefix", "cache", "draft"):
        a[r] = None if a[r] is None else C.byref(a[r])
    _refused(rbt_lib, rbt_lib.rbt_gqa_prefix_d(None, C.byref(abi.RbtGqaPrefixDesc(**d)), *a.values()), status, text)


@pytest.mark.parametrize("desc,args,status,text", [
    (dict(vocab=0), {}, RBT_E_INVALID, "vocabulary"), (dict(vocab=(1 << 24) + 1, row_stride=1 << 25), {}, RBT_E_UNSUPPORTED, "vocabulary"),
    (dict(row_stride=49), {}, RBT_E_INVALID, "apart"), (dict(row_stride=1 << 41), {}, RBT_E_INVALID, "apart"),
    (dict(logits_dtype=8), {}, RBT_E_INVALID, "type"), ({}, dict(n=65536), RBT_E_INVALID, "rows"), ({}, dict(x=None), RBT_E_INVALID, "null"),
    ({}, dict(u=None), RBT_E_INVALID, "null"), ({}, dict(tok=None), RBT_E_INVALID, "null"), ({}, dict(x=A + 2), RBT_E_INVALID, "aligned"),
    ({}, dict(p=A + 1), RBT_E_INVALID, "aligned"), ({}, {}, RBT_E_INVALID, "null context"), ({}, dict(n=0, x=None), RBT_E_INVALID, "null context")])
def test_sample_refusals(rbt_lib, desc, args, status, text):
    d = dict(vocab=50, row_stride=50, logits_dtype=0)
    d.update(desc)
    a = dict(n=3, x=A, temp=None, k=None, top_p=None, min_p=None, u=A, tok=A, p=None)
    a.update(args)
    _refused(rbt_lib, rbt_lib.rbt_sample_d(None, C.byref(abi.RbtSampleDesc(**d)), *a.values()), status, text)


def test_other_calls_refuse_8bit_rows(rbt_lib):
    """8-bit rows carry scales, which rotation and tree attention do not take; the commit moves them."""
    d = abi.RbtGqaTreeDesc(8, 4, 64, 0.125, abi.DT_I8, 100, 0, 0, 0)
    _refused(rbt_lib, rbt_lib.rbt_gqa_tree_d(None, C.byref(d), 2, 3, A, A, A, A, A, A, A, A, None, A), RBT_E_INVALID, "type")
    ptr = (C.c_void_p * 1)(A + 1)
    d = abi.RbtKvCommitDesc(1, 4, 63, abi.DT_I8, 100)
    _refused(rbt_lib, rbt_lib.rbt_kv_commit_d(None, C.byref(d), 2, 3, ptr, ptr, ptr, ptr, A, A, A, 2 * A), RBT_E_INVALID, "null context")


def test_python_calls_fit_their_tensors(rbt_lib):
    """Shapes and types that disagree are refused before the library; right ones reach it."""
    import rabbit_amd as R
    ctx = _no_gpu(rbt_lib)
    i32 = lambda *s: _Tensor(*s, dtype="int32")  # noqa: E731
    cache8 = lambda B=2, cap=9, K=2, D=64, **kw: (_Tensor(B, cap, K, D, dtype="int8"), _Tensor(B, cap, K, D, dtype=kw.get("v", "int8")),  # noqa: E731
                                                  _Tensor(B, cap, K), _Tensor(B, cap, K))
    x = _Tensor(2, 3, 2, 64)
    for k, v, c, kw in ((x, _Tensor(2, 3, 2, 63), cache8(), {}), (x, _Tensor(2, 3, 2, 64, dtype="bfloat16"), cache8(), {}), (x, x, cache8(K=3), {}),
                        (x, x, cache8(v="float32"), {}), (x, x, cache8()[:2], {}), (x, x, cache8(), dict(length=i32(3))),
                        (x, _Tensor(2, 3, 2, 64, stride=(384, 128, 32, 1)), cache8(), {}),
                        (_Tensor(2, 3, 2, 64, stride=(384, 128, 64, 2)), _Tensor(2, 3, 2, 64, stride=(384, 128, 64, 2)), cache8(), {})):
        with pytest.raises(ValueError):
            ctx.kv_quant(k, v, c, sync=False, **kw)
        with pytest.raises(ValueError):
            ctx.kv_dequant(c, k, v, sync=False, **kw)
    with pytest.raises(R.RbtError, match="null context"):
        ctx.kv_quant(x, x, cache8(), length=i32(2), n_rows=i32(2), sync=False)
    q, out = _Tensor(2, 1, 4, 64), _Tensor(2, 1, 4, 64)
    pre = dict(prefix=cache8(3, 20), prefix_len=i32(3), prefix_first=i32(4))
    with pytest.raises(R.RbtError, match="null context"):
        ctx.gqa_prefix(q, cache8(), i32(2), i32(2), 0.1, out, sync=False, **pre)
    for kw in ({**pre, "prefix_first": i32(3)}, {**pre, "prefix": cache8(3, 20)[:2]}, {**pre, "prefix": cache8(3, 20, K=4)},
               dict(draft=cache8(2, 2)), dict(parent=i32(2, 2)), dict(gate=_Tensor(2, 1, 4, 63))):
        with pytest.raises(ValueError):
            ctx.gqa_prefix(q, cache8(), i32(2), i32(2), 0.1, out, sync=False, **kw)
    lg, tok, u = _Tensor(5, 99, stride=(128, 1)), i32(5), _Tensor(5)
    with pytest.raises(R.RbtError, match="null context"):
        ctx.sample(lg, u, tok, top_k=i32(5), probs=_Tensor(5, 99), sync=False)
    for kw in (dict(top_k=_Tensor(5)), dict(temperature=_Tensor(4)), dict(probs=_Tensor(5, 98))):
        with pytest.raises(ValueError):
            ctx.sample(lg, u, tok, sync=False, **kw)
    with pytest.raises(ValueError):
        ctx.sample(_Tensor(5, 99, stride=(198, 2)), u, tok, sync=False)


def test_truth_quantise_by_hand():
    q, s = BT.quantise(np.array([[254.0, -127.0, 1.0, 3.0], [0, 0, 0, 0], [1, np.nan, 2, 3], [1e-45, 0, 0, 0]], np.float32))
    # scale 2: 1 / 2 and 3 / 2 go to the even neighbour
    assert q.tolist() == [[127, -64, 0, 2], [0, 0, 0, 0], [0, 0, 0, 0], [0, 0, 0, 0]]
    assert s[0] == 2.0 and s[1] == 0.0 and np.isnan(s[2]) and s[3] == 0.0
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    q, s = BT.quantise(x)
    assert (np.abs(BT.values(q, s) - x) <= s[:, None] * (0.5 + 2.0 ** -16)).all() and (np.abs(q).max(-1) == 127).all()


def test_truth_sample_by_hand():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3], np.float64))
    tok, p, _ = BT.sample(x, 0.45)
    assert tok == 1 and np.allclose(p, [0.1, 0.4, 0.2, 0.3])
    tok, p, _ = BT.sample(x, 0.6, k=2)
    assert tok == 3 and np.allclose(p, [0, 4 / 7, 0, 3 / 7])
    tok, p, _ = BT.sample(x, 0.6, top_p=0.75)  # 0.4 + 0.3 do not reach it
    assert np.allclose(p, [0, 4 / 9, 2 / 9, 3 / 9]) and tok == 2
    assert np.allclose(BT.sample(x, 0.6, min_p=0.6)[1], [0, 4 / 7, 0, 3 / 7])
    assert np.allclose(BT.sample(x, 0.6, k=3, top_p=0.7)[1], [0, 4 / 7, 0, 3 / 7])  # of what top-k left
    assert BT.sample(x, 0.99, t=0)[0] == 1 and BT.sample(np.full(4, -np.inf), 0.5)[0] == -1


def test_truth_prefix_attention_is_attention_over_the_joined_rows():
    rng = np.random.default_rng(1)
    B, N, H, K, D = 3, 2, 4, 2, 8
    q = rng.standard_normal((B, N, H, D))
    kc, vc, kp, vp = (rng.standard_normal((n, c, K, D)) for n, c in ((B, 6), (B, 6), (1, 5), (1, 5)))
    par = np.array([[-1, 0]] * B, np.int32)
    o, _, _, _ = BT.prefix_attention(q, kc, vc, None, None, [3, 0, 4], [2, 1, 2], par, 0.5, kp, vp, [5], [1, 3])
    for b, n in ((0, 3), (1, 0), (2, 4)):
        for i in range((2, 1, 2)[b]):
            for h in range(H):
                k = np.concatenate([kp[0, :, h // 2]] * (b > 0) + [kc[b, :n + i + 1, h // 2]])
                v = np.concatenate([vp[0, :, h // 2]] * (b > 0) + [vc[b, :n + i + 1, h // 2]])
                s = np.exp(k @ q[b, i, h] * 0.5)
                assert np.allclose(o[b, i, h], s / s.sum() @ v)
