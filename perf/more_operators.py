"""Performance cases of a batch's decode step, through its public entry points (include/rabbit_amd.h).

A server that decodes a batch of users calls, per attention layer, the quantisation of the new keys and values into
an 8-bit cache and the attention over the cache, whose first rows (a system prompt, a document) many users may share,
and once per step the draw of the next tokens from the logits. The kinds:

    attend   rbt_gqa_prefix_d: tokens (or trees of drafted ones) of a batch over shared prefixes and their own caches
    quant    rbt_kv_quant_d and rbt_kv_dequant_d: rows into an 8-bit cache, and as the cache then holds them
    read     rbt_kv_dequant_d: rows of an 8-bit cache for a program that wants them in bf16
    sample   rbt_sample_d: tokens, and probabilities, from logits by temperature, top-k, top-p and min-p

Where `own` is false, run() computes them in elementary torch operations.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DEV = "cuda"


def listed():
    # The attention layers of the repository's own mixer workload: 64 query heads over 4 KV heads of 256.
    return [
        # a chat service: eight users behind a short system prompt, one new token each. The smallest: latency
        {"name": "attend_chat8_1500", "kind": "attend", "kv": "bf16", "heads": 64, "kv_heads": 4, "dim": 256, "seqs": 8,
         "nodes": 1, "prefix": 1500, "groups": 1, "len": 300, "tree": False, "gate": True},
        # a large batch behind a long system prompt with its tools and examples
        {"name": "attend_system64_8192", "kind": "attend", "kv": "bf16", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 64, "nodes": 1, "prefix": 8192, "groups": 1, "len": 512, "tree": False, "gate": True},
        # questions about one long document, kept in 8 bits
        {"name": "attend_document32_32749_i8", "kind": "attend", "kv": "i8", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 32, "nodes": 1, "prefix": 32749, "groups": 1, "len": 1000, "tree": False, "gate": True},
        # users with nothing in common, long conversations in 8 bits: plain batch decoding
        {"name": "attend_batch16_8192_i8", "kind": "attend", "kv": "i8", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 16, "nodes": 1, "prefix": 0, "groups": 0, "len": 8192, "tree": False, "gate": True},
        # odd everything: five query heads per KV head, head_dim 128, f32 rows, three prompts of different lengths, one
        # user without any, trees of drafted tokens, no gate
        {"name": "attend_odd11_1001_f32", "kind": "attend", "kv": "f32", "heads": 20, "kv_heads": 4, "dim": 128,
         "seqs": 11, "nodes": 5, "prefix": 1001, "groups": 3, "len": 333, "tree": True, "gate": False},
        # the new token's keys and values: the smallest
        {"name": "quant_token", "kind": "quant", "src": "f32", "kv_heads": 4, "dim": 256, "seqs": 1, "rows": 1,
         "cap": 1024, "ragged": False, "wide": False},
        # long prompts of a batch, bf16 rows inside the projection's q, k, v rows
        {"name": "quant_prompts4_4095", "kind": "quant", "src": "bf16", "kv_heads": 4, "dim": 256, "seqs": 4,
         "rows": 4095, "cap": 4352, "ragged": True, "wide": True},
        # a short conversation read back: latency
        {"name": "read_chat_77", "kind": "read", "kv_heads": 8, "dim": 128, "seqs": 1, "rows": 77, "cap": 512},
        # a batch's long caches read back
        {"name": "read_batch16_8192", "kind": "read", "kv_heads": 4, "dim": 256, "seqs": 16, "rows": 8192, "cap": 8200},
        # one user's next token: latency
        {"name": "sample_token_32000", "kind": "sample", "rows": 1, "vocab": 32000, "type": "f32", "temp": 0.8,
         "top_k": 40, "top_p": 0.95, "min_p": 0.0, "mixed": False, "probs": False},
        # a large batch, every user with settings of their own, large vocabulary
        {"name": "sample_batch64_131072", "kind": "sample", "rows": 64, "vocab": 131072, "type": "f32", "temp": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.02, "mixed": True, "probs": False},
        # the rows of drafted trees, whose probabilities the verification wants; bf16 logits, odd vocabulary
        {"name": "sample_nodes96_100003", "kind": "sample", "rows": 96, "vocab": 100003, "type": "bf16", "temp": 0.7,
         "top_k": 200, "top_p": 0.98, "min_p": 0.0, "mixed": False, "probs": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "quant", "read", "sample", "sample", "sample"])
    if kind == "attend":
        heads, kv_heads, dim = rng.choice([(64, 4, 256), (64, 4, 256), (20, 4, 128), (16, 2, 64), (32, 8, 128), (48, 3, 192),
                                           (12, 12, 64), (6, 2, 80)])
        seqs, nodes = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 12])
        groups = rng.choice([0, 1, 1, 2, 3, 5])
        groups = min(groups, max(1, seqs - 1))
        if dim == 80:  # head dims outside the matrix cores' tiles
            seqs, nodes, most, own_most = min(seqs, 6), min(nodes, 5), 500, 200
        else:
            most = max(64, min(32749, 32 * 32749 // (seqs * nodes), 32 * 32749 // max(1, 8 * groups)))
            own_most = max(64, min(8192, 16 * 8192 // seqs // (1 if nodes < 5 else 4)))
        return {"kind": kind, "kv": rng.choice(["bf16", "f32", "i8", "i8"]), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "seqs": seqs, "nodes": nodes, "prefix": _log_int(rng, 64, most) if groups else 0, "groups": groups,
                "len": _log_int(rng, 1, own_most), "tree": rng.random() < 0.5, "gate": rng.random() < 0.5}
    if kind in ("quant", "read"):
        kv_heads, dim = rng.choice([(4, 256), (8, 128), (1, 192), (2, 64), (3, 80), (5, 33)])
        seqs = _log_int(rng, 1, 16)
        rows = _log_int(rng, 1, min(4095, 16384 // seqs))
        case = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "seqs": seqs, "rows": rows, "cap": rows + rng.choice([1, 9, 500])}
        if kind == "quant":
            case.update(src=rng.choice(["f32", "bf16"]), ragged=rng.random() < 0.5, wide=rng.random() < 0.5)
        return case
    rows = _log_int(rng, 1, 64)
    return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 1000, 131072), "type": rng.choice(["f32", "bf16"]),
            "temp": rng.choice([0.0, 0.6, 1.0, 1.3]), "top_k": rng.choice([0, 1, 20, 50, 700]),
            "top_p": rng.choice([1.0, 0.95, 0.8]), "min_p": rng.choice([0.0, 0.0, 0.05]), "mixed": rng.random() < 0.4,
            "probs": rng.random() < 0.4}


# ---- what a program has in hand -------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _f32(v):
    return torch.tensor(v, dtype=torch.float32, device=DEV)


def _spread(n, hi, lo):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * b // max(1, n - 1) for b in range(n)]


def _lengths(case):
    """Own rows of the sequences: the longest first, the others down to half (short ones down to none)."""
    n = case["len"]
    return _spread(case["seqs"], n, n // 2 if n > 2048 or case["seqs"] == 1 else 0)


def _counts(case):
    """Nodes of the sequences: all of them first, the others down to half."""
    return _spread(case["seqs"], case["nodes"], (case["nodes"] + 1) // 2)


def _prefixes(case):
    """The prefixes' lengths, and the first sequence of each (and one past the last): with several prefixes the
    groups differ in size and the last sequence has none."""
    G, S = case["groups"], case["seqs"]
    if G == 0:
        return [], [0]
    last = S - 1 if G > 1 and S > G else S
    return _spread(G, case["prefix"], (case["prefix"] + 1) // 2), [last * i * (i + 1) // (G * (G + 1)) for i in range(G + 1)]


def _parents(case, seed):
    """parent[b, i] < i; node 0 is the root. Chains, or trees whose nodes hang from one of the last eight."""
    B, T = case["seqs"], case["nodes"]
    r = np.random.default_rng(seed)
    par = np.full((B, T), -1, np.int32)
    for i in range(1, T):
        par[:, i] = r.integers(max(0, i - 8), i, B) if case["tree"] else i - 1
    return _i32(par)


def _quantised(x):
    """Rows [.., D] as (int8 entries, f32 scales [..])."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = top / torch.full_like(top, 127.0)  # (a division by a plain number may multiply by its reciprocal)
    return torch.where(scale[..., None] > 0, torch.round(x / scale[..., None]), torch.zeros_like(x)).to(torch.int8), scale


def _rows(g, kv, *shape):
    """Keys or values as a cache holds them: {"x"} or {"x", "scale"}."""
    x = _normal(g, *shape)
    if kv == "i8":
        x, scale = _quantised(x)
        return {"x": x, "scale": scale.contiguous()}
    return {"x": x.to(torch.bfloat16) if kv == "bf16" else x}


def _attend(case, seed):
    g, B, T, H, K, D = _gen(seed), case["seqs"], case["nodes"], case["heads"], case["kv_heads"], case["dim"]
    cap, G, P = case["len"] + 8, case["groups"], case["prefix"]
    lens, first = _prefixes(case)
    s = {"q": _normal(g, B, T, H, D), "len": _i32(_lengths(case)), "n": _i32(_counts(case)), "parent": _parents(case, seed),
         "out": torch.zeros(B, T, H, D, device=DEV), "prefix_len": _i32(lens), "first": _i32(first)}
    for side in "kv":
        s[side + "c"] = _rows(g, case["kv"], B, cap, K, D)
        s[side + "d"] = _rows(g, case["kv"], B, T, K, D)
        s[side + "p"] = _rows(g, case["kv"], G, P, K, D) if G else None
    s["gate"] = _normal(g, B, T, H, D) if case["gate"] else None
    return s


def _row_counts(case):
    n = case["rows"]
    return _spread(case["seqs"], n, (n + 1) // 2) if case["ragged"] else [n] * case["seqs"]


def _quant(case, seed):
    g, B, T, K, D, cap = _gen(seed), case["seqs"], case["rows"], case["kv_heads"], case["dim"], case["cap"]
    t = torch.bfloat16 if case["src"] == "bf16" else torch.float32
    # wide: rows [q, k, v] of a fused projection, as many query heads as 4 per KV head
    rows = _normal(g, B, T, (6 if case["wide"] else 2) * K, D)
    rows *= torch.exp(_normal(g, B, T, 1, 1))  # rows of different sizes
    rows = rows.to(t)
    s = {"rows": rows, "k": rows[:, :, -2 * K:-K], "v": rows[:, :, -K:], "n": _i32(_row_counts(case)),
         "len": _i32(np.random.default_rng(seed).integers(0, cap - T + 1, B).astype(np.int32))}
    for side in "kv":
        s[side + "c"] = {"x": torch.zeros(B, cap, K, D, dtype=torch.int8, device=DEV),
                         "scale": torch.zeros(B, cap, K, device=DEV)}
        s[side + "o"] = torch.zeros(B, T, K, D, device=DEV)
    return s


def _read(case, seed):
    g, B, T, K, D, cap = _gen(seed), case["seqs"], case["rows"], case["kv_heads"], case["dim"], case["cap"]
    s = {"n": _i32([T] * B), "len": _i32(np.random.default_rng(seed).integers(0, cap - T + 1, B).astype(np.int32))}
    for side in "kv":
        s[side + "c"] = {"x": torch.randint(-127, 128, (B, cap, K, D), dtype=torch.int8, device=DEV, generator=g),
                         "scale": torch.rand(B, cap, K, device=DEV, generator=g) * 0.05}
        s[side + "o"] = torch.zeros(B, T, K, D, dtype=torch.bfloat16, device=DEV)
    return s


def _settings(case):
    """Temperature, top-k, top-p and min-p of each row; mixed: users with settings of their own."""
    n, base = case["rows"], (case["temp"], case["top_k"], case["top_p"], case["min_p"])
    if not case["mixed"]:
        return [[v] * n for v in base]
    some = [base, (0.7, 50, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 0.95, 0.05), base, (0.9, 0, 0.7, 0.0)]
    return [list(v) for v in zip(*[some[i % len(some)] for i in range(n)])]


def _sample(case, seed):
    g, n, V = _gen(seed), case["rows"], case["vocab"]
    # a few tokens hold most of the mass, as a language model's rows do
    x = 2.5 * _normal(g, n, V)
    x += torch.where(torch.rand(n, V, device=DEV, generator=g) < 30.0 / V, 12.0, 0.0)
    t, k, p, m = _settings(case)
    return {"x": x.to(torch.bfloat16) if case["type"] == "bf16" else x, "temp": _f32(t), "top_k": _i32(k), "top_p": _f32(p),
            "min_p": _f32(m), "u": torch.rand(n, device=DEV, generator=g),
            "tok": torch.zeros(n, dtype=torch.int32, device=DEV),
            "p": torch.zeros(n, V, device=DEV) if case["probs"] else None}


_MAKE = {"attend": _attend, "quant": _quant, "read": _read, "sample": _sample}


def prepare(case, seed):
    s = _MAKE[case["kind"]](case, seed)
    s["case"] = case
    torch.cuda.synchronize()  # the inputs were made on torch's stream
    return s


# ---- the plain forms --------------------------------------------------------------------------------
def _values(rows):
    x = rows["x"].float()
    return x * rows["scale"][..., None] if "scale" in rows else x


def _plain_attend(s):
    c = s["case"]
    B, T, H, K, D, G = c["seqs"], c["nodes"], c["heads"], c["kv_heads"], c["dim"], c["groups"]
    L, R, scale = c["len"], H // K, 1.0 / math.sqrt(D)
    k = torch.cat([_values(s["kc"])[:, :L], _values(s["kd"])], 1).permute(0, 2, 3, 1)      # [B, K, D, keys]
    v = torch.cat([_values(s["vc"])[:, :L], _values(s["vd"])], 1).permute(0, 2, 1, 3)      # [B, K, keys, D]
    q = s["q"].view(B, T, K, R, D).permute(0, 2, 1, 3, 4).reshape(B, K, T * R, D)
    idx = torch.arange(T, device=DEV)
    step = (s["parent"][:, :, None] == idx).double() + torch.eye(T, dtype=torch.float64, device=DEV)
    above = torch.linalg.matrix_power(step, max(1, T - 1)) > 0                             # node i sees node j
    old = torch.arange(L, device=DEV) < s["len"][:, None]
    sees = torch.cat([old[:, None, :].expand(B, T, L), above], 2)                          # [B, T, keys]
    a = torch.matmul(q, k).view(B, K, T, R, -1) * scale
    a = a.masked_fill(~sees[:, None, :, None, :], -math.inf).view(B, K, T * R, -1)
    m = a.amax(-1, keepdim=True)
    if G:
        # the sequences of each prefix side by side, so that its rows meet all of them in one product
        P, first = c["prefix"], s["first"].long()
        b = torch.arange(B, device=DEV)
        grp = (b[:, None] >= first[None, 1:]).sum(1)                                       # G: has no prefix
        has, grp = grp < G, grp.clamp(max=G - 1)
        M = max(y - x for x, y in zip(_prefixes(c)[1], _prefixes(c)[1][1:]))
        at = (b - first[grp]).clamp(min=0, max=M - 1)
        qg = torch.zeros(G, M, K, T * R, D, device=DEV)
        qg[grp[has], at[has]] = q[has]
        qg = qg.permute(0, 2, 1, 3, 4).reshape(G, K, M * T * R, D)
        kp, vp = _values(s["kp"]).permute(0, 2, 3, 1), _values(s["vp"]).permute(0, 2, 1, 3)
        e = torch.matmul(qg, kp) * scale
        e = e.masked_fill((torch.arange(P, device=DEV) >= s["prefix_len"][:, None])[:, None, None, :], -math.inf)
        of_seq = lambda t: t.view(G, K, M, T * R, -1).permute(0, 2, 1, 3, 4)[grp, at]      # noqa: E731
        me = e.amax(-1, keepdim=True)
        m = torch.where(has[:, None, None, None], torch.maximum(m, of_seq(me)), m)
        mg = torch.full((G, M, K, T * R, 1), math.inf, device=DEV)
        mg[grp[has], at[has]] = m[has]
        e = torch.exp(e - mg.permute(0, 2, 1, 3, 4).reshape(G, K, M * T * R, 1))
        le, oe = of_seq(e.sum(-1, keepdim=True)), of_seq(torch.matmul(e, vp))
    a = torch.exp(a - m)
    l, o = a.sum(-1, keepdim=True), torch.matmul(a, v)
    if G:
        keep = has[:, None, None, None]
        l, o = torch.where(keep, l + le, l), torch.where(keep, o + oe, o)
    o = (o / l).view(B, K, T, R, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    if s["gate"] is not None:
        o = o * (1.0 / (1.0 + torch.exp(-s["gate"])))
    return torch.where((idx < s["n"][:, None])[:, :, None, None], o, s["out"])


def _slots(s):
    c = s["case"]
    j = torch.arange(c["rows"], device=DEV)
    live = j < s["n"][:, None]
    b = torch.arange(c["seqs"], device=DEV)[:, None].expand_as(live)
    return live, b[live], (s["len"][:, None] + j)[live].long(), j.expand_as(live)[live]


def _plain_read(s):
    live, b, at, j = _slots(s)
    out = {}
    for side in "kv":
        o, c = s[side + "o"], s[side + "c"]
        o[b, j] = (c["x"][b, at].float() * c["scale"][b, at][..., None]).to(o.dtype)
        out[side] = o
    return out


def _plain_quant(s):
    live, b, at, j = _slots(s)
    for side in "kv":
        c = s[side + "c"]
        c["x"][b, at], c["scale"][b, at] = _quantised(s[side][b, j])
    return {**_plain_read(s), "k_scale": s["kc"]["scale"], "v_scale": s["vc"]["scale"]}


def _plain_sample(s):
    x, V = s["x"].double(), s["x"].shape[1]
    greedy = (s["temp"] == 0)[:, None]
    t = torch.where(greedy, 1.0, s["temp"].double()[:, None])
    srt, idx = torch.sort(x, dim=-1, descending=True, stable=True)  # equal logits: the lower index first
    w = torch.exp((srt - srt[:, :1]) / t)
    rank = torch.arange(V, device=DEV)
    k = torch.where(greedy, 1, s["top_k"].long()[:, None])
    w = torch.where((rank < k) | (k == 0), w, 0.0)
    cum = torch.cumsum(w, -1)
    top_p = s["top_p"].double()[:, None]
    keep = (cum - w < top_p * cum[:, -1:]) | (top_p >= 1.0) | (rank == 0)
    keep = keep & (w >= s["min_p"].double()[:, None])
    w = torch.where(keep, w, 0.0)
    p = torch.zeros_like(w).scatter_(1, idx, w / w.sum(-1, keepdim=True))
    cum = torch.cumsum(p, -1)
    tok = (cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(-1).to(torch.int32)
    return {"tok": tok} if s["p"] is None else {"tok": tok, "p": p.float()}


_PLAIN = {"attend": _plain_attend, "quant": _plain_quant, "read": _plain_read, "sample": _plain_sample}


# ---- the framework's calls ----------------------------------------------------------------------------
_CTX = None


def _context():
    global _CTX
    if _CTX is None:
        import rabbit_amd as R
        _CTX = R.Context(0)
    return _CTX


def _call(s):
    """The state's device calls as [(entry point, its arguments)], and their outputs."""
    import rabbit_amd as R
    from rabbit_amd import abi
    ctx, c, p = _context(), s["case"], lambda t: None if t is None else t.data_ptr()
    if c["kind"] == "attend":
        kinds = {"bf16": R.DT_BF16, "f32": R.DT_F32, "i8": R.DT_I8}
        d = abi.RbtGqaPrefixDesc(c["heads"], c["kv_heads"], c["dim"], 1.0 / math.sqrt(c["dim"]), kinds[c["kv"]],
                                 c["len"] + 8, c["len"], c["prefix"], c["prefix"], c["heads"] * c["dim"], c["dim"])
        rows = [None if s["k" + x] is None else
                abi.RbtKvRows(p(s["k" + x]["x"]), p(s["v" + x]["x"]), p(s["k" + x].get("scale")), p(s["v" + x].get("scale")))
                for x in "pcd"]
        refs = [None if r is None else C.byref(r) for r in rows]
        return [(ctx.lib.rbt_gqa_prefix_d, (ctx.h, C.byref(d), c["seqs"], c["nodes"], c["groups"], p(s["q"]), *refs,
                                            p(s["prefix_len"]), p(s["first"]), p(s["len"]), p(s["n"]), p(s["parent"]),
                                            p(s["gate"]), p(s["out"])))], s["out"]
    if c["kind"] == "sample":
        d = abi.RbtSampleDesc(c["vocab"], c["vocab"], R.DT_BF16 if c["type"] == "bf16" else R.DT_F32)
        return [(ctx.lib.rbt_sample_d, (ctx.h, C.byref(d), c["rows"], p(s["x"]), p(s["temp"]), p(s["top_k"]), p(s["top_p"]),
                                        p(s["min_p"]), p(s["u"]), p(s["tok"]), p(s["p"])))], \
            {"tok": s["tok"]} if s["p"] is None else {"tok": s["tok"], "p": s["p"]}
    K, D = c["kv_heads"], c["dim"]
    cache = abi.RbtKvRows(p(s["kc"]["x"]), p(s["vc"]["x"]), p(s["kc"]["scale"]), p(s["vc"]["scale"]))
    to = R.DT_BF16 if c["kind"] == "read" else R.DT_F32
    d = abi.RbtKvQuantDesc(K, D, c["cap"], to, c["rows"] * K * D, K * D, D)
    calls = [(ctx.lib.rbt_kv_dequant_d, (ctx.h, C.byref(d), c["seqs"], c["rows"], C.byref(cache), p(s["len"]), p(s["n"]),
                                         p(s["ko"]), p(s["vo"])))]
    outs = {"k": s["ko"], "v": s["vo"]}
    if c["kind"] == "quant":
        d = abi.RbtKvQuantDesc(K, D, c["cap"], R.DT_BF16 if c["src"] == "bf16" else R.DT_F32, *s["k"].stride()[:3])
        calls.insert(0, (ctx.lib.rbt_kv_quant_d, (ctx.h, C.byref(d), c["seqs"], c["rows"], p(s["k"]), p(s["v"]), p(s["len"]),
                                                  p(s["n"]), C.byref(cache))))
        outs.update(k_scale=s["kc"]["scale"], v_scale=s["vc"]["scale"])
    return calls, outs


def run(state):
    if not own:
        return _PLAIN[state["case"]["kind"]](state)
    if "call" not in state:  # the descriptors that a program keeps
        state["call"] = _call(state)
    calls, outs = state["call"]
    for fn, args in calls:
        rc = fn(*args)
        if rc:
            _context().check(rc)
    return outs


# ---- the work -----------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "attend":
        K, D, w = case["kv_heads"], case["dim"], case["heads"] * case["dim"]
        counts, lens = _counts(case), _lengths(case)
        plens, first = _prefixes(case)
        members = [b - a for a, b in zip(first, first[1:])]
        rows = sum(counts)
        keys = sum(lens) + rows + sum(n for n, m in zip(plens, members) if m)
        pairs = sum(n * (m + (n + 1) / 2) for n, m in zip(counts, lens))
        pairs += sum(n * sum(counts[a:b]) for n, a, b in zip(plens, first, first[1:]))
        row = D * {"bf16": 2, "f32": 4, "i8": 1}[case["kv"]] + (4 if case["kv"] == "i8" else 0)
        return {"bytes": keys * K * 2.0 * row + rows * w * 4.0 * (3 if case["gate"] else 2), "flops": 4.0 * pairs * w}
    if kind in ("quant", "read"):
        n = case["seqs"] * case["rows"] if kind == "read" else sum(_row_counts(case))
        size = 2 if kind == "read" else 5 + (2 if case["src"] == "bf16" else 4)  # in, 8 bits; and out again as f32
        return {"bytes": 2.0 * n * case["kv_heads"] * (case["dim"] * (1 + size) + 4 * (1 if kind == "read" else 2)),
                "flops": 2.0 * n * case["kv_heads"] * case["dim"] * (1 if kind == "read" else 4)}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * ((2.0 if case["type"] == "bf16" else 4.0) + (4.0 if case["probs"] else 0.0)) + 24.0 * case["rows"],
            "flops": 4.0 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------
def _exact_attend(c, s):
    out, R = s["out"].double(), c["heads"] // c["kv_heads"]
    plens, first = _prefixes(c)

    def part(name, b, upto, g):
        r = s[name]
        x = r["x"][b, upto, g].double()
        return x * r["scale"][b, upto, g].double()[:, None] if "scale" in r else x

    for b, (m, n) in enumerate(zip(_lengths(c), _counts(c))):
        par, mine = s["parent"][b].tolist(), [p for p in range(len(plens)) if first[p] <= b < first[p + 1]]
        for g in range(c["kv_heads"]):
            h = slice(g * R, g * R + R)
            keys, vals = [[part(side + "p", p, slice(0, plens[p]), g) for p in mine] + [part(side + "c", b, slice(0, m), g)]
                          for side in "kv"]
            keys, vals = torch.cat(keys), torch.cat(vals)
            for i in range(n):
                seen, j = [], i
                while j >= 0:
                    seen.append(j)
                    j = par[j]
                q = s["q"][b, i, h].double() / math.sqrt(c["dim"])
                w = torch.softmax(torch.cat([q @ keys.T, q @ part("kd", b, seen, g).T], -1), -1)
                out[b, i, h] = w[:, :len(keys)] @ vals + w[:, len(keys):] @ part("vd", b, seen, g)
        if s["gate"] is not None:
            out[b, :n] *= torch.sigmoid(s["gate"][b, :n].double())
    return out


def _exact_quant(c, s):
    out, start = {}, s["len"].tolist()
    for side in "kv":
        o, sc = s[side + "o"].double(), s[side + "c"]["scale"].double()
        for b, n in enumerate(_row_counts(c)):
            x = s[side][b, :n].double()
            f = (x.abs().max(-1).values / 127.0).float().double()  # the scale that the cache holds
            q = (x / f[..., None]).float().double()  # the quotient is rounded to f32, then to a whole number
            o[b, :n] = torch.round(q).nan_to_num(0.0) * f[..., None]
            sc[b, start[b]:start[b] + n] = f
        out[side], out[side + "_scale"] = o, sc
    return {k: out[k] for k in ("k", "v", "k_scale", "v_scale")}


def _exact_read(c, s):
    out = {}
    for side in "kv":
        r = s[side + "c"]
        out[side] = torch.stack([r["x"][b, a:a + c["rows"]].double() * r["scale"][b, a:a + c["rows"], :, None].double()
                                 for b, a in enumerate(s["len"].tolist())])
    return out


def _exact_sample(c, s):
    x = s["x"].double().cpu().numpy()
    toks, ps = np.zeros(len(x), np.int32), np.zeros(x.shape) if c["probs"] else None
    for r, (t, k, top_p, min_p) in enumerate(zip(*_settings(c))):
        t, top_p, min_p = (float(np.float32(v)) for v in (t, top_p, min_p))
        order = np.lexsort((np.arange(x.shape[1]), -x[r]))
        if t == 0:
            t, k = 1.0, 1
        order = order[:k] if k else order
        w = np.exp((x[r, order] - x[r, order[0]]) / t)
        n = len(w)
        if top_p < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), top_p * w.sum(), side="left"))
        n = max(1, min(n, int((w >= min_p).sum())))
        p = np.zeros(x.shape[1])
        p[order[:n]] = w[:n] / w[:n].sum()
        toks[r] = np.searchsorted(np.cumsum(p), float(s["u"][r]) * p.sum(), side="right")
        if ps is not None:
            ps[r] = p
    out = {"tok": torch.from_numpy(toks)}
    return out if ps is None else {**out, "p": torch.from_numpy(ps)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "quant": _exact_quant, "read": _exact_read, "sample": _exact_sample}[case["kind"]](case, s)
