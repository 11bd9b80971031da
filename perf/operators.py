"""Performance cases of the drafted-token operators, through their public entry points (include/rabbit_amd.h).

A decode step that checks several drafted tokens at once calls, per attention layer, the rotation of the new
queries and keys and the attention of the draft tree over the cache, and once per step the verification and the
move of the accepted rows into the caches. The kinds:

    rope     rbt_rope_d: per-head norm, rotary positions and the push of q, k, v, one call for the three
    attend   rbt_gqa_tree_d: a tree of drafted tokens per sequence over the sequence's cache
    verify   rbt_draft_verify_d: accepted path and next token from given random numbers
    commit   rbt_kv_commit_d: the accepted tokens' keys and values into every layer's cache

Where `own` is false, run() computes them in elementary torch operations.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DEV = "cuda"
# The attention layers of the repository's own mixer workload: 64 query heads over 4 KV heads, head_dim 256,
# 64 rotated entries, theta 1e7, 23 such layers in the model.
KV_HEADS, DIM, THETA, EPS = 4, 256, 1e7, 1e-6


def listed():
    return [
        # plain decoding: one token, a short chat over a bf16 cache. The smallest attention call: latency
        {"name": "attend_token_513", "kind": "attend", "kv": "bf16", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 1, "nodes": 1, "len": 513, "tree": False, "gate": True},
        # a chain of five drafted tokens over the f32 cache that the one-token step fills
        {"name": "attend_chain5_f32_4096", "kind": "attend", "kv": "f32", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 1, "nodes": 5, "len": 4096, "tree": False, "gate": True},
        # one user's long document with a large draft tree: the largest attention call
        {"name": "attend_tree64_32749", "kind": "attend", "kv": "bf16", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 1, "nodes": 64, "len": 32749, "tree": True, "gate": True},
        # a batch of users with trees of their own, ragged lengths
        {"name": "attend_batch16_8192", "kind": "attend", "kv": "bf16", "heads": 64, "kv_heads": 4, "dim": 256,
         "seqs": 16, "nodes": 24, "len": 8192, "tree": True, "gate": True},
        # odd everything: five query heads per KV head, head_dim 128, three short sequences, no gate
        {"name": "attend_odd_1001", "kind": "attend", "kv": "f32", "heads": 20, "kv_heads": 4, "dim": 128,
         "seqs": 3, "nodes": 7, "len": 1001, "tree": True, "gate": False},
        # the new token of plain decoding: norms, partial rotation, bf16 rows for the cache
        {"name": "rope_token", "kind": "rope", "layout": "half", "heads": 64, "kv_heads": 4, "dim": 256, "start": 0,
         "rope": 64, "tokens": 1, "padded": False, "norm": True, "kv": "bf16", "far": False},
        # a long prompt far into the context: interleaved pairs in the last third of the head, stretched
        # frequencies, no norm
        {"name": "rope_prompt_4095", "kind": "rope", "layout": "pairs", "heads": 64, "kv_heads": 4, "dim": 192,
         "start": 128, "rope": 64, "tokens": 4095, "padded": False, "norm": False, "kv": "f32", "far": True},
        # a chain of four drafts after the root, one user, small vocabulary
        {"name": "verify_chain5_32000", "kind": "verify", "seqs": 1, "nodes": 5, "vocab": 32000, "tree": False,
         "draft": True},
        # trees of sampled drafts for a batch of users, large vocabulary
        {"name": "verify_trees16_131072", "kind": "verify", "seqs": 16, "nodes": 32, "vocab": 131072, "tree": True,
         "draft": True},
        # drafts without probabilities (looked up in the text so far), odd vocabulary
        {"name": "verify_lookup8_100003", "kind": "verify", "seqs": 8, "nodes": 16, "vocab": 100003, "tree": True,
         "draft": False},
        # one user's three accepted tokens into the caches of every attention layer
        {"name": "commit_token", "kind": "commit", "kv": "bf16", "seqs": 1, "nodes": 5, "cap": 1024, "layers": 23},
        # a batch of users with deep trees
        {"name": "commit_batch32", "kind": "commit", "kv": "bf16", "seqs": 32, "nodes": 32, "cap": 256, "layers": 23},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "rope", "rope", "verify", "verify", "commit"])
    if kind == "attend":
        heads, kv_heads, dim = rng.choice([(64, 4, 256), (64, 4, 256), (20, 4, 128), (16, 2, 64), (32, 8, 128), (48, 3, 192),
                                           (12, 12, 64), (6, 2, 80)])
        nodes = _log_int(rng, 1, 64)
        seqs = _log_int(rng, 1, 16)
        longest = max(64, min(32749, int(64 * 32749 / (nodes * seqs)), int(16 * 8192 / seqs)))
        if dim == 80:  # head dims outside the matrix cores' tiles
            longest, nodes, seqs = 500, min(nodes, 8), min(seqs, 4)
        return {"kind": kind, "kv": rng.choice(["bf16", "f32"]), "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs,
                "nodes": nodes, "len": _log_int(rng, 1, longest), "tree": rng.random() < 0.6, "gate": rng.random() < 0.5}
    if kind == "rope":
        dim = rng.choice([64, 80, 128, 192, 256])
        rope = rng.choice([16, 32, 64, dim // 2, dim])
        rope = min(rope, dim)
        return {"kind": kind, "layout": rng.choice(["half", "pairs"]), "heads": rng.choice([5, 16, 20, 32, 64]),
                "kv_heads": rng.choice([1, 2, 4, 8]), "dim": dim, "start": rng.choice([0, dim - rope]), "rope": rope,
                "tokens": _log_int(rng, 1, 3000), "padded": rng.random() < 0.4, "norm": rng.random() < 0.5,
                "kv": rng.choice(["bf16", "f32"]), "far": rng.random() < 0.5}
    if kind == "verify":
        nodes, vocab = _log_int(rng, 1, 32), _log_int(rng, 1000, 131072)
        return {"kind": kind, "seqs": _log_int(rng, 1, 16), "nodes": nodes, "vocab": vocab, "tree": rng.random() < 0.7,
                "draft": rng.random() < 0.6}
    nodes = _log_int(rng, 1, 32)
    return {"kind": kind, "kv": rng.choice(["bf16", "f32"]), "seqs": _log_int(rng, 1, 16), "nodes": nodes,
            "cap": _log_int(rng, nodes + 1, 256), "layers": rng.choice([1, 5, 23])}


# ---- what a program has in hand -------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def _type(case):
    return torch.bfloat16 if case["kv"] == "bf16" else torch.float32


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _spread(n, hi, lo):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * b // max(1, n - 1) for b in range(n)]


def _lengths(case):
    """Committed lengths: the longest first, the others down to half of it (a short batch's last is empty)."""
    n = case["len"]
    return _spread(case["seqs"], n, n // 2 if n > 2048 or case["seqs"] == 1 else 0)


def _counts(case):
    """Drafted nodes per sequence: all of them first, the others down to half."""
    return _spread(case["seqs"], case["nodes"], (case["nodes"] + 1) // 2)


def _parents(case, seed):
    """parent[b, i] < i; node 0 is the root. Chains, or trees whose nodes hang from one of the last eight."""
    B, T = case["seqs"], case["nodes"]
    r = np.random.default_rng(seed)
    par = np.full((B, T), -1, np.int32)
    for i in range(1, T):
        par[:, i] = r.integers(max(0, i - 8), i, B) if case["tree"] else i - 1
    return _i32(par)


def _attend(case, seed):
    g, B, T, H, K, D = _gen(seed), case["seqs"], case["nodes"], case["heads"], case["kv_heads"], case["dim"]
    cap, t = case["len"] + 8, _type(case)
    s = {"q": _normal(g, B, T, H, D), "kc": _normal(g, B, cap, K, D).to(t), "vc": _normal(g, B, cap, K, D).to(t),
         "kd": _normal(g, B, T, K, D).to(t), "vd": _normal(g, B, T, K, D).to(t), "len": _i32(_lengths(case)),
         "n": _i32(_counts(case)), "parent": _parents(case, seed), "out": torch.zeros(B, T, H, D, device=DEV)}
    s["gate"] = _normal(g, B, T, H, D) if case["gate"] else None
    return s


def _rope(case, seed):
    g, S, H, K, D, R = _gen(seed), case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rope"]
    t = _type(case)
    first = 131072 if case["far"] else 17
    pos = torch.arange(first, first + S, dtype=torch.int32, device=DEV)
    if case["padded"]:  # the unused nodes of a batch of trees
        pos = torch.where(torch.rand(S, device=DEV, generator=g) < 0.25, torch.full_like(pos, -1), pos)
    inv = THETA ** (-np.arange(0, R, 2, dtype=np.float64) / R)
    if case["far"]:  # positions interpolated by four in the slow half of the frequencies
        inv = np.where(np.arange(R // 2) >= R // 4, inv / 4.0, inv)
    # q_proj's row holds [query, gate] per head; the queries are a strided view of it
    s = {"pos": pos, "inv": torch.from_numpy(inv).to(DEV), "factor": 1.0 + 0.1 * math.log(4.0) if case["far"] else 1.0,
         "qg": _normal(g, S, H, 2, D) if case["norm"] else _normal(g, S, H, 1, D),
         "k": _normal(g, S, K, D), "v": _normal(g, S, K, D), "q_out": torch.zeros(S, H, D, device=DEV),
         "k_out": torch.zeros(S, K, D, dtype=t, device=DEV), "v_out": torch.zeros(S, K, D, dtype=t, device=DEV)}
    s["q"] = s["qg"][:, :, 0]
    s["qn"], s["kn"] = (_normal(g, D, std=0.1), _normal(g, D, std=0.1)) if case["norm"] else (None, None)
    return s


def _verify(case, seed):
    g, B, T, V = _gen(seed), case["seqs"], case["nodes"], case["vocab"]
    logits = _normal(g, B, T, V, std=5.0)  # a few tokens hold most of the mass, as a language model's rows do
    parent = _parents(case, seed)
    at = parent.clamp(min=0).long()
    s = {"p": torch.softmax(logits, -1), "q": None, "u": torch.rand(B, T, device=DEV, generator=g), "parent": parent,
         "n": _i32(_counts(case))}
    # the drafter's distribution is near the target's; a node's token is drawn from its parent's row
    d = torch.softmax(logits + _normal(g, B, T, V), -1)
    del logits
    sharp = d if case["draft"] else torch.softmax(torch.log(d) * 3.0, -1)
    drawn = torch.stack([torch.multinomial(sharp[b], T, replacement=True, generator=g) for b in range(B)])  # [B, node, draw]
    s["tok"] = torch.gather(drawn, 1, at[:, None, :])[:, 0].to(torch.int32).contiguous()
    if case["draft"]:
        s["q"] = d
    s["path"] = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    s["n_path"] = torch.zeros(B, dtype=torch.int32, device=DEV)
    s["next"] = torch.zeros(B, dtype=torch.int32, device=DEV)
    return s


def _commit(case, seed):
    g, B, T, L, cap = _gen(seed), case["seqs"], case["nodes"], case["layers"], case["cap"]
    r, t = np.random.default_rng(seed), _type(case)
    W = KV_HEADS * DIM
    path, n = np.full((B, T), -1, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        n[b] = min(T, 1 + b % 9 if B > 1 else 3)
        path[b, :n[b]] = np.concatenate([[0], 1 + np.sort(r.choice(T - 1, n[b] - 1, replace=False))]) if T > 1 else [0]
    # one slab per side, a layer's cache and draft rows are slices of it
    return {"cache": torch.randn(L, 2, B, cap, W, device=DEV, generator=g, dtype=t),
            "draft": torch.randn(L, 2, B, T, W, device=DEV, generator=g, dtype=t), "path": _i32(path), "n_path": _i32(n),
            "len": _i32(r.integers(0, cap - T + 1, B).astype(np.int32)), "len_out": torch.zeros(B, dtype=torch.int32, device=DEV)}


_MAKE = {"attend": _attend, "rope": _rope, "verify": _verify, "commit": _commit}


def prepare(case, seed):
    s = _MAKE[case["kind"]](case, seed)
    s["case"] = case
    torch.cuda.synchronize()  # the inputs were made on torch's stream
    return s


# ---- the plain forms --------------------------------------------------------------------------------
def _plain_attend(s):
    c = s["case"]
    B, T, H, K, D = c["seqs"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    L, R = c["len"], H // K
    k = torch.cat([s["kc"][:, :L], s["kd"]], 1).float().permute(0, 2, 3, 1)      # [B, K, D, keys]
    v = torch.cat([s["vc"][:, :L], s["vd"]], 1).float().permute(0, 2, 1, 3)      # [B, K, keys, D]
    q = s["q"].view(B, T, K, R, D).permute(0, 2, 1, 3, 4).reshape(B, K, T * R, D)
    idx = torch.arange(T, device=DEV)
    step = (s["parent"][:, :, None] == idx).double() + torch.eye(T, dtype=torch.float64, device=DEV)
    above = torch.linalg.matrix_power(step, max(1, T - 1)) > 0                   # node i sees node j
    old = torch.arange(L, device=DEV) < s["len"][:, None]
    sees = torch.cat([old[:, None, :].expand(B, T, L), above], 2)                # [B, T, keys]
    a = torch.matmul(q, k).view(B, K, T, R, -1) * (1.0 / math.sqrt(D))
    a = a.masked_fill(~sees[:, None, :, None, :], -math.inf)
    a = torch.exp(a - a.amax(-1, keepdim=True))
    a = a / a.sum(-1, keepdim=True)
    o = torch.matmul(a.view(B, K, T * R, -1), v).view(B, K, T, R, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    if s["gate"] is not None:
        o = o * (1.0 / (1.0 + torch.exp(-s["gate"])))
    return torch.where((idx < s["n"][:, None])[:, :, None, None], o, s["out"])


def _plain_rope(s):
    c = s["case"]
    angle = s["pos"].double()[:, None] * s["inv"]
    cos, sin = (torch.cos(angle) * s["factor"]).float()[:, None], (torch.sin(angle) * s["factor"]).float()[:, None]
    lo, r = c["start"], c["rope"]
    live = (s["pos"] >= 0)[:, None, None]

    def turned(x, w, out):
        if w is not None:
            x = x * (torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + w))
        y = x.clone()
        a, b = (x[..., lo:lo + r:2], x[..., lo + 1:lo + r:2]) if c["layout"] == "pairs" else \
            (x[..., lo:lo + r // 2], x[..., lo + r // 2:lo + r])
        at, bt = a * cos - b * sin, b * cos + a * sin
        y[..., lo:lo + r] = torch.stack([at, bt], -1).flatten(-2) if c["layout"] == "pairs" else torch.cat([at, bt], -1)
        return torch.where(live, y.to(out.dtype), out)

    return {"q": turned(s["q"], s["qn"], s["q_out"]), "k": turned(s["k"], s["kn"], s["k_out"]),
            "v": torch.where(live, s["v"].to(s["v_out"].dtype), s["v_out"])}


def _plain_verify(s):
    """The walk is one step per drafted node, children after their parents; every sequence takes it at once."""
    p, q, tok, parent, n, u = s["p"], s["q"], s["tok"].long(), s["parent"], s["n"], s["u"].double()
    B, T, V = p.shape
    rows = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.int64, device=DEV)
    mass, c = torch.ones(B, dtype=torch.float64, device=DEV), torch.zeros(B, dtype=torch.float64, device=DEV)
    gone = torch.zeros(B, V, dtype=torch.bool, device=DEV)      # without q: the children that were rejected
    taken = torch.zeros(B, T, dtype=torch.bool, device=DEV)
    taken[:, 0] = n > 0

    def residual():
        if q is None:
            return p[rows, cur].double().masked_fill(gone, 0.0)
        return (p[rows, cur].double() - c[:, None] * q[rows, cur].double()).clamp(min=0.0)

    for i in range(1, T):
        child, x = (parent[:, i] == cur) & (i < n), tok[:, i]
        px = p[rows, cur, x].double()
        if q is None:
            here = torch.where(gone[rows, x], torch.zeros_like(px), px)
            ok = child & (u[:, i] * mass < here)
            no = child & ~ok
            mass = torch.where(ok, 1.0, torch.where(no, mass - here, mass))
            gone = gone & ~ok[:, None]
            gone[rows, x] = gone[rows, x] | no
        else:
            qx = q[rows, cur, x].double()
            ok = child & (u[:, i] * (mass * qx) < (px - c * qx).clamp(min=0.0))
            no = child & ~ok
            c = torch.where(ok, 0.0, torch.where(no, c + mass, c))
            mass = torch.where(ok, 1.0, torch.where(no, residual().sum(-1), mass))
        cur = torch.where(ok, torch.full_like(cur, i), cur)
        taken[:, i] = ok
    r = residual()
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p[rows, cur].double())
    cum = r.cumsum(-1)
    nxt = (cum <= u[:, :1] * cum[:, -1:]).sum(-1)
    idx = torch.arange(T, device=DEV)
    path = torch.where(taken, idx, torch.full_like(idx, T)).sort(-1).values
    return {"path": torch.where(path == T, -1, path).to(torch.int32), "n_path": taken.sum(-1).to(torch.int32),
            "next": nxt.to(torch.int32)}


def _plain_commit(s):
    T = s["path"].shape[1]
    j = torch.arange(T, device=DEV)
    rows = torch.arange(s["path"].shape[0], device=DEV)[:, None]
    dst, src = (s["len"][:, None] + j).long(), s["path"].clamp(min=0).long()
    new = torch.where((j < s["n_path"][:, None])[:, :, None], s["draft"][:, :, rows, src], s["cache"][:, :, rows, dst])
    s["cache"][:, :, rows, dst] = new
    return {"cache": s["cache"], "len": s["len"] + s["n_path"]}


_PLAIN = {"attend": _plain_attend, "rope": _plain_rope, "verify": _plain_verify, "commit": _plain_commit}


# ---- the framework's calls ----------------------------------------------------------------------------
_CTX = None


def _context():
    global _CTX
    if _CTX is None:
        import rabbit_amd as R
        _CTX = R.Context(0)
    return _CTX


def _call(s):
    """The state's device call as (entry point, its arguments, its outputs)."""
    import rabbit_amd as R
    from rabbit_amd import abi
    ctx, c, p = _context(), s["case"], lambda t: None if t is None else t.data_ptr()
    if c["kind"] == "attend":
        d = abi.RbtGqaTreeDesc(c["heads"], c["kv_heads"], c["dim"], 1.0 / math.sqrt(c["dim"]),
                               R.DT_BF16 if c["kv"] == "bf16" else R.DT_F32, c["len"] + 8, c["len"],
                               c["heads"] * c["dim"], c["dim"])
        return ctx.lib.rbt_gqa_tree_d, (ctx.h, C.byref(d), c["seqs"], c["nodes"], p(s["q"]), p(s["kc"]), p(s["vc"]),
                                        p(s["kd"]), p(s["vd"]), p(s["len"]), p(s["n"]), p(s["parent"]), p(s["gate"]),
                                        p(s["out"])), s["out"]
    if c["kind"] == "rope":
        d = abi.RbtRopeDesc(R.ROPE_INTERLEAVED if c["layout"] == "pairs" else R.ROPE_HALF, c["dim"], c["start"], c["rope"],
                            p(s["inv"]), s["factor"], 0, EPS)
        parts = (abi.RbtRopePart * 3)(R.rope_part(s["q"], s["q_out"], norm=s["qn"]),
                                      R.rope_part(s["k"], s["k_out"], norm=s["kn"]),
                                      R.rope_part(s["v"], s["v_out"], rotate=False))
        return ctx.lib.rbt_rope_d, (ctx.h, C.byref(d), parts, 3, p(s["pos"]), c["tokens"]), \
            {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if c["kind"] == "verify":
        children = 0 if c["tree"] else 1
        return ctx.lib.rbt_draft_verify_d, (ctx.h, c["seqs"], c["nodes"], c["vocab"], children, p(s["tok"]), p(s["parent"]),
                                            p(s["n"]), p(s["p"]), p(s["q"]), p(s["u"]), p(s["path"]), p(s["n_path"]),
                                            p(s["next"])), {"path": s["path"], "n_path": s["n_path"], "next": s["next"]}
    L = c["layers"]
    ptrs = [(C.c_void_p * L)(*[p(s[side][i, kv]) for i in range(L)]) for side in ("cache", "draft") for kv in (0, 1)]
    d = abi.RbtKvCommitDesc(L, KV_HEADS, DIM, R.DT_BF16 if c["kv"] == "bf16" else R.DT_F32, c["cap"])
    return ctx.lib.rbt_kv_commit_d, (ctx.h, C.byref(d), c["seqs"], c["nodes"], *ptrs, p(s["path"]), p(s["n_path"]),
                                     p(s["len"]), p(s["len_out"])), {"cache": s["cache"], "len": s["len_out"]}


def run(state):
    if not own:
        return _PLAIN[state["case"]["kind"]](state)
    if "call" not in state:  # the descriptors that a program keeps
        state["call"] = _call(state)
    fn, args, outs = state["call"]
    rc = fn(*args)
    if rc:
        _context().check(rc)
    return outs


# ---- the work -----------------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], 2 if case.get("kv") == "bf16" else 4
    if kind == "attend":
        rows, w = sum(_counts(case)), case["heads"] * case["dim"]
        keys = sum(_lengths(case)) + rows
        pairs = sum(n * (m + (n + 1) / 2) for n, m in zip(_counts(case), _lengths(case)))
        return {"bytes": keys * case["kv_heads"] * case["dim"] * 2 * size + rows * w * 4 * (3 if case["gate"] else 2),
                "flops": 4.0 * pairs * w}
    if kind == "rope":
        rows = case["tokens"] * (0.75 if case["padded"] else 1.0)
        return {"bytes": rows * case["dim"] * (case["heads"] * 8 + 2 * case["kv_heads"] * (4 + size)),
                "flops": rows * (case["heads"] + case["kv_heads"]) * (3.0 * case["rope"] + 4.0 * case["dim"] * case["norm"])}
    if kind == "verify":  # the rows that the next token is drawn from
        return {"bytes": case["seqs"] * case["vocab"] * 4.0 * (2 if case["draft"] else 1) + case["seqs"] * case["nodes"] * 24.0,
                "flops": case["seqs"] * case["vocab"] * 4.0}
    rows = sum(min(case["nodes"], 1 + b % 9 if case["seqs"] > 1 else 3) for b in range(case["seqs"]))
    return {"bytes": rows * case["layers"] * 2.0 * 2 * KV_HEADS * DIM * size, "flops": 0.0}


# ---- the definitions in 64 bits -------------------------------------------------------------------------
def _exact_attend(c, s):
    out, R = s["out"].double(), c["heads"] // c["kv_heads"]
    for b, (m, n) in enumerate(zip(_lengths(c), _counts(c))):
        par = s["parent"][b].tolist()
        for g in range(c["kv_heads"]):
            h = slice(g * R, g * R + R)
            keys, vals = s["kc"][b, :m, g].double(), s["vc"][b, :m, g].double()
            for i in range(n):
                seen, j = [], i
                while j >= 0:
                    seen.append(j)
                    j = par[j]
                q = s["q"][b, i, h].double() / math.sqrt(c["dim"])
                w = torch.softmax(torch.cat([q @ keys.T, q @ s["kd"][b, seen, g].double().T], -1), -1)
                out[b, i, h] = w[:, :m] @ vals + w[:, m:] @ s["vd"][b, seen, g].double()
        if s["gate"] is not None:
            out[b, :n] *= torch.sigmoid(s["gate"][b, :n].double())
    return out


def _exact_rope(c, s):
    z = s["factor"] * torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                                  torch.outer(s["pos"].double(), s["inv"]))[:, None, :]
    lo, hi, half = c["start"], c["start"] + c["rope"], c["rope"] // 2

    def one(x, w, turn):
        x = x.double().clone()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w.double())
        if turn:
            part = x[..., lo:hi].unflatten(-1, (half, 2) if c["layout"] == "pairs" else (2, half))
            part = part if c["layout"] == "pairs" else part.transpose(-1, -2)
            part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * z)
            x[..., lo:hi] = (part if c["layout"] == "pairs" else part.transpose(-1, -2)).flatten(-2)
        x[s["pos"] < 0] = 0.0
        return x

    return {"q": one(s["q"], s["qn"], True), "k": one(s["k"], s["kn"], True), "v": one(s["v"], None, False)}


def _exact_verify(c, s):
    tok, par, u = s["tok"].cpu().numpy(), s["parent"].cpu().numpy(), s["u"].double().cpu().numpy()
    path, count, nxt = np.full(tok.shape, -1, np.int32), np.zeros(len(tok), np.int32), np.zeros(len(tok), np.int32)
    row = lambda t, b, i: t[b, i].double().cpu().numpy()  # noqa: E731
    for b, n in enumerate(_counts(c)):
        way, r, total, q = [0], row(s["p"], b, 0), 1.0, None if s["q"] is None else row(s["q"], b, 0)
        scale = 1.0  # of the residual distribution that r / scale is
        for i in range(1, n):
            if par[b, i] != way[-1]:
                continue
            x = tok[b, i]
            drafted = 1.0 if q is None else q[x]
            if u[b, i] * drafted * total < r[x]:
                way.append(i)
                r, total, q = row(s["p"], b, i), 1.0, None if q is None else row(s["q"], b, i)
                scale = 1.0
            elif q is None:
                total -= r[x]
                r[x] = 0.0
            else:  # the residual of r / total against q, left unnormalised
                r = np.maximum(r - total * q, 0.0)
                total = r.sum()
        if not r.sum() > 0:
            r = row(s["p"], b, way[-1])
        path[b, :len(way)], count[b] = way, len(way)
        nxt[b] = np.searchsorted(np.cumsum(r), u[b, 0] * r.sum(), side="right")
    return {"path": torch.from_numpy(path), "n_path": torch.from_numpy(count), "next": torch.from_numpy(nxt)}


def exact(case, seed):
    kind = case["kind"]
    if kind == "commit":  # rows are moved, nothing is computed
        return None
    s = prepare(case, seed)
    return {"attend": _exact_attend, "rope": _exact_rope, "verify": _exact_verify}[kind](case, s)
