"""What is measured of the speculative-decoding operators: attention of a tree of drafted tokens over the KV
cache (tf_op_attn_tree), verification of the drafted tokens against the target's distribution
(tf_op_verify_tree), and the commit of the accepted path's cache rows (tf_op_kv_commit).

listed() and draw() give cases, prepare() a case's inputs on the GPU, run() one pass, in plain torch operations
or (where `own` is set) through the library's entry points, exact() the same results in 64 bits, and work() the
bytes and operations that a pass cannot do without.
"""
import math
import os
import random
import sys

import torch

own = False

KV = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KV_ID = {"f32": 0, "f16": 1, "bf16": 2}

# (query heads, kv heads, head dim) of the 1B, 0.5B and 1.5B configurations, and a generic 128-wide one
SHAPES = {"32x8x64": (32, 8, 64), "14x2x64": (14, 2, 64), "12x2x128": (12, 2, 128), "32x8x128": (32, 8, 128)}


def listed():
    attn = dict(op="attn")
    verify = dict(op="verify")
    commit = dict(op="commit")
    return [
        # the single-token form at the start of a conversation: latency
        dict(attn, name="attn b1 t1 ctx96", kv="f32", shape="32x8x64", batch=1, nodes=1, ctx=96, ragged=0, tree="chain"),
        # a short drafted chain of one user, 0.5B shapes, an odd context
        dict(attn, name="attn b1 t5 ctx1733", kv="f32", shape="14x2x64", batch=1, nodes=5, ctx=1733, ragged=0, tree="chain"),
        # a tree of one user over the longest cache that the engine keeps
        dict(attn, name="attn b1 t64 ctx16000", kv="f32", shape="32x8x64", batch=1, nodes=64, ctx=16000, ragged=0, tree="tree"),
        # batched serving at the 1.5B shapes and its bench context, ragged
        dict(attn, name="attn b32 t8 ctx1144", kv="f32", shape="12x2x128", batch=32, nodes=8, ctx=1144, ragged=1, tree="tree"),
        # bf16 cache, an odd tree size
        dict(attn, name="attn b12 t31 ctx4001 bf16", kv="bf16", shape="32x8x128", batch=12, nodes=31, ctx=4001, ragged=1, tree="tree"),
        # the largest: wide trees for many users over long fp16 caches
        dict(attn, name="attn b32 t64 ctx8128 f16", kv="f16", shape="32x8x64", batch=32, nodes=64, ctx=8128, ragged=1, tree="tree"),
        # one user's chain with the draft model's distribution: latency
        dict(verify, name="verify b1 t6", vocab=128256, batch=1, nodes=6, mode="draft", temp=0.8, tree="chain"),
        # one user's tree, greedy
        dict(verify, name="verify b1 t32 greedy", vocab=128256, batch=1, nodes=32, mode="greedy", temp=0.0, tree="tree"),
        # batched chains with distributions
        dict(verify, name="verify b32 t8", vocab=151936, batch=32, nodes=8, mode="draft", temp=1.0, tree="chain"),
        # batched trees whose drafts come without a distribution (n-gram lookup, fixed proposals)
        dict(verify, name="verify b16 t25 nodist", vocab=151936, batch=16, nodes=25, mode="nodist", temp=0.7, tree="tree"),
        # one user's accepted path, the 1B configuration's cache
        dict(commit, name="commit b1 l16", kv="f32", shape="32x8x64", layers=16, batch=1, nodes=16, kept=5, cap=2048),
        # every user's accepted path, the 1.5B configuration's cache
        dict(commit, name="commit b64 l28", kv="f32", shape="12x2x128", layers=28, batch=64, nodes=33, kept=7, cap=1152),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "verify", "commit"])
    if op == "attn":
        c = dict(op=op, kv=rng.choice(list(KV)), shape=rng.choice(list(SHAPES)), batch=_spread(rng, 1, 32),
                 nodes=_spread(rng, 1, 64), ctx=_spread(rng, 16, 16000), ragged=rng.randint(0, 1),
                 tree=rng.choice(["chain", "tree"]))
        big = work(listed()[5])
        while work(c)["bytes"] > big["bytes"] or work(c)["flops"] > big["flops"]:
            c["ctx"] = c["ctx"] * 3 // 5
        return c
    if op == "verify":
        mode = rng.choice(["draft", "draft", "nodist", "greedy"])
        c = dict(op=op, vocab=rng.choice([128256, 151936, _spread(rng, 1000, 150000)]), batch=_spread(rng, 1, 32),
                 nodes=_spread(rng, 1, 64), mode=mode, temp=0.0 if mode == "greedy" else round(rng.uniform(0.4, 1.3), 2),
                 tree=rng.choice(["chain", "tree"]))
        while c["batch"] * c["nodes"] * c["vocab"] > 400 * 151936:
            c["batch"] = max(1, c["batch"] * 3 // 5)
            c["nodes"] = max(1, c["nodes"] * 4 // 5)
        return c
    nodes = _spread(rng, 2, 64)
    return dict(op=op, kv=rng.choice(list(KV)), shape=rng.choice(["32x8x64", "14x2x64", "12x2x128"]),
                layers=rng.choice([2, 16, 24, 28]), batch=_spread(rng, 1, 64), nodes=nodes,
                kept=rng.randint(1, min(nodes, 10)), cap=rng.choice([600, 1152]))


def _lengths(case):
    """Context lengths of the batch: equal, or spread evenly from a seventh of the longest up to it."""
    b, n = case["batch"], case["ctx"]
    if not case["ragged"] or b == 1:
        return [n] * b
    return [n - (n - n // 7) * i // (b - 1) for i in range(b)]


def _counts(case):
    """Drafted tokens of each sequence: all of them, or (ragged batches) one less for every third."""
    return [case["nodes"] - (1 if case.get("ragged") and i % 3 == 2 and case["nodes"] > 1 else 0)
            for i in range(case["batch"])]


def _parents(kind, nodes, rng):
    """parents[0] = -1 (the root); a chain, or a tree whose nodes hang mostly from the earlier ones."""
    if kind == "chain":
        return list(range(-1, nodes - 1))
    return [-1] + [int(t * rng.random() ** 1.6) for t in range(1, nodes)]


def _words(parents):
    """Bit j of node t's words: node j is t itself or one of its ancestors."""
    n = len(parents)
    sets = []
    for t in range(n):
        sets.append((sets[parents[t]] if t else 0) | (1 << t))
    w = (n + 63) // 64
    as_signed = lambda x: x - (1 << 64) if x >> 63 else x
    return [[as_signed((s >> (64 * i)) & (2**64 - 1)) for i in range(w)] for s in sets]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    dev = "cuda"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    s = dict(case)
    b, t = case["batch"], case["nodes"]
    slots = list(range(b))
    r.shuffle(slots)
    if case["op"] == "attn":
        h, hk, d = SHAPES[case["shape"]]
        lens, counts = _lengths(case), _counts(case)
        cap = (max(lens) + t + 15) // 16 * 16
        dt = KV[case["kv"]]
        trees = [_parents(case["tree"], t, r) for _ in range(b)]
        # the step's fused q | k | v rows, as the QKV product leaves them; attention reads the q part
        s["qkv"] = torch.randn((b, t, (h + 2 * hk) * d), generator=g, device=dev) * 2.0
        s["k"] = torch.randn((b, hk, cap, d), generator=g, device=dev, dtype=dt)
        s["v"] = torch.randn((b, hk, cap, d), generator=g, device=dev, dtype=dt)
        s["slots"], s["n_ctx"], s["n_node"] = i32(slots), i32(lens), i32(counts)
        s["mask"] = torch.tensor([_words(p) for p in trees], dtype=torch.int64, device=dev)
        s["out"] = torch.empty((b, t, h * d), device=dev)
        s["longest"] = max(lens) + t
    elif case["op"] == "verify":
        v = case["vocab"]
        trees = [_parents(case["tree"], t, r) for _ in range(b)]
        par = i32(trees)
        # a model's logits: a bulk of small values and a tail of likely tokens
        e = torch.empty((b, t, v), device=dev)
        target = torch.randn((b, t, v), generator=g, device=dev).mul_(1.5)
        target += e.exponential_(generator=g).mul_(1.2)
        rows = torch.arange(b, device=dev)[:, None]
        if case["mode"] == "draft":
            draft = target + 0.6 * torch.randn((b, t, v), generator=g, device=dev)
            # each child is drawn from its parent's draft distribution
            e.exponential_(generator=g).log_().neg_()
            tok = (draft[rows, par.long().clamp(min=0)] / case["temp"]).add_(e).argmax(-1)
            s["draft"] = draft
        else:
            # likely tokens of the parent's row, some of them the likeliest
            e.uniform_(0.0, 3.0, generator=g)
            tok = target[rows, par.long().clamp(min=0)].add_(e).argmax(-1)
            s["draft"] = None
        s["logits"], s["parents"], s["tokens"] = target, par, tok.int()
        s["n_node"] = i32([t] * b)
        s["u"] = torch.rand((b, t), generator=g, device=dev)
        s["path"] = torch.empty((b, t), dtype=torch.int32, device=dev)
        s["n_path"] = torch.empty(b, dtype=torch.int32, device=dev)
        s["next"] = torch.empty(b, dtype=torch.int32, device=dev)
    else:
        h, hk, d = SHAPES[case["shape"]]
        dt, cap, kept = KV[case["kv"]], case["cap"], case["kept"]
        s["k"] = torch.randn((case["layers"], b, hk, cap, d), generator=g, device=dev, dtype=dt)
        s["v"] = torch.randn((case["layers"], b, hk, cap, d), generator=g, device=dev, dtype=dt)
        s["slots"] = i32(slots)
        s["n_ctx"] = i32([r.randint(0, cap - t) for _ in range(b)])
        # the root, then a path of nodes behind it
        paths = [[0] + sorted(r.sample(range(1, t), kept - 1)) + [-1] * (t - kept) for _ in range(b)]
        s["path"] = i32(paths)
        s["n_path"] = i32([kept] * b)
        s["n_new"] = torch.empty(b, dtype=torch.int32, device=dev)
    return s


# ---- the library's calls -------------------------------------------------------------------------

_native = None


def _lib():
    global _native
    if _native is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "agent-serve_b200"))
        from tinferno_b200 import native
        _native = native
    return _native.lib()


def _workspace(s, size_call, *shape):
    """The call's workspace, made once for a state and kept with it, zeroed before its first use."""
    if "ws" not in s:
        import ctypes
        n = ctypes.c_size_t(0)
        _native.check(size_call(*shape, ctypes.byref(n)))
        s["ws"] = torch.zeros(n.value, dtype=torch.uint8, device="cuda")
    return s["ws"]


def _run_own(s):
    lib = _lib()
    stream = torch.cuda.current_stream().cuda_stream
    b, t = s["batch"], s["nodes"]
    if s["op"] == "attn":
        h, hk, d = SHAPES[s["shape"]]
        ws = _workspace(s, lib.tf_op_attn_tree_workspace, b, t, h, hk, d)
        k = s["k"]
        _native.check(lib.tf_op_attn_tree(
            s["out"].data_ptr(), h * d, s["qkv"].data_ptr(), s["qkv"].shape[2], k.data_ptr(), s["v"].data_ptr(),
            KV_ID[s["kv"]], k.stride(0), k.shape[2], k.shape[0], s["slots"].data_ptr(), s["n_ctx"].data_ptr(),
            s["n_node"].data_ptr(), s["mask"].data_ptr(), b, t, h, hk, d, ws.data_ptr(), ws.numel(), stream))
        return s["out"]
    if s["op"] == "verify":
        v = s["vocab"]
        ws = _workspace(s, lib.tf_op_verify_tree_workspace, b, t, v)
        _native.check(lib.tf_op_verify_tree(
            s["path"].data_ptr(), s["n_path"].data_ptr(), s["next"].data_ptr(), s["logits"].data_ptr(), v,
            s["draft"].data_ptr() if s["draft"] is not None else None, v, s["tokens"].data_ptr(),
            s["parents"].data_ptr(), s["n_node"].data_ptr(), s["u"].data_ptr(), s["temp"], b, t, v, ws.data_ptr(),
            ws.numel(), stream))
        return s["path"], s["n_path"], s["next"]
    k = s["k"]
    _native.check(lib.tf_op_kv_commit(
        k.data_ptr(), s["v"].data_ptr(), KV_ID[s["kv"]], k.shape[0], k.stride(0), k.stride(1), k.shape[3], k.shape[1],
        s["slots"].data_ptr(), s["n_ctx"].data_ptr(), s["path"].data_ptr(), t, s["n_path"].data_ptr(),
        s["n_new"].data_ptr(), b, k.shape[2], k.shape[4], stream))
    return k, s["v"], s["n_new"]


# ---- the plain forms -----------------------------------------------------------------------------

def _visible(s):
    """[b][t][position]: what each node attends to."""
    t, dev = s["nodes"], s["qkv"].device
    pos = torch.arange(s["longest"], device=dev)
    j = pos[None, :] - s["n_ctx"].long()[:, None]                       # drafted index of each position
    jc = j.clamp(0, t - 1)
    bit = torch.arange(t, device=dev)
    seen = (s["mask"][..., bit // 64] >> (bit % 64)) & 1                # [b][node][drafted]
    seen = torch.gather(seen, 2, jc[:, None, :].expand(-1, t, -1)).bool()
    inside = (j >= 0) & (j < s["n_node"].long()[:, None])
    rows = bit[None, :] < s["n_node"].long()[:, None]
    return ((j < 0)[:, None, :] | (inside[:, None, :] & seen)) & rows[:, :, None], inside | (j < 0)


def _plain_attn(s):
    h, hk, d = SHAPES[s["shape"]]
    b, t, n = s["batch"], s["nodes"], s["longest"]
    vis, held = _visible(s)
    q = s["qkv"][:, :, :h * d].reshape(b, t, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    k = s["k"][s["slots"].long(), :, :n].float()
    v = s["v"][s["slots"].long(), :, :n].float().masked_fill(~held[:, None, :, None], 0.0)
    x = (q @ k.transpose(2, 3)).reshape(b, hk, t, h // hk, n) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~vis[:, None, :, None, :], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == float("-inf"), 0.0))
    den = p.sum(-1, keepdim=True)
    o = (p.reshape(b, hk, -1, n) @ v).reshape(b, hk, t, h // hk, d)
    o = o / den.masked_fill(den == 0.0, 1.0)
    return o.permute(0, 2, 1, 3, 4).reshape(b, t, h * d)


def _soft(x, temp):
    """exp of the scaled logits over their row's maximum, and each row's sum.  A pick by a cumulative sum of 10^5
    terms is a discontinuous function of those terms, so sums, probabilities and residuals are held in 64 bits."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) * (1.0 / torch.tensor(temp, dtype=torch.float32).item()))
    return e, e.sum(-1, dtype=torch.float64)


def _plain_verify(s):
    b, t, v = s["batch"], s["nodes"], s["vocab"]
    dev = s["logits"].device
    rows, at = torch.arange(b, device=dev), torch.arange(t, device=dev)
    cur = torch.zeros(b, dtype=torch.long, device=dev)
    path = torch.full((b, t), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    count = torch.ones(b, dtype=torch.long, device=dev)
    if s["mode"] == "greedy":
        best = s["logits"].argmax(-1)
    else:
        ep, sp = _soft(s["logits"], s["temp"])
        if s["draft"] is not None:
            eq, sq = _soft(s["draft"], s["temp"])
        c, w = torch.zeros(b, dtype=torch.float64, device=dev), torch.ones(b, dtype=torch.float64, device=dev)
        gone = torch.zeros((b, v), dtype=torch.bool, device=dev)
    for i in range(1, t):  # nodes come in an order in which parents precede their children
        child = (s["parents"][:, i] == cur) & (i < s["n_node"])
        x, u = s["tokens"][:, i].long(), s["u"][:, i].double()
        if s["mode"] == "greedy":
            take = child & (best[rows, cur] == x)
        elif s["draft"] is not None:
            px = ep[rows, cur, x].double() / sp[rows, cur]
            qx = eq[rows, cur, x].double() / sq[rows, cur]
            take = child & (u * w * qx < (px - c * qx).clamp(min=0.0))
            drop = child & ~take
            c2 = c + w
            left = ep[rows, cur].double() / sp[rows, cur][:, None] - eq[rows, cur].double() * (c2 / sq[rows, cur])[:, None]
            w2 = left.clamp_(min=0.0).sum(-1)
            c2, w2 = torch.where(w2 > 0, c2, 0.0), torch.where(w2 > 0, w2, 1.0)
            c, w = torch.where(drop, c2, torch.where(take, 0.0, c)), torch.where(drop, w2, torch.where(take, 1.0, w))
        else:
            px = torch.where(gone[rows, x], 0.0, ep[rows, cur, x].double() / sp[rows, cur])
            take = child & (u * w < px)
            drop = child & ~take
            gone[rows, x] |= drop
            gone &= ~take[:, None]
            w = torch.where(drop, w - px, torch.where(take, 1.0, w))
        path[rows, count.clamp(max=t - 1)] = torch.where(take, i, path[rows, count.clamp(max=t - 1)]).int()
        count = count + take
        cur = torch.where(take, i, cur)
    if s["mode"] == "greedy":
        nxt = best[rows, cur]
    else:
        left = ep[rows, cur].double() / sp[rows, cur][:, None]
        if s["draft"] is not None:
            left = (left - eq[rows, cur].double() * (c / sq[rows, cur])[:, None]).clamp_(min=0.0)
        else:
            left = left.masked_fill(gone, 0.0)
        acc = left.cumsum(-1)
        nxt = (acc > (s["u"][:, 0].double() * acc[:, -1])[:, None]).int().argmax(-1)
    return path, count.int(), nxt.int()


def _plain_commit(s):
    at = torch.arange(s["kept"], device=s["k"].device)  # no path of these inputs is longer
    slot, dst = s["slots"].long()[:, None], s["n_ctx"].long()[:, None] + at
    src = torch.where(at < s["n_path"][:, None], s["n_ctx"].long()[:, None] + s["path"][:, :s["kept"]].long(), dst)
    for c in (s["k"], s["v"]):
        c[:, slot, :, dst] = c[:, slot, :, src]
    s["n_new"].copy_(s["n_ctx"] + s["n_path"])
    return s["k"], s["v"], s["n_new"]


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "verify": _plain_verify, "commit": _plain_commit}[state["op"]](state)


# ---- the same in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] != "attn":
        return None  # whole numbers, and copies
    s = prepare(case, seed)
    h, hk, d = SHAPES[case["shape"]]
    rep, t = h // hk, case["nodes"]
    out = torch.zeros((case["batch"], t, h, d), dtype=torch.float64, device="cuda")
    words = s["mask"].cpu().tolist()
    for b, (slot, n, m) in enumerate(zip(s["slots"].tolist(), s["n_ctx"].tolist(), s["n_node"].tolist())):
        bias = torch.zeros((m, n + m), dtype=torch.float64)
        for i in range(m):
            for j in range(m):
                if not (words[b][i][j // 64] >> (j % 64)) & 1:
                    bias[i, n + j] = -math.inf
        bias = bias.cuda()
        for g in range(hk):
            k, v = s["k"][slot, g, :n + m].double(), s["v"][slot, g, :n + m].double()
            for e in range(g * rep, (g + 1) * rep):
                q = s["qkv"][b, :m, e * d:(e + 1) * d].double()
                out[b, :m, e] = torch.softmax(q.mm(k.t()) / math.sqrt(d) + bias, dim=1).mm(v)
    return out.reshape(case["batch"], t, h * d)


def work(case):
    b, t = case["batch"], case["nodes"]
    if case["op"] == "attn":
        h, hk, d = SHAPES[case["shape"]]
        size = 4 if case["kv"] == "f32" else 2
        lens, counts = _lengths(case), _counts(case)
        held = sum(lens) + sum(counts)
        return {"bytes": 2 * hk * d * size * held + 8 * h * d * b * t,
                "flops": 4 * h * d * sum(m * (n + 1) for n, m in zip(lens, counts))}
    if case["op"] == "verify":
        # only the rows of the nodes that the walk visits have to be read; on these inputs it visits this many of a
        # sequence's on average (the root's row always)
        rows = min(t, {"draft": 3.5, "greedy": 3.0, "nodist": 1.5}[case["mode"]])
        return {"bytes": int(b * rows * case["vocab"]) * (8 if case["mode"] == "draft" else 4), "flops": 0}
    h, hk, d = SHAPES[case["shape"]]
    size = 4 if case["kv"] == "f32" else 2
    return {"bytes": 4 * case["layers"] * b * hk * d * size * max(1, case["kept"] - 1), "flops": 0}
