"""What is measured of the quantised-cache operators: norms of queries and keys per head with the rotation
(tf_op_qk_norm_rope), rows written into a Q4_0 or Q8_0 cache and read back (tf_op_kv_quant, tf_op_kv_dequant), the
decode step's form of both in one launch (tf_op_qkv_store), and attention over such a cache (tf_op_attn_quant).

listed() and draw() give cases, prepare() a case's inputs on the GPU, run() one pass, in plain torch operations
or (where `own` is set) through the library's entry points, exact() the same results in 64 bits, and work() the
bytes and operations that a pass cannot do without.

A quantised cache holds blocks of 16 positions, [slot][kv head][cap / 16][block]: the codes in the order in which
the attention's matrix instructions take them, then the scales (f16).  The layout is the header's; `_places` below
is its formula.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

KV_ID = {"q4": 3, "q8": 4}
BITS = {"q4": 4, "q8": 8}
EPS = 1e-6

# (query heads, kv heads, head dim) of the 1B, 0.5B and 1.5B configurations, and a generic 128-wide one
SHAPES = {"32x8x64": (32, 8, 64), "14x2x64": (14, 2, 64), "12x2x128": (12, 2, 128), "32x8x128": (32, 8, 128)}


def listed():
    rope, quant, read, store, attn = (dict(op=o) for o in ("rope", "quant", "read", "store", "attn"))
    return [
        # one decoded token: latency
        dict(rope, name="norm+rope 1 row", shape="32x8x64", rows=1, norm=1, rot=64, far=2000),
        # the rows of several prompts packed together, half of each head rotated
        dict(rope, name="norm+rope 9001 rows", shape="32x8x128", rows=9001, norm=1, rot=64, far=131000),
        # the new rows of a small batch, written and read back
        dict(quant, name="write+read 7 rows q8", kv="q8", shape="14x2x64", rows=7, slots=7, cap=2048),
        # packed prompts written into their slots and read back
        dict(quant, name="write+read 8192 rows q4", kv="q4", shape="32x8x64", rows=8192, slots=4, cap=4096),
        # a short prefix read back
        dict(read, name="read 301 rows q4", kv="q4", shape="12x2x128", rows=301, slots=1, cap=1152),
        # the contexts of several sequences read back for an operator that wants fp32
        dict(read, name="read 16384 rows q8", kv="q8", shape="32x8x128", rows=16384, slots=8, cap=2304),
        # a batched decode step: queries normed and rotated, keys and values into the cache (and read back)
        dict(store, name="store+read 64 rows q4", kv="q4", shape="12x2x128", rows=64, slots=64, cap=1152, norm=0, rot=128, far=1152),
        # the same for packed prompts, with norms
        dict(store, name="store+read 5003 rows q8", kv="q8", shape="32x8x128", rows=5003, slots=3, cap=2048, norm=1, rot=128, far=2048),
        # the single-token form at the start of a conversation: latency
        dict(attn, name="attn b1 t1 ctx96 q4", kv="q4", shape="32x8x64", batch=1, rows=1, ctx=96, ragged=0),
        # one user's long document, 8 bits
        dict(attn, name="attn b1 t1 ctx32001 q8", kv="q8", shape="14x2x64", batch=1, rows=1, ctx=32001, ragged=0),
        # batched serving at the 1.5B shapes and its bench context, a few drafted tokens each, ragged
        dict(attn, name="attn b32 t5 ctx1144 q4", kv="q4", shape="12x2x128", batch=32, rows=5, ctx=1144, ragged=1),
        # the largest: decode for many users over long caches
        dict(attn, name="attn b64 t1 ctx8128 q4", kv="q4", shape="32x8x128", batch=64, rows=1, ctx=8128, ragged=1),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "quant", "read", "store", "attn", "attn", "attn"])
    shape, kv = rng.choice(list(SHAPES)), rng.choice(list(KV_ID))
    d = SHAPES[shape][2]
    if op == "attn":
        c = dict(op=op, kv=kv, shape=shape, batch=_spread(rng, 1, 64), rows=rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(9, 16)]),
                 ctx=_spread(rng, 1, 40000), ragged=rng.randint(0, 1))
        big = work(listed()[-1])
        while work(c)["bytes"] > big["bytes"] or work(c)["flops"] > big["flops"]:
            c["ctx"] = c["ctx"] * 3 // 5
        return c
    if op == "rope":
        return dict(op=op, shape=shape, rows=_spread(rng, 1, 9001), norm=rng.randint(0, 1), rot=rng.choice([d, d, d // 2]),
                    far=_spread(rng, 100, 1000000))
    rows = _spread(rng, 1, 8192)
    slots = rows if rows <= 64 and rng.randint(0, 1) else rng.randint(1, min(8, rows))
    cap = (-(-rows // slots) + rng.randint(1, 400) + 15) // 16 * 16
    c = dict(op=op, kv=kv, shape=shape, rows=rows, slots=slots, cap=cap)
    if op == "store":
        c.update(norm=rng.randint(0, 1), rot=rng.choice([d, d, d // 2]), far=cap)
    return c


def _lengths(case):
    """Context lengths of the batch: equal, or spread evenly from a seventh of the longest up to it."""
    b, n = case["batch"], case["ctx"]
    if not case["ragged"] or b == 1:
        return [n] * b
    return [n - (n - n // 7) * i // (b - 1) for i in range(b)]


def _counts(case):
    """New rows of each sequence: all of them, or (ragged batches) one less for every third."""
    return [case["rows"] - (1 if case["ragged"] and i % 3 == 2 and case["rows"] > 1 else 0) for i in range(case["batch"])]


# ---- the cache's layout ------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _places(kind, bits, d):
    """For element (position p, dim e) of a block, flat index 16 d: the byte of its code in the block, and the
    shift of the code in it; and for scale (p, group) its index among the block's scales."""
    p = torch.arange(16)[:, None].expand(16, d)
    e = torch.arange(d)[None, :].expand(16, d)
    half, g = p >> 3, p & 7
    if kind == "k":
        lane, r = g * 4 + (e % 32 >> 3), e % 8
        if bits == 4:
            word, byte, shift = half * (d // 32) + e // 32, r >> 1, (r & 1) * 4
        else:
            word, byte, shift = half * (d // 16) + e // 32 * 2 + (r >> 2), r & 3, r * 0
    else:
        lane = (e % 16 >> 1) * 4 + (g >> 1)
        byte = (p & 1) * 2 + half
        if bits == 4:
            word, shift = e // 16, (e & 1) * 4
        else:
            word, shift = e // 16 * 2 + (e & 1), e * 0
    words = d * bits // 64                                             # of each of 32 lanes
    full = words // 4 * 4
    at = torch.where(word < full, word // 4 * 512 + lane * 16, full // 4 * 512 + lane * 8) + word % 4 * 4 + byte
    ps = torch.arange(16)[:, None].expand(16, d // 32)
    grp = torch.arange(d // 32)[None, :].expand(16, d // 32)
    scale = ((ps & 7) * 2 + (ps >> 3)) * (d // 32) + grp
    return at.reshape(-1).cuda(), shift.reshape(-1).cuda(), scale.reshape(-1).cuda()


def _block_bytes(bits, d):
    return 16 * d * bits // 8 + d


def _pack(kind, bits, codes, scales):
    """codes [n][16][d] (0 .. 2^bits - 1) and scales [n][16][d / 32] (f16) -> blocks [n][bytes]."""
    n, _, d = codes.shape
    at, shift, place = _places(kind, bits, d)
    out = torch.zeros((n, _block_bytes(bits, d)), dtype=torch.uint8, device=codes.device)
    flat = codes.reshape(n, -1)
    for s in range(0, 8, bits):
        i = (shift == s).nonzero().flatten()
        out[:, at[i]] |= flat[:, i] << s
    packed = torch.empty((n, d // 2), dtype=torch.float16, device=codes.device)
    packed[:, place] = scales.reshape(n, -1)
    out[:, 16 * d * bits // 8:] = packed.view(torch.uint8)
    return out


def _unpack(kind, bits, blocks, d):
    """blocks [n][bytes] -> values [n][16][d] in fp32."""
    n = blocks.shape[0]
    at, shift, place = _places(kind, bits, d)
    codes = (blocks[:, at] >> shift.to(torch.uint8)) & (2 ** bits - 1)
    scales = blocks[:, 16 * d * bits // 8:].contiguous().view(torch.float16)[:, place].float()
    x = codes.float().sub_(2.0 ** (bits - 1)).reshape(n, 16, d // 32, 32)
    return x.mul_(scales.reshape(n, 16, d // 32, 1)).reshape(n, 16, d)


def _quantise(bits, x):
    """x [...][d] in fp32 -> codes (uint8) and scales (f16) of its groups of 32."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    if bits == 4:
        top = g.abs().amax(-1, keepdim=True)
        first = (g.abs() == top).to(torch.uint8).argmax(-1, keepdim=True)
        scale = (g.gather(-1, first) / -8.0).half()
    else:
        scale = (g.abs().amax(-1, keepdim=True) / 127.0).half()
    lim = (-8, 7) if bits == 4 else (-127, 127)
    s = scale.float()
    q = torch.where(s == 0, 0.0, torch.round(g / s.masked_fill(s == 0, 1.0))).clamp(*lim)
    return (q + 2 ** (bits - 1)).to(torch.uint8).reshape(x.shape), scale.squeeze(-1)


# ---- inputs ------------------------------------------------------------------------------------------

def _cache(case, kind, g, slots, cap):
    """A cache that holds quantised rows of a model's size."""
    _, hk, d = SHAPES[case["shape"]]
    bits = BITS[case["kv"]]
    out = torch.empty((slots, hk, cap // 16, _block_bytes(bits, d)), dtype=torch.uint8, device="cuda")
    for s in range(slots):
        x = torch.randn((hk * cap // 16, 16, d), generator=g, device="cuda")
        if kind == "k":  # some channels of the keys are larger than the others
            x *= 1.0 + 3.0 * (torch.rand(d, generator=g, device="cuda") < 0.06)
        out[s] = _pack(kind, bits, *_quantise(bits, x)).reshape(out.shape[1:])
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    dev = "cuda"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    s = dict(case)
    h, hk, d = SHAPES[case["shape"]]
    rows = case["rows"]
    if case["op"] == "attn":
        b = case["batch"]
        lens, counts = _lengths(case), _counts(case)
        cap = (max(lens) + rows + 15) // 16 * 16
        order = list(range(b))
        r.shuffle(order)
        # the step's fused q | k | v rows, as the QKV product leaves them; attention reads the q part
        s["qkv"] = torch.randn((b, rows, (h + 2 * hk) * d), generator=g, device=dev) * 1.5
        s["k"], s["v"] = _cache(case, "k", g, b, cap), _cache(case, "v", g, b, cap)
        s["slots"], s["n_ctx"], s["n_new"] = i32(order), i32(lens), i32(counts)
        s["cap"], s["longest"] = cap, (max(lens) + rows + 15) // 16 * 16
        s["out"] = torch.empty((b, rows, h * d), device=dev)
        return s
    s["qkv"] = torch.randn((rows, (h + 2 * hk) * d), generator=g, device=dev) * 2.0
    if case["op"] in ("rope", "store"):
        s["q_w"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=dev) if case["norm"] else None
        s["k_w"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=dev) if case["norm"] else None
        s["freq"] = torch.pow(500000.0, -torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev) / case["rot"]).float()
    if case["op"] == "rope":
        # several prompts' rows one after the other, each from a position of its own on
        pos, left = [], rows
        while left:
            n = min(left, r.randint(1, max(1, rows // 2)))
            first = r.randint(0, max(0, case["far"] - n))
            pos += range(first, first + n)
            left -= n
        s["pos"] = i32(pos)
        s["q_out"] = torch.empty((rows, h * d), device=dev)
        s["k_out"] = torch.empty((rows, hk * d), device=dev)
        return s
    # each slot's rows follow one another from a position of its own on
    n_slots, cap = case["slots"], case["cap"]
    order = list(range(n_slots))
    r.shuffle(order)
    slot, pos = [], []
    for i, o in enumerate(order):
        n = rows // n_slots + (i < rows % n_slots)
        first = r.randint(0, cap - n)
        slot += [o] * n
        pos += range(first, first + n)
    s["row_slot"], s["pos"] = i32(slot), i32(pos)
    s["k"], s["v"] = _cache(case, "k", g, n_slots, cap), _cache(case, "v", g, n_slots, cap)
    s["k_rows"] = torch.empty((rows, hk * d), device=dev)
    s["v_rows"] = torch.empty((rows, hk * d), device=dev)
    if case["op"] == "store":
        s["q_out"] = torch.empty((rows, h * d), device=dev)
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


def _ptr(t, offset=0):
    return None if t is None else t.data_ptr() + 4 * offset


def _run_own(s):
    lib, ok = _lib(), _native.check
    stream = torch.cuda.current_stream().cuda_stream
    h, hk, d = SHAPES[s["shape"]]
    qkv, rows, op = s["qkv"], s["rows"], s["op"]
    ld = (h + 2 * hk) * d
    if op == "rope":
        ok(lib.tf_op_qk_norm_rope(_ptr(s["q_out"]), h * d, _ptr(s["k_out"]), hk * d, _ptr(qkv), ld, _ptr(qkv, h * d), ld,
                                  _ptr(s["q_w"]), _ptr(s["k_w"]), EPS, _ptr(s["freq"]), s["rot"], _ptr(s["pos"]), rows, h, hk, d,
                                  stream))
        return s["q_out"], s["k_out"]
    k, v, cap = s["k"], s["v"], s["cap"]
    cache = (_ptr(k), _ptr(v), KV_ID[s["kv"]], hk * cap * d, cap, k.shape[0])
    if op == "attn":
        b = s["batch"]
        if "ws" not in s:  # made once for a state and kept with it
            import ctypes
            n = ctypes.c_size_t(0)
            ok(lib.tf_op_attn_quant_workspace(b, rows, h, hk, d, ctypes.byref(n)))
            s["ws"] = torch.empty(n.value, dtype=torch.uint8, device="cuda")
        ok(lib.tf_op_attn_quant(_ptr(s["out"]), h * d, _ptr(qkv), ld, *cache, _ptr(s["slots"]), _ptr(s["n_ctx"]), _ptr(s["n_new"]),
                                b, rows, h, hk, d, _ptr(s["ws"]), s["ws"].numel(), stream))
        return s["out"]
    where = (_ptr(s["row_slot"]), _ptr(s["pos"]))
    if op == "quant":
        ok(lib.tf_op_kv_quant(*cache, *where, _ptr(qkv, h * d), ld, _ptr(qkv, (h + hk) * d), ld, rows, hk, d, stream))
    elif op == "store":
        ok(lib.tf_op_qkv_store(_ptr(s["q_out"]), h * d, *cache, *where, _ptr(qkv), ld, _ptr(qkv, h * d), ld,
                               _ptr(qkv, (h + hk) * d), ld, _ptr(s["q_w"]), _ptr(s["k_w"]), EPS, _ptr(s["freq"]), s["rot"], rows,
                               h, hk, d, stream))
    ok(lib.tf_op_kv_dequant(_ptr(s["k_rows"]), hk * d, _ptr(s["v_rows"]), hk * d, *cache, *where, rows, hk, d, stream))
    return ((s["q_out"],) if op == "store" else ()) + (s["k_rows"], s["v_rows"])


# ---- the plain forms -----------------------------------------------------------------------------

def _norm(x, w):
    if w is None:
        return x
    mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1]).float()
    return x * (1.0 / torch.sqrt(mean + EPS)) * w


def _rotate(x, pos, freq):
    """Pairs (j, j + n) of x [rows][heads][d]; far angles in 64 bits, and a rotated value rounded once."""
    n = freq.shape[0]
    a = pos.double()[:, None, None] * freq.double()
    c, s = torch.cos(a).float().double(), torch.sin(a).float().double()
    x0, x1 = x[..., :n].double(), x[..., n:2 * n].double()
    return torch.cat([(x0 * c - x1 * s).float(), (x0 * s + x1 * c).float(), x[..., 2 * n:]], -1)


def _heads(s):
    h, hk, d = SHAPES[s["shape"]]
    x = s["qkv"].reshape(s["rows"], h + 2 * hk, d)
    return x[:, :h], x[:, h:h + hk], x[:, h + hk:]


def _plain_rope(s):
    q, k, _ = _heads(s)
    return (_rotate(_norm(q, s["q_w"]), s["pos"], s["freq"]).flatten(1), _rotate(_norm(k, s["k_w"]), s["pos"], s["freq"]).flatten(1))


def _element(s, kind):
    """Byte and shift of the code of element (row, kv head, dim) in the whole cache, and the place of its scale."""
    _, hk, d = SHAPES[s["shape"]]
    bits, c = BITS[s["kv"]], s[kind]
    at, shift, place = _places(kind, bits, d)
    pos = s["pos"].long()
    block = (s["row_slot"].long()[:, None] * hk + torch.arange(hk, device=pos.device)) * c.shape[2] + (pos // 16)[:, None]
    start = block[..., None] * c.shape[3]
    inside = pos % 16
    return (start + at.reshape(16, d)[inside][:, None], shift.reshape(16, d)[inside][:, None].expand(-1, hk, -1),
            (start + 16 * d * bits // 8) // 2 + place.reshape(16, d // 32)[inside][:, None])


def _write(s, kind, x):
    bits, flat = BITS[s["kv"]], s[kind].view(-1)
    at, shift, place = _element(s, kind)
    codes, scales = _quantise(bits, x)
    if bits == 8:
        flat[at] = codes
    else:  # the two codes of a byte are dims 2 i and 2 i + 1 of one row
        flat[at[..., ::2]] = codes[..., ::2] | codes[..., 1::2] << 4
    flat.view(torch.float16)[place] = scales


def _read(s, kind):
    bits, flat = BITS[s["kv"]], s[kind].view(-1)
    at, shift, place = _element(s, kind)
    codes = (flat[at] >> shift.to(torch.uint8)) & (2 ** bits - 1)
    scale = flat.view(torch.float16)[place].float().repeat_interleave(32, -1)
    return ((codes.float() - 2.0 ** (bits - 1)) * scale).flatten(1)


def _plain_cache(s):
    q, k, v = _heads(s)
    out = ()
    if s["op"] == "store":
        out = (_rotate(_norm(q, s["q_w"]), s["pos"], s["freq"]).flatten(1),)
        k = _rotate(_norm(k, s["k_w"]), s["pos"], s["freq"])
    if s["op"] != "read":
        _write(s, "k", k)
        _write(s, "v", v)
    return out + (_read(s, "k"), _read(s, "v"))


def _plain_attn(s):
    h, hk, d = SHAPES[s["shape"]]
    b, t, n, bits = s["batch"], s["rows"], s["longest"], BITS[s["kv"]]
    slots = s["slots"].long()
    kv = []
    for kind in "kv":
        blocks = s[kind][slots, :, :n // 16]
        kv.append(_unpack(kind, bits, blocks.reshape(-1, blocks.shape[-1]), d).reshape(b, hk, n, d))
    k, v = kv
    at = torch.arange(n, device=slots.device)
    new = torch.arange(t, device=slots.device)
    seen = (at[None, None] <= (s["n_ctx"][:, None] + new)[..., None]) & (new < s["n_new"][:, None])[..., None]  # [b][t][n]
    held = at < (s["n_ctx"] + s["n_new"])[:, None]
    v = v.masked_fill(~held[:, None, :, None], 0.0)
    q = s["qkv"][:, :, :h * d].reshape(b, t, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    x = (q @ k.transpose(2, 3)).reshape(b, hk, t, h // hk, n) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~seen[:, None, :, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == float("-inf"), 0.0))
    den = p.sum(-1, keepdim=True)
    o = (p.reshape(b, hk, -1, n) @ v).reshape(b, hk, t, h // hk, d)
    o = o / den.masked_fill(den == 0.0, 1.0)
    return o.permute(0, 2, 1, 3, 4).reshape(b, t, h * d)


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "attn": _plain_attn}.get(state["op"], _plain_cache)(state)


# ---- the same in 64 bits ---------------------------------------------------------------------------

def _exact_heads(x, w, pos, freq):
    """x [rows][heads][d] in 64 bits: norm, then the rotation as a product of complex numbers."""
    if w is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
    n = freq.numel()
    z = torch.complex(x[..., :n], x[..., n:2 * n]) * torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                                                               torch.outer(pos.double(), freq.double()))[:, None]
    return torch.cat((z.real, z.imag, x[..., 2 * n:]), -1).reshape(x.shape[0], -1)


def _exact_levels(bits, x):
    """The values that a quantised row stands for, from the definition: the nearest of the group's levels, ties to even."""
    x = x.double().reshape(*x.shape[:-1], -1, 32)
    big = x.abs().max(-1, keepdim=True)
    if bits == 4:
        lead = torch.where(x.abs() == big.values, torch.arange(32, device=x.device), 32).min(-1, keepdim=True).values
        step = (torch.take_along_dim(x, lead, -1) / -8).half().double()
    else:
        step = (big.values / 127).half().double()
    level = torch.nan_to_num(x / step, nan=0.0, posinf=0.0, neginf=0.0).round()
    level = level.clamp(-8, 7) if bits == 4 else level.clamp(-127, 127)
    return (level * step).flatten(-2).flatten(1)


def _stored(bits, kind, block_rows, d):
    """Values of every position of blocks [n][bytes], walking the block's words: [n][16][d] in 64 bits."""
    n, per = block_rows.shape[0], d * bits // 64
    codes = block_rows[:, :2 * d * bits].to(torch.int16)
    out = torch.empty((n, 16, d), dtype=torch.float64, device=block_rows.device)
    whole, lanes = per - per % 4, torch.arange(32, device=block_rows.device)
    for w in range(per):
        base = (w // 4) * 512 + lanes * 16 + (w % 4) * 4 if w < whole else (whole // 4) * 512 + lanes * 8 + (w % 4) * 4
        for i in range(4):
            byte = codes[:, base + i]
            for j in range(8 // bits):
                if kind == "k":
                    per_half = per // 2
                    p = lanes // 4 + 8 * (w // per_half)
                    wi = w % per_half
                    e = (wi * 32 + lanes % 4 * 8 + 2 * i + j) if bits == 4 else (wi // 2 * 32 + lanes % 4 * 8 + wi % 2 * 4 + i)
                else:
                    p = lanes % 4 * 2 + i // 2 + 8 * (i % 2)
                    e = (w * 16 + lanes // 4 * 2 + j) if bits == 4 else (w // 2 * 16 + lanes // 4 * 2 + w % 2)
                out[:, p, e] = ((byte >> (bits * j)) & (2 ** bits - 1)).double() - 2 ** (bits - 1)
    steps = block_rows[:, 2 * d * bits:].contiguous().view(torch.float16).double().reshape(n, 8, 2, d // 32)
    steps = steps.transpose(1, 2).reshape(n, 16, d // 32)
    return out * steps.repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    h, hk, d = SHAPES[case["shape"]]
    op, rows = case["op"], case["rows"]
    if op == "attn":
        bits = BITS[case["kv"]]
        out = torch.zeros((case["batch"], rows, h, d), dtype=torch.float64, device="cuda")
        for b, (slot, n, m) in enumerate(zip(s["slots"].tolist(), s["n_ctx"].tolist(), s["n_new"].tolist())):
            hidden = torch.ones((m, n + m), dtype=torch.bool, device="cuda").triu(n + 1)
            nb = (n + m + 15) // 16
            k = _stored(bits, "k", s["k"][slot, :, :nb].flatten(0, 1), d).reshape(hk, nb * 16, d)[:, :n + m]
            v = _stored(bits, "v", s["v"][slot, :, :nb].flatten(0, 1), d).reshape(hk, nb * 16, d)[:, :n + m]
            q = s["qkv"][b, :m, :h * d].double().reshape(m, hk, h // hk, d)
            w = torch.einsum("tgrd,gnd->tgrn", q, k) / math.sqrt(d)
            w = torch.softmax(w.masked_fill(hidden[:, None, None], -math.inf), -1)
            out[b, :m] = torch.einsum("tgrn,gnd->tgrd", w, v).reshape(m, h, d)
        return out.flatten(2)
    x = s["qkv"].double().reshape(rows, -1, d)
    if op == "rope":
        return (_exact_heads(x[:, :h], s["q_w"], s["pos"], s["freq"]), _exact_heads(x[:, h:h + hk], s["k_w"], s["pos"], s["freq"]))
    bits = BITS[case["kv"]]
    if op == "read":
        out = []
        for kind in "kv":
            blocks = s[kind][s["row_slot"].long(), :, s["pos"].long() // 16]
            vals = torch.cat([_stored(bits, kind, part.flatten(0, 1), d).reshape(-1, hk, 16, d)
                              .take_along_dim((p.long() % 16)[:, None, None, None], 2)
                              for part, p in zip(blocks.split(512), s["pos"].split(512))])
            out.append(vals.reshape(rows, hk * d))
        return tuple(out)
    v = _exact_levels(bits, x[:, h + hk:])
    if op == "quant":
        return _exact_levels(bits, x[:, h:h + hk]), v
    # a key's code hangs on its rounding to fp32 after norm and rotation: no value of its own in 64 bits
    return _exact_heads(x[:, :h], s["q_w"], s["pos"], s["freq"]), None, v


def work(case):
    h, hk, d = SHAPES[case["shape"]]
    rows = case["rows"]
    if case["op"] == "rope":
        return {"bytes": 8 * (h + hk) * d * rows, "flops": 0}
    size = (BITS[case["kv"]] * 32 + 16) / 256                          # bytes of a value in the cache
    if case["op"] == "attn":
        lens, counts = _lengths(case), _counts(case)
        held = sum(lens) + sum(counts)
        return {"bytes": int(2 * hk * d * size * held) + 8 * h * d * case["batch"] * rows,
                "flops": 4 * h * d * sum(m * (n + (m + 1) / 2) for n, m in zip(lens, counts))}
    moved = 2 * hk * d * (4 + size)                                    # K and V read back
    if case["op"] != "read":
        moved += 2 * hk * d * (4 + size)                               # and written before
    if case["op"] == "store":
        moved += 8 * h * d                                             # the queries
    return {"bytes": int(moved * rows), "flops": 0}
