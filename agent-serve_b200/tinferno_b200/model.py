"""Host-side mirror of the reference engine's ``Model`` API (src/model.hpp:24-90 of
RohanDisa/agent-serve) over the CUDA C-ABI.

    m = Model(path, RunConfig(max_seq=2048))
    logits = m.prefill(tokens)          # Model::prefill(tokens, n, logits)
    logits = m.decode(token)            # Model::decode(token, logits)
    m.reset()                           # Model::reset()

Hyper-parameters are read from the GGUF exactly as the reference reads them
(src/model.cpp:14-41); tensors are handed to the library by pointer and copied once into
HBM in their GGUF block layouts.  Failures raise ``TFError`` (the reference throws
std::runtime_error).  ``stage_preset("b200")`` is the GPU stage next to the reference's
v0..v5 (src/common.hpp:289-322).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import native
from .gguf import GGUFReader


class Mt19937Uniform:
    """std::uniform_real_distribution<float>(0, 1) over std::mt19937(seed) as libstdc++ draws
    it: one 32-bit output x per value, r = float(x) * 2^-32 (rounded to float first), and a
    value that rounds to 1 becomes the float just below 1."""

    def __init__(self, seed: int):
        self.bg = np.random.MT19937()
        self.bg._legacy_seeding(seed)  # init_genrand(seed), std::mt19937's seeding

    def next(self) -> float:
        x = int(self.bg.random_raw())
        r = np.float32(np.float32(x) / np.float32(4294967296.0))
        if r >= np.float32(1.0):
            r = np.nextafter(np.float32(1.0), np.float32(0.0))
        return float(r)


@dataclass
class RunConfig:
    """RunConfig (src/common.hpp:103-116) fields that apply to the GPU stage."""
    stage: str = "b200"
    max_seq: int = 4096
    max_batch: int = 1
    device: int = 0
    kv_type: int = native.TF_KV_F32
    use_graph: bool = True
    decode_mode: int = native.TF_DECODE_KERNELS
    n_predict: int = 64
    temperature: float = 0.0
    top_p: float = 0.9
    seed: int = 42


def stage_preset(stage: str) -> RunConfig:
    if stage != "b200":
        raise ValueError(f"unknown stage {stage} (the CUDA engine is stage b200)")
    return RunConfig()


_KV_NAMES = {native.TF_KV_F32: "f32", native.TF_KV_F16: "f16", native.TF_KV_BF16: "bf16"}


def describe(arch: str, hp: native.HParams, weight_bytes: int, cfg: RunConfig) -> str:
    """Model::describe (src/model.cpp:91-105): one line of the model's shape and the run
    configuration, with the GPU stage's own settings in place of threads / SIMD / blocking."""
    mode = "persistent" if cfg.decode_mode == native.TF_DECODE_PERSISTENT else "kernels"
    return (f"arch={arch} layers={hp.n_layer} dim={hp.n_embd} heads={hp.n_head}/{hp.n_kv_head} "
            f"ff={hp.n_ff} vocab={hp.n_vocab} weights={weight_bytes / 1e6:g} MB stage={cfg.stage} "
            f"device={cfg.device} kv={_KV_NAMES.get(cfg.kv_type, cfg.kv_type)} max_seq={cfg.max_seq} "
            f"slots={cfg.max_batch} graph={'on' if cfg.use_graph else 'off'} decode={mode}")


def hparams_from_gguf(g: GGUFReader) -> native.HParams:
    a = g.arch
    key = lambda f: f"{a}.{f}"
    n_embd = g.u64(key("embedding_length"))
    n_head = g.u64(key("attention.head_count"))
    n_vocab = g.u64(key("vocab_size"), 0)
    if not n_vocab:
        toks = g.kv.get("tokenizer.ggml.tokens")
        n_vocab = len(toks) if isinstance(toks, list) else 0
    if not n_vocab:
        n_vocab = g.tensors["token_embd.weight"].rows
    hp = native.HParams()
    hp.n_vocab = n_vocab
    hp.n_embd = n_embd
    hp.n_ff = g.u64(key("feed_forward_length"))
    hp.n_layer = g.u64(key("block_count"))
    hp.n_head = n_head
    hp.n_kv_head = g.u64(key("attention.head_count_kv"), n_head)
    hp.head_dim = n_embd // n_head if n_head else 0
    hp.rms_eps = g.f32(key("attention.layer_norm_rms_epsilon"), 1e-5)
    hp.rope_theta = g.f32(key("rope.freq_base"), 10000.0)
    llama3 = g.str(key("rope.scaling.type"), "") == "llama3"
    hp.rope_llama3 = 1 if llama3 else 0
    hp.rope_scale = g.f32(key("rope.scaling.factor"), 32.0) if llama3 else 1.0
    hp.rope_low_freq_f = g.f32(key("rope.scaling.low_freq_factor"), 1.0) if llama3 else 1.0
    hp.rope_high_freq_f = g.f32(key("rope.scaling.high_freq_factor"), 4.0) if llama3 else 4.0
    hp.rope_orig_ctx = float(g.u64(key("rope.scaling.original_context_length"), 8192)) if llama3 else 8192.0
    hp.bos = g.u64("tokenizer.ggml.bos_token_id", 1)
    hp.eos = g.u64("tokenizer.ggml.eos_token_id", 2)
    return hp


def tensor_descs(g: GGUFReader):
    names = list(g.order)
    arr = (native.TensorDesc * len(names))()
    keep = []
    for i, n in enumerate(names):
        t = g.tensors[n]
        nb = n.encode()
        keep.append(nb)
        arr[i].name = nb
        arr[i].ggml_type = t.ggml_type
        arr[i].ndim = len(t.ne)
        for d in range(4):
            arr[i].ne[d] = int(t.ne[d]) if d < len(t.ne) else 1
        arr[i].data = t.data.ctypes.data
        arr[i].nbytes = t.nbytes
    return arr, keep


def lookup_tree(text: Sequence[int], width: int, depth: int, room: int):
    """(tokens, parents) of a drafted tree under the text's last token: the continuations of up to
    `width` latest earlier occurrences of the last two tokens (else of the last one), `depth` tokens
    each, common beginnings shared, at most `room` nodes."""
    tokens, parents, kids = [int(text[-1])], [-1], {}
    for g in (2, 1):
        if len(text) <= g:
            continue
        key, found = list(text[-g:]), 0
        for i in range(len(text) - g - 1, -1, -1):
            if list(text[i:i + g]) != key:
                continue
            cur = 0
            for x in text[i + g:i + g + depth]:
                nxt = kids.get((cur, x))
                if nxt is None:
                    if len(tokens) >= room:
                        break
                    nxt = kids[(cur, x)] = len(tokens)
                    tokens.append(int(x))
                    parents.append(cur)
                cur = nxt
            found += 1
            if found >= width or len(tokens) >= room:
                break
        if found:
            break
    return tokens, parents


class Model:
    def __init__(self, path: str, cfg: Optional[RunConfig] = None):
        self.cfg = cfg or RunConfig()
        self.L = native.lib()
        self.gguf = GGUFReader(path)
        self.hp = hparams_from_gguf(self.gguf)
        descs, keep = tensor_descs(self.gguf)
        opt = native.Options(self.cfg.max_seq, self.cfg.max_batch, self.cfg.device, self.cfg.kv_type,
                             1 if self.cfg.use_graph else 0, self.cfg.decode_mode)
        h = C.c_void_p()
        native.check(self.L.tf_cuda_create(descs, len(descs), C.byref(self.hp), C.byref(opt), C.byref(h)))
        self.h = h
        del keep
        self.gguf.close()  # weights now live in HBM
        self.n_vocab = self.hp.n_vocab
        self.n_embd = self.hp.n_embd
        self.n_layer = self.hp.n_layer
        self.bos = self.hp.bos
        self.eos = self.hp.eos
        self.weight_bytes = int(self.L.tf_cuda_weight_bytes(self.h))
        self.kernels_per_step = int(self.L.tf_cuda_kernels_per_step(self.h))
        self.arch = self.gguf.str("general.architecture", "llama")
        self._tree = np.zeros(0, np.int32)  # tokens of the last tree step

    def describe(self) -> str:
        return describe(self.arch, self.hp, self.weight_bytes, self.cfg)

    # ---- the reference API ----
    def prefill(self, tokens: Sequence[int], logits: Optional[np.ndarray] = None, seq: int = 0) -> np.ndarray:
        toks = np.ascontiguousarray(tokens, dtype=np.int32)
        out = logits if logits is not None else np.empty(self.n_vocab, np.float32)
        am = C.c_int(-1)
        native.check(self.L.tf_cuda_prefill(self.h, seq, toks.ctypes.data_as(native.i32p), len(toks),
                                            out.ctypes.data_as(native.f32p), C.byref(am)), self.h)
        self.last_argmax = am.value
        return out

    def decode(self, token: int, logits: Optional[np.ndarray] = None, seq: int = 0) -> np.ndarray:
        out = logits if logits is not None else np.empty(self.n_vocab, np.float32)
        am = C.c_int(-1)
        native.check(self.L.tf_cuda_decode(self.h, seq, int(token), out.ctypes.data_as(native.f32p), C.byref(am)),
                     self.h)
        self.last_argmax = am.value
        return out

    def decode_argmax(self, token: int, seq: int = 0) -> int:
        am = C.c_int(-1)
        native.check(self.L.tf_cuda_decode(self.h, seq, int(token), None, C.byref(am)), self.h)
        return am.value

    def reset(self, seq: int = -1):
        native.check(self.L.tf_cuda_reset(self.h, seq), self.h)

    def n_pos(self, seq: int = 0) -> int:
        return int(self.L.tf_cuda_n_pos(self.h, seq))

    # ---- engine extras ----
    def generate_greedy(self, first_token: int, n: int, eos: int = -1, seq: int = 0) -> list:
        out = np.zeros(max(1, n), np.int32)
        n_out = C.c_int(0)
        native.check(self.L.tf_cuda_generate_greedy(self.h, seq, int(first_token), int(n), int(eos),
                                                     out.ctypes.data_as(native.i32p), C.byref(n_out)), self.h)
        return out[:n_out.value].tolist()

    def decode_batch(self, seq_ids: Sequence[int], tokens: Sequence[int], want_logits: bool = False):
        s = np.ascontiguousarray(seq_ids, dtype=np.int32)
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        am = np.zeros(len(t), np.int32)
        lg = np.empty((len(t), self.n_vocab), np.float32) if want_logits else None
        native.check(self.L.tf_cuda_decode_batch(self.h, s.ctypes.data_as(native.i32p), t.ctypes.data_as(native.i32p),
                                                 len(t), am.ctypes.data_as(native.i32p),
                                                 lg.ctypes.data_as(native.f32p) if lg is not None else None), self.h)
        return (am, lg) if want_logits else am

    def prefill_batch(self, seq_ids: Sequence[int], prompts) -> np.ndarray:
        """Prefill equal-length prompts of several sequences at once; returns each sequence's
        greedy next id."""
        s = np.ascontiguousarray(seq_ids, dtype=np.int32)
        t = np.ascontiguousarray(prompts, dtype=np.int32)
        if t.ndim != 2 or t.shape[0] != len(s):
            raise ValueError("prompts must be [len(seq_ids)][n]")
        am = np.zeros(len(s), np.int32)
        native.check(self.L.tf_cuda_prefill_batch(self.h, s.ctypes.data_as(native.i32p), t.ctypes.data_as(native.i32p),
                                                  len(s), t.shape[1], am.ctypes.data_as(native.i32p)), self.h)
        return am

    def sample(self, temperature: float, top_p: float, r: float, row: int = 0) -> int:
        """sample_logits (src/sampler.cpp:15-52) on the device over the last step's logits of
        `row`, with the caller's uniform draw r (see Mt19937Uniform)."""
        out = C.c_int(0)
        native.check(self.L.tf_cuda_sample(self.h, row, float(temperature), float(top_p), float(r), C.byref(out)),
                     self.h)
        return out.value

    def generate(self, prompt: Sequence[int], n: int, temperature: float, top_p: float, seed: int = 42,
                 eos: int = -1) -> list:
        """The CLI's generation loop (src/main.cpp:106-122): prefill, then sample / stop at eos
        (i > 0) / decode, with std::mt19937(seed) draws for temperature > 0."""
        rng = Mt19937Uniform(seed)
        self.prefill(prompt)
        out = []
        for i in range(n):
            t = self.sample(temperature, top_p, rng.next() if temperature > 0 else 0.0)
            if t == eos and i > 0:
                break
            out.append(t)
            self.decode(t)
        return out

    # ---- speculative decoding (include/tinferno_b200.h, tf_cuda_tree_step / tf_cuda_tree_accept) ----
    @property
    def tree_capacity(self) -> int:
        """Drafted tokens per tree, the root included."""
        return int(self.L.tf_cuda_tree_capacity(self.h))

    @property
    def logits_ptr(self) -> int:
        """Device address of the last step's logits [rows][n_vocab]."""
        return int(self.L.tf_cuda_logits(self.h) or 0)

    def tree_step(self, tokens: Sequence[int], parents: Sequence[int], seq: int = 0, want_logits: bool = False):
        """One forward pass over a tree of drafted tokens: tokens[0] is the token decode() would take
        next, parents[0] = -1, every other node's parent precedes it.  Returns the greedy id after
        each node (and the logits).  The position stays; tree_accept keeps what is right."""
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        p = np.ascontiguousarray(parents, dtype=np.int32)
        if t.ndim != 1 or t.shape != p.shape:
            raise ValueError("tokens and parents must be lists of the same length")
        am = np.zeros(max(1, len(t)), np.int32)
        lg = np.empty((len(t), self.n_vocab), np.float32) if want_logits else None
        native.check(self.L.tf_cuda_tree_step(self.h, seq, t.ctypes.data_as(native.i32p), p.ctypes.data_as(native.i32p),
                                              len(t), lg.ctypes.data_as(native.f32p) if want_logits else None,
                                              am.ctypes.data_as(native.i32p)), self.h)
        self._tree = t.copy()  # (t may be the caller's array)
        return (am, lg) if want_logits else am

    def tree_accept(self, temperature: float = 0.0, u: Optional[Sequence[float]] = None, draft_ptr: int = 0, seq: int = 0):
        """Verifies the last tree_step's tree against the model's distribution at `temperature`
        (draft_ptr: device address of the [nodes][n_vocab] logits that each node's children were drawn
        from, 0 for drafts without a distribution; u: one uniform number per node, needed at a positive
        temperature).  Returns (accepted tokens, next token); the accepted path stays in the cache, next
        is the next root."""
        n = len(self._tree)
        nodes, k, nxt = np.zeros(max(1, n), np.int32), C.c_int(0), C.c_int(0)
        uu = None if u is None else np.ascontiguousarray(u, dtype=np.float32)
        if uu is not None and len(uu) < n:
            raise ValueError("u needs one number per node")
        native.check(self.L.tf_cuda_tree_accept(self.h, seq, C.c_void_p(draft_ptr) if draft_ptr else None, float(temperature),
                                                None if uu is None else uu.ctypes.data_as(native.f32p), nodes.ctypes.data_as(native.i32p),
                                                C.byref(k), C.byref(nxt)), self.h)
        return [int(self._tree[i]) for i in nodes[1:k.value]], nxt.value

    def rewind(self, n_pos: int, seq: int = 0):
        """Back to an earlier position of the sequence (the cache rows behind it are overwritten later)."""
        native.check(self.L.tf_cuda_rewind(self.h, seq, int(n_pos)), self.h)

    def generate_lookup(self, prompt: Sequence[int], n: int, temperature: float = 0.0, seed: int = 42, eos: int = -1,
                        width: int = 3, depth: int = 6, seq: int = 0) -> list:
        """generate() with drafts looked up in the text so far: each step drafts the tokens that
        followed the latest occurrences of the last two tokens (else of the last one), as a tree of up
        to `width` branches of `depth` tokens, and keeps what the model's own distribution keeps.  The
        tokens follow the same distribution as generate() at top_p = 1; at temperature 0 they are the
        greedy ones."""
        rng = Mt19937Uniform(seed)
        text = [int(t) for t in prompt]
        self.prefill(text, seq=seq)
        root = self.sample(temperature, 1.0, rng.next() if temperature > 0 else 0.0)
        out = [root]
        while len(out) < n and not (root == eos and len(out) > 1):
            text.append(root)
            room = min(self.tree_capacity, self.cfg.max_seq - self.n_pos(seq), n - len(out))
            tokens, parents = lookup_tree(text, width, depth, room)
            self.tree_step(tokens, parents, seq=seq)
            u = [rng.next() for _ in tokens] if temperature > 0 else None
            kept, root = self.tree_accept(temperature, u, seq=seq)
            text += kept
            out += kept + [root]
            if eos >= 0 and eos in out[1:]:
                out = out[:out.index(eos, 1)]
                break
        return out[:n]

    # ---- vocab-split lm_head (include/tinferno_b200.h, tf_cuda_set_vocab_shard) ----
    def set_vocab_shard(self, rank: int, world: int):
        native.check(self.L.tf_cuda_set_vocab_shard(self.h, int(rank), int(world)), self.h)

    @property
    def shard_key_ptr(self) -> int:
        """Device address of this GPU's order-flipped greedy key (one int64)."""
        return int(self.L.tf_cuda_shard_key(self.h) or 0)

    def decode_shard(self, token: int = -1, seq: int = 0):
        """One asynchronous step with the split lm_head; token < 0 continues from the reduced key."""
        native.check(self.L.tf_cuda_decode_shard(self.h, seq, int(token)), self.h)

    def shard_token(self, seq: int = 0) -> int:
        out = C.c_int(0)
        native.check(self.L.tf_cuda_shard_token(self.h, seq, C.byref(out)), self.h)
        return out.value

    def history(self, n: int) -> list:
        """The first n ids of the last device-side greedy run (tf_cuda_history)."""
        out = np.zeros(max(1, n), np.int32)
        native.check(self.L.tf_cuda_history(self.h, int(n), out.ctypes.data_as(native.i32p)), self.h)
        return out[:n].tolist()

    @property
    def stream(self) -> int:
        return int(self.L.tf_cuda_stream(self.h) or 0)

    def close(self):
        if getattr(self, "h", None):
            self.L.tf_cuda_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
