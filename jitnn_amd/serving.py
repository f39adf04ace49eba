"""Operators of a served batch (jitnn_hip_rope_*, jitnn_hip_paged_*, jitnn_hip_verify_*): rotary positions, a paged cache of keys and values with its
append and its attention, and the verification of drafted tokens.  `*_ptr` arguments are addresses in device memory, `stream_ptr` a hipStream_t (0:
the null stream); the calls only enqueue.  What each does, checks and leaves alone is said in include/jitnn_hip.h.

The reference has the plain rotary embedding (core/ops/Rope.java:86-150) and attention without a cache (core/F.java:588-624); batches over a cache
are its third-party engine's."""
from __future__ import annotations

import ctypes as C
import weakref

import numpy as np

from . import _lib
from ._lib import Batch  # noqa: F401

ROPE_KINDS = {None: 0, "none": 0, "linear": 1, "yarn": 2}


class Rope:
    """The frequencies of rotary positions: `rot_dim` values of a head in pairs (i, i + rot_dim / 2), or (2 i, 2 i + 1) when interleaved.
    scaling None, "linear" or "yarn" by `factor`; freq_factors [rot_dim / 2] divide the frequencies (rope_freqs.weight of GGUF files)."""

    def __init__(self, rot_dim, theta=10000.0, interleaved=False, scaling=None, factor=1.0, original_context=0, beta_fast=32.0, beta_slow=1.0,
                 attention_factor=0.0, freq_factors=None):
        if scaling not in ROPE_KINDS:
            raise ValueError(f"rotary scaling {scaling!r} (None, 'linear' and 'yarn' are built)")
        factors = None if freq_factors is None else np.ascontiguousarray(freq_factors, dtype=np.float32).reshape(-1)
        if factors is not None and factors.size != rot_dim // 2:
            raise ValueError(f"{factors.size} frequency factors for {rot_dim // 2} pairs")
        _lib.init()
        sc = _lib.RopeScaling(ROPE_KINDS[scaling], original_context, factor, beta_fast, beta_slow, attention_factor)
        h = C.c_void_p()
        _lib.check(_lib.lib.jitnn_hip_rope_create(rot_dim, bool(interleaved), theta, C.byref(sc),
                                                  None if factors is None else factors.ctypes.data_as(C.POINTER(C.c_float)), C.byref(h)), "jitnn_hip_rope_create")
        self.rot_dim, self.interleaved, self._h = rot_dim, bool(interleaved), h
        weakref.finalize(self, _lib.lib.jitnn_hip_rope_free, h)

    @property
    def handle(self):
        return self._h

    def apply_dev(self, x_ptr: int, positions_ptr: int, tokens: int, heads: int, head_dim: int, y_ptr: int, x_stride: int = 0, y_stride: int = 0,
                  stream_ptr: int = 0) -> None:
        """y [tokens, heads, head_dim] = x, token t turned by positions[t]; y may be x.  Strides in floats from token to token (0: dense)."""
        dense = heads * head_dim
        rc = _lib.lib.jitnn_hip_rope_dev(self._h, x_ptr, x_stride or dense, positions_ptr, tokens, heads, head_dim, y_ptr, y_stride or dense, stream_ptr)
        if rc:
            _lib.check(rc, "jitnn_hip_rope_dev")


class PagedCache:
    """Keys and values of many sequences in `pages` pages of `page_tokens` positions, ggml type F32 (0) or F16 (1)."""

    def __init__(self, layers, kv_heads, head_dim, pages, page_tokens=64, ggml_type=1):
        _lib.init()
        h = C.c_void_p()
        _lib.check(_lib.lib.jitnn_hip_paged_cache_create(layers, kv_heads, head_dim, pages, page_tokens, ggml_type, C.byref(h)), "jitnn_hip_paged_cache_create")
        self._own(h, layers, kv_heads, head_dim, pages, page_tokens, ggml_type)

    @classmethod
    def wrap_dev(cls, k_ptr: int, v_ptr: int, layers, kv_heads, head_dim, pages, page_tokens=64, ggml_type=1) -> "PagedCache":
        """The same in memory of the caller, who keeps it alive: keys and values [layers][pages][kv_heads][page_tokens][head_dim]."""
        _lib.init()
        h = C.c_void_p()
        _lib.check(_lib.lib.jitnn_hip_paged_cache_wrap_dev(k_ptr, v_ptr, layers, kv_heads, head_dim, pages, page_tokens, ggml_type, C.byref(h)),
                   "jitnn_hip_paged_cache_wrap_dev")
        self = cls.__new__(cls)
        self._own(h, layers, kv_heads, head_dim, pages, page_tokens, ggml_type)
        return self

    def _own(self, h, layers, kv_heads, head_dim, pages, page_tokens, ggml_type):
        self.layers, self.kv_heads, self.head_dim, self.pages, self.page_tokens, self.ggml_type = layers, kv_heads, head_dim, pages, page_tokens, ggml_type
        self._h = h
        weakref.finalize(self, _lib.lib.jitnn_hip_paged_cache_free, h)

    @property
    def handle(self):
        return self._h

    def copy_page_dev(self, source: int, target: int, stream_ptr: int = 0) -> None:
        """Page `source` of every layer to page `target`."""
        _lib.check(_lib.lib.jitnn_hip_paged_cache_copy_page_dev(self._h, source, target, stream_ptr), "jitnn_hip_paged_cache_copy_page_dev")

    def append_dev(self, layer: int, batch: Batch, rope: Rope | None, heads: int, q_ptr: int, q_out_ptr: int, k_ptr: int, v_ptr: int, q_stride: int = 0,
                   q_out_stride: int = 0, k_stride: int = 0, v_stride: int = 0, stream_ptr: int = 0) -> None:
        """Keys (turned by rope) and values of the batch's rows into their pages, queries turned to q_out (which may be q; heads 0: none)."""
        q, kv = heads * self.head_dim, self.kv_heads * self.head_dim
        rc = _lib.lib.jitnn_hip_paged_append_dev(self._h, layer, batch, None if rope is None else rope.handle, q_ptr, q_stride or q, heads, q_out_ptr,
                                                 q_out_stride or q, k_ptr, k_stride or kv, v_ptr, v_stride or kv, stream_ptr)
        if rc:
            _lib.check(rc, "jitnn_hip_paged_append_dev")

    def attention_workspace(self, batch: Batch, heads: int) -> int:
        """Bytes of device memory that attention_dev needs for such a batch."""
        n = _lib.lib.jitnn_hip_paged_attention_workspace(self._h, batch, heads)
        if n < 0:
            _lib.check(n, "jitnn_hip_paged_attention_workspace")
        return n

    def attention_dev(self, layer: int, batch: Batch, heads: int, q_ptr: int, scale: float, y_ptr: int, workspace_ptr: int, workspace_bytes: int, q_stride: int = 0,
                      y_stride: int = 0, stream_ptr: int = 0) -> None:
        """y = softmax(scale q K^T) V of every row over its sequence's positions up to its own."""
        dense = heads * self.head_dim
        rc = _lib.lib.jitnn_hip_paged_attention_dev(self._h, layer, batch, heads, q_ptr, q_stride or dense, scale, y_ptr, y_stride or dense, workspace_ptr,
                                                    workspace_bytes, stream_ptr)
        if rc:
            _lib.check(rc, "jitnn_hip_paged_attention_dev")


def verify_workspace(rows: int, sequences: int, vocab: int) -> int:
    """Bytes of device memory that verify_drafts_dev needs."""
    n = _lib.lib.jitnn_hip_verify_workspace(rows, sequences, vocab)
    if n < 0:
        _lib.check(n, "jitnn_hip_verify_workspace")
    return n


def verify_drafts_dev(logits_ptr: int, rows: int, vocab: int, starts_ptr: int, sequences: int, tokens_ptr: int, temperatures_ptr: int, uniforms_ptr: int, out_ptr: int,
                      accepted_ptr: int, workspace_ptr: int, workspace_bytes: int, draft_probs_ptr: int = 0, logits_stride: int = 0, draft_stride: int = 0,
                      stream_ptr: int = 0) -> None:
    """Which drafted tokens each sequence keeps, and the token drawn behind them, from given random numbers."""
    rc = _lib.lib.jitnn_hip_verify_drafts_dev(logits_ptr, logits_stride or vocab, rows, vocab, starts_ptr, sequences, tokens_ptr, draft_probs_ptr or None,
                                              draft_stride or vocab, temperatures_ptr, uniforms_ptr, out_ptr, accepted_ptr, workspace_ptr, workspace_bytes, stream_ptr)
    if rc:
        _lib.check(rc, "jitnn_hip_verify_drafts_dev")


class DeviceArray:
    """Device memory of the library's for `count` values of a numpy type."""

    def __init__(self, count: int, dtype):
        self.dtype, self.count = np.dtype(dtype), int(count)
        h = C.c_void_p()
        _lib.check(_lib.lib.jitnn_hip_malloc(max(16, self.count * self.dtype.itemsize), C.byref(h)), "jitnn_hip_malloc")
        self.ptr = h.value
        weakref.finalize(self, _lib.lib.jitnn_hip_free, h)

    def put(self, values) -> "DeviceArray":
        a = np.ascontiguousarray(values, dtype=self.dtype).reshape(-1)
        if a.size > self.count:
            raise ValueError(f"{a.size} values for {self.count}")
        if a.size:
            _lib.check(_lib.lib.jitnn_hip_memcpy_h2d(self.ptr, a.ctypes.data_as(C.c_void_p), a.nbytes), "jitnn_hip_memcpy_h2d")
        return self

    def get(self, count: int) -> np.ndarray:
        a = np.empty(min(count, self.count), dtype=self.dtype)
        if a.size:
            _lib.check(_lib.lib.jitnn_hip_memcpy_d2h(a.ctypes.data_as(C.c_void_p), self.ptr, a.nbytes), "jitnn_hip_memcpy_d2h")
        return a


class SharedPrompt:
    """`count` sequences that go on from one prompt, over a paged cache of their own: the prompt runs through the model once, its whole pages belong to all of
    them and are read once a pass for all of them, and each gets a copy of the page it ends in.  decoder: llama.LlamaDecoder with its embedding table;
    each sequence may grow to max_len positions, with at most `rows` tokens of a sequence in one pass."""

    PROMPT_ROWS = 512  # of a pass over the prompt

    def __init__(self, decoder, prompt_ids, count: int, max_len: int, rows: int = 1, page_tokens: int = 64, ggml_type: int = 1):
        cfg = decoder.cfg
        prompt = [int(t) for t in prompt_ids]
        if not prompt or count < 1 or rows < 1 or max_len < len(prompt):
            raise ValueError(f"{len(prompt)} prompt tokens, {count} sequences of up to {max_len} positions, {rows} rows a pass")
        if min(prompt) < 0 or max(prompt) >= cfg["vocab"]:
            raise ValueError(f"token id outside [0, {cfg['vocab']})")
        self._dec, self._vocab, self._rows, self.max_len = decoder, cfg["vocab"], rows, max_len
        self.shared = len(prompt) // page_tokens
        self._width = -(-max_len // page_tokens)
        own = self._width - self.shared
        self._cache = PagedCache(cfg["layers"], cfg["kv_heads"], cfg["head_dim"], max(1, self.shared + count * own), page_tokens, ggml_type)
        self._tables = np.empty((count, self._width), dtype=np.int32)
        self._tables[:, : self.shared] = np.arange(self.shared)
        self._tables[:, self.shared:] = self.shared + np.arange(count * own).reshape(count, own)
        self.lens = [len(prompt)] * count  # positions whose tokens are known
        most = max(min(len(prompt), self.PROMPT_ROWS), count * rows)
        self._tok, self._x, self._logits = DeviceArray(most, np.int32), DeviceArray(most * cfg["d_model"], np.float32), DeviceArray(count * rows * self._vocab, np.float32)
        self._ints = [DeviceArray(n, np.int32) for n in (self._tables.size, count + 1, count, most)]  # tables, starts, lens, rows of the logits
        self._verify = None
        for at in range(0, len(prompt), self.PROMPT_ROWS):
            chunk = prompt[at:at + self.PROMPT_ROWS]
            last = at + len(chunk) == len(prompt)
            self._pass([0], [chunk], [at + len(chunk)], 0, [len(chunk) - 1] if last else [])
        self.prompt_logits = self._logits.get(self._vocab)  # of the token after the prompt
        if len(prompt) % page_tokens:
            for i in range(1, count):
                self._cache.copy_page_dev(int(self._tables[0, self.shared]), int(self._tables[i, self.shared]))

    def _pass(self, which, tokens, lens, shared, logit_rows):
        counts = [len(t) for t in tokens]
        flat = [t for ts in tokens for t in ts]
        tables, starts, ends, rows = self._ints
        tables.put(self._tables[list(which)])
        starts.put(np.concatenate([[0], np.cumsum(counts)]))
        ends.put(lens)
        rows.put(logit_rows)
        self._tok.put(flat)
        batch = Batch(len(counts), len(flat), max(counts), max(lens), tables.ptr, self._width, starts.ptr, ends.ptr, shared)
        _lib.check(_lib.lib.jitnn_hip_llama_embed_dev(self._dec.handle, self._tok.ptr, len(flat), self._x.ptr, None), "jitnn_hip_llama_embed_dev")
        self._dec.step_dev(self._cache, batch, self._x.ptr, rows.ptr, len(logit_rows), self._logits.ptr)

    def _named(self, which):
        return [range(len(self._tables))[i] for i in which]

    def _step(self, which, tokens):
        if not which or len(set(which)) != len(which) or len(tokens) != len(which) or any(not 0 < len(t) <= self._rows for t in tokens):
            raise ValueError(f"sequences {which} with {[len(t) for t in tokens]} tokens (1 to {self._rows} each)")
        if any(not 0 <= t < self._vocab for ts in tokens for t in ts):
            raise ValueError(f"token id outside [0, {self._vocab})")
        lens = [self.lens[i] + len(t) for i, t in zip(which, tokens)]
        if max(lens) > self.max_len:
            raise ValueError(f"position {max(lens) - 1} of {self.max_len}")
        self._pass(which, tokens, lens, self.shared, range(sum(len(t) for t in tokens)))
        return lens

    def step(self, which, tokens) -> np.ndarray:
        """The next tokens of the sequences `which` (a list per sequence): appended, and the logits [rows, vocab] after each of them."""
        which = self._named(which)
        lens = self._step(which, tokens)
        for i, n in zip(which, lens):
            self.lens[i] = n
        n = sum(len(t) for t in tokens)
        return self._logits.get(n * self._vocab).reshape(n, self._vocab)

    def verify(self, which, tokens, temperatures, uniforms):
        """The same for sequences whose tokens after the first are drafted: [(drafts kept, the token drawn after them)].  Of each sequence the first token and the kept
        drafts are appended.  temperatures: one for each of these sequences; uniforms [rows, 2]: two random numbers in [0, 1) for each token."""
        which, rows = self._named(which), sum(len(t) for t in tokens)
        temperatures, uniforms = np.asarray(temperatures, dtype=np.float32), np.asarray(uniforms, dtype=np.float32)
        if temperatures.shape != (len(which),) or uniforms.shape not in ((rows, 2), (2 * rows,)):
            raise ValueError(f"temperatures {temperatures.shape} and uniforms {uniforms.shape} of {len(which)} sequences with {rows} tokens")
        uniforms = np.minimum(uniforms, np.float32(1 - 2.0 ** -24))  # (64-bit numbers below 1 may have become 1, which keeps no draft)
        self._step(which, tokens)
        count, most = len(self._tables), len(self._tables) * self._rows
        if self._verify is None:
            n = verify_workspace(most, count, self._vocab)
            self._verify = [DeviceArray(count, np.float32), DeviceArray(2 * most, np.float32), DeviceArray(most, np.int32), DeviceArray(count, np.int32), DeviceArray(n, np.uint8)]
        temps, nums, out, accepted, space = self._verify
        temps.put(temperatures)
        nums.put(uniforms)
        verify_drafts_dev(self._logits.ptr, rows, self._vocab, self._ints[1].ptr, len(tokens), self._tok.ptr, temps.ptr, nums.ptr, out.ptr, accepted.ptr, space.ptr, space.count)
        got, kept, at, result = out.get(rows), accepted.get(len(tokens)), 0, []
        for i, ts, k in zip(which, tokens, kept):
            result.append((int(k), int(got[at + k])))
            self.lens[i] += 1 + int(k)
            at += len(ts)
        return result
