"""Host mirror of jitnn-llm's Llm (jitnn-llm/src/main/java/ai/beestream/jitnn/llm/Llm.java:48-120): a GGUF language model
that generates text.  The reference hands generation to the third-party jitllm engine; here the file's quantised weights
are attached to the decode step of libjitnn_hip.so (jitnn_hip_llama_*), the token loop runs in the library
(jitnn_hip_llama_generate: embedding lookup, prompt pass, greedy choice, token-by-token decode over the KV cache) and the
tokenizer is built from the file's metadata (tokenizer.py).

    with Llm.load("model.gguf") as llm:
        answer = llm.generate("What is the capital of France?", 64)
        result = llm.generate(GenerationRequest("Once upon a time", 200, temperature=0.8, top_p=0.95, seed=1, stop=["\n\n"]))

Llama-style architectures only (RMSNorm, rotary embedding, grouped-query attention, SwiGLU: general.architecture "llama",
and the same tensor layout under other names where the metadata says so), with a SwiGLU or a mixture of experts in each layer; anything else raises
(a file without experts that has more tensors than those loads with a warning).
"""
from __future__ import annotations

import ctypes as C
import math
import re
import warnings

import numpy as np

from . import _lib
from .experts import Moe, Router
from .gguf_file import GgufFile
from .llama import LlamaDecoder, W_OUTPUT
from .serving import Rope, SharedPrompt
from .tokenizer import StreamDecoder, Tokenizer

# GGUF tensor names of a Llama-style layer in the order of the decoder's weight slots
LAYER_TENSORS = ["attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down"]
ATTENTION_TENSORS = LAYER_TENSORS[:4]
EXPERT_TENSORS = ["ffn_gate_inp", "ffn_gate_exps", "ffn_up_exps", "ffn_down_exps"]
NORM_TENSORS = ["attn_norm", "ffn_norm"]
LAYER_TENSOR = re.compile(r"blk\.(0|[1-9][0-9]{0,8})\.(.+)")
NORMALISING_ARCHS = {"llama"}  # whose chosen experts' weights sum to one where the file does not say (expert_weights_norm)
INTERLEAVED_ROPE_ARCHS = {"llama", "mistral", "granite"}  # llama.cpp's "NORM" rotary embedding: q and k stored permuted for pairs (2i, 2i + 1)

_TOKEN_CB = C.CFUNCTYPE(None, C.c_int, C.c_void_p)


class GenerationRequest:
    """What Llm.generate(request) hands to the engine (Llm.java:84-93 passes a jitllm GenerationRequest through): the prompt,
    the length limit, sampling and stop sequences.  temperature 0 is the greedy choice; top_k 0 and top_p 1 put no limit
    on the candidates; seed None draws from a fresh generator.  Chat messages and tools are jitllm's and are not built.
    draft_tokens: up to so many tokens per pass are drafted by looking up what followed the text's last tokens before, and verified in that pass; the
    text follows the model's distribution all the same.  With a temperature it takes top_k 0 and top_p 1."""

    def __init__(self, prompt: str, max_new_tokens: int = 128, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, seed=None,
                 stop=(), on_token=None, draft_tokens: int = 0):
        if max_new_tokens < 0 or temperature < 0 or top_k < 0 or not 0.0 < top_p <= 1.0:
            raise ValueError(f"max_new_tokens {max_new_tokens}, temperature {temperature}, top_k {top_k}, top_p {top_p}")
        if draft_tokens < 0 or (draft_tokens and temperature > 0 and (top_k not in (0, 1) or top_p < 1.0)):
            raise ValueError(f"draft_tokens {draft_tokens} with temperature {temperature}, top_k {top_k}, top_p {top_p}")
        self.draft_tokens = int(draft_tokens)
        self.prompt, self.max_new_tokens, self.temperature, self.top_k, self.top_p = prompt, max_new_tokens, float(temperature), int(top_k), float(top_p)
        self.seed, self.stop, self.on_token = seed, tuple(s for s in ([stop] if isinstance(stop, str) else stop) if s), on_token


class GenerationResult:
    """text: the continuation (cut in front of the stop sequence that ended it); tokens: the ids that were produced;
    finish_reason: "eos" (the model's end-of-sequence token), "stop" (a stop sequence) or "length"."""

    def __init__(self, text, tokens, prompt_tokens, finish_reason):
        self.text, self.tokens, self.prompt_tokens, self.finish_reason = text, tokens, prompt_tokens, finish_reason

    def __repr__(self):
        return f"GenerationResult({self.text!r}, {len(self.tokens)} tokens after {self.prompt_tokens}, {self.finish_reason})"


def sample_token(logits, temperature: float, top_k: int, top_p: float, rng) -> int:
    """One token id from logits [vocab].  temperature 0: the largest logit, the lowest index among equals, NaN never (what
    the device kernel of the greedy loop picks).  Otherwise softmax(logits / temperature) over the top_k largest (0: all),
    cut to the smallest set of most likely tokens whose probability reaches top_p, renormalised, and one draw of rng."""
    a = np.asarray(logits, dtype=np.float64).reshape(-1)
    a = np.where(np.isnan(a), -np.inf, a)
    if temperature <= 0.0 or top_k == 1:
        return int(np.argmax(a))
    order = np.argsort(-a, kind="stable")  # most likely first, the lower index first among equals
    if top_k > 0:
        order = order[:top_k]
    z = a[order] / temperature
    z -= z[0]
    p = np.exp(z)
    p /= p.sum()
    if top_p < 1.0:
        keep = int(np.searchsorted(np.cumsum(p), top_p, side="left")) + 1
        order, p = order[:keep], p[:keep] / p[:keep].sum()
    return int(order[min(int(np.searchsorted(np.cumsum(p), rng.random(), side="right")), len(order) - 1)])


def look_up_draft(tokens, count: int) -> list:
    """Up to `count` tokens that followed the last two tokens, or else the last one, where these stood last before."""
    for n in (2, 1):
        if len(tokens) <= n:
            continue
        tail = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at:at + n] == tail:
                return tokens[at + n:at + n + count]
    return []


class StopFilter:
    """Text pieces in, text pieces out, holding back whatever could still turn into a stop sequence: push returns
    (text to emit, stopped); after a stop nothing more comes out and the stop sequence itself is never emitted."""

    def __init__(self, stop):
        self._stop, self._held, self.stopped = tuple(stop), "", False

    def push(self, piece: str):
        if self.stopped:
            return "", True
        text = self._held + piece
        cut = min((i for i in (text.find(s) for s in self._stop) if i >= 0), default=-1)
        if cut >= 0:
            self._held, self.stopped = "", True
            return text[:cut], True
        hold = 0
        for s in self._stop:  # the longest tail of the text that begins a stop sequence stays back
            for n in range(min(len(s) - 1, len(text)), 0, -1):
                if text.endswith(s[:n]):
                    hold = max(hold, n)
                    break
        self._held = text[len(text) - hold:] if hold else ""
        return text[:len(text) - hold] if hold else text, False

    def flush(self) -> str:
        out, self._held = ("" if self.stopped else self._held), ""
        return out


class _Text:
    """One sequence of Llm.continuations: its tokens, their text, and why it ended (None: it has not)."""

    def __init__(self, tokenizer, rq: "GenerationRequest", prompt_ids, seed, emit):
        self.known, self.out, self.pieces, self.reason = list(prompt_ids), [], [], None
        self.rng = np.random.default_rng(seed)
        self._eos, self._rq, self._emit = tokenizer.eos if tokenizer.eos is not None else -1, rq, emit
        self._stream, self._stops = StreamDecoder(tokenizer), StopFilter(rq.stop)

    def _push(self, s, stopped):
        if s:
            self.pieces.append(s)
            if self._emit is not None:
                self._emit(s)
        return stopped

    def take(self, token: int) -> None:
        if token == self._eos:
            self.reason = "eos"
        else:
            self.out.append(token)
            self.known.append(token)
            if self._push(*self._stops.push(self._stream.push(token))):
                self.reason = "stop"
            elif len(self.out) == self._rq.max_new_tokens:
                self.reason = "length"

    def result(self, prompt_tokens: int) -> "GenerationResult":
        if self.reason != "stop":
            if self._push(*self._stops.push(self._stream.flush())):
                self.reason = "stop"
            self._push(self._stops.flush(), False)
        return GenerationResult("".join(self.pieces), self.out, prompt_tokens, self.reason or "length")


class ModelInfo:
    def __init__(self, architecture, name, layers, d_model, heads, kv_heads, head_dim, ffn, vocab, context, quantisation):
        self.architecture, self.name, self.layers, self.d_model, self.heads, self.kv_heads = architecture, name, layers, d_model, heads, kv_heads
        self.head_dim, self.ffn, self.vocab, self.context, self.quantisation = head_dim, ffn, vocab, context, quantisation

    def __repr__(self):
        return (f"ModelInfo({self.architecture} {self.name!r}: {self.layers} layers, d_model {self.d_model}, {self.heads}/{self.kv_heads} heads of "
                f"{self.head_dim}, ffn {self.ffn}, vocab {self.vocab}, context {self.context}, weights {self.quantisation})")


class Llm:
    def __init__(self, gguf: GgufFile, decoder: LlamaDecoder, tokenizer: Tokenizer, info: ModelInfo):
        self._gguf, self._dec, self._tok, self._info = gguf, decoder, tokenizer, info

    @staticmethod
    def load(path, max_context: int | None = None) -> "Llm":
        """Opens the file, uploads its weights (raw blocks, unchanged) and builds the tokenizer (Llm.load, Llm.java:58-72)."""
        f = GgufFile.open(path)
        try:
            arch = f.architecture()
            if arch is None:
                raise ValueError(f"{path}: no general.architecture")
            layers = f.integer(f"{arch}.block_count")
            d = f.integer(f"{arch}.embedding_length")
            heads = f.integer(f"{arch}.attention.head_count")
            kv = f.integer(f"{arch}.attention.head_count_kv", heads)
            experts = f.integer(f"{arch}.expert_count", 0)
            ffn = f.integer(f"{arch}.feed_forward_length", 0 if experts else None)
            if experts and not ffn:  # (no dense layers)
                ffn = f.integer(f"{arch}.expert_feed_forward_length")
            hd = f.integer(f"{arch}.attention.key_length", d // heads)
            eps = f.float_value(f"{arch}.attention.layer_norm_rms_epsilon", 1e-5)
            theta = f.float_value(f"{arch}.rope.freq_base", 10000.0)
            ctx_file = f.integer(f"{arch}.context_length", 2048)
            for name in ("token_embd.weight", "output_norm.weight", "blk.0.attn_q.weight") + (() if experts else ("blk.0.ffn_gate.weight",)):
                if not f.has_tensor(name):
                    raise ValueError(f"{path}: architecture {arch} does not generate text here (no tensor {name}; Llama-style layers are built)")
            routed = {int(m[1]) for m in map(LAYER_TENSOR.fullmatch, f.tensor_infos()) if experts > 0 and m and m[2] == "ffn_gate_inp.weight"}
            unread = Llm._unread(f, layers, routed)
            if unread:
                what = ", ".join(unread[:4]) + (f" and {len(unread) - 4} more" if len(unread) > 4 else "")
                if routed:
                    raise ValueError(f"{path}: what {what} are for is not built")
                warnings.warn(f"{path}: nothing here reads {what}; the text is that of a model without them")
            routing = Llm._routing(f, arch) if routed else None
            emb = f.info("token_embd.weight")
            vocab = emb.shape[0]
            ctx = min(ctx_file, max_context) if max_context else min(ctx_file, 4096)
            dec = LlamaDecoder(layers, d, heads, kv, hd, ffn, vocab, ctx, eps, theta)
            fmts = set()
            for l in range(layers):
                for slot, tn in enumerate(ATTENTION_TENSORS if l in routed else LAYER_TENSORS):
                    w = f.tensor(f"blk.{l}.{tn}.weight")
                    fmts.add(w.dtype().name)
                    dec.set_weight(l, slot, w)
                if l in routed:
                    moe, names = Llm._experts(f, l, experts, routing)
                    dec.set_moe(l, moe)
                    fmts |= names
                dec.set_norm(l, 0, f.raw(f"blk.{l}.attn_norm.weight").view(np.float32))
                dec.set_norm(l, 1, f.raw(f"blk.{l}.ffn_norm.weight").view(np.float32))
            dec.set_norm(0, 2, f.raw("output_norm.weight").view(np.float32))
            # the output head; files with tied embeddings have none and use the token table
            dec.set_weight(0, W_OUTPUT, f.tensor("output.weight" if f.has_tensor("output.weight") else "token_embd.weight"))
            dec.set_embedding(emb.type_id, f.raw("token_embd.weight"))
            dec.set_rope_interleaved(arch in INTERLEAVED_ROPE_ARCHS)
            rope = Llm._rope(f, arch, hd, theta)
            if rope is not None:
                dec.set_rope(rope)
            tok = Tokenizer.from_gguf(f)
            if len(tok.tokens) != vocab:
                raise ValueError(f"{path}: {len(tok.tokens)} tokens for an embedding table of {vocab} rows")
            name = f.get("general.name") if f.has("general.name") else ""
            info = ModelInfo(arch, name, layers, d, heads, kv, hd, ffn, vocab, ctx, "+".join(sorted(fmts)))
            return Llm(f, dec, tok, info)
        except Exception:
            f.close()
            raise

    @staticmethod
    def _unread(f: GgufFile, layers: int, routed) -> list:
        """The tensors that nothing here reads - norms of the heads' queries and keys, biases, experts for every token, layers beyond the model's: it would be another model without
        them.  (Those of the rotary positions are _rope's.)"""
        dense = {f"{n}.weight" for n in LAYER_TENSORS + NORM_TENSORS}
        sparse = {f"{n}.weight" for n in ATTENTION_TENSORS + EXPERT_TENSORS + NORM_TENSORS} | {"exp_probs_b.bias", "exp_probs_b"}

        def is_read(name):
            m = LAYER_TENSOR.fullmatch(name)
            if m:
                return int(m[1]) < layers and m[2] in (sparse if int(m[1]) in routed else dense)
            return name in ("token_embd.weight", "output_norm.weight", "output.weight") or name.startswith("rope_")

        return [n for n in f.tensor_infos() if not is_read(n)]

    @staticmethod
    def _routing(f: GgufFile, arch: str) -> dict:
        """How a file's routers choose: weights of the chosen are normalised or not as the file says (expert_weights_norm; one that does not has to be of NORMALISING_ARCHS), times
        expert_weights_scale; gating by softmax or, expert_gating_func 2, sigmoid.  Other gating functions and groups of experts are not built and raise."""
        gating = f.integer(f"{arch}.expert_gating_func", 1)
        if gating not in (1, 2):
            raise ValueError(f"{f.path()}: expert gating function {gating} is not built")
        if f.integer(f"{arch}.expert_group_count", 1) > 1:
            raise ValueError(f"{f.path()}: experts in groups are not built")
        norm = f"{arch}.expert_weights_norm"
        if not f.has(norm) and arch not in NORMALISING_ARCHS:
            raise ValueError(f"{f.path()}: no {norm}: whether the weights of the chosen experts sum to one is not known for {arch}")
        return dict(used=f.integer(f"{arch}.expert_used_count"), gating="softmax" if gating == 1 else "sigmoid", normalise=f.bool(norm) if f.has(norm) else True,
                    scale=f.float_value(f"{arch}.expert_weights_scale", 1.0) or 1.0)

    @staticmethod
    def _experts(f: GgufFile, l: int, experts: int, routing: dict):
        """The experts of a layer and their formats: the router's weights (ffn_gate_inp), the experts' own (ffn_gate_exps, ffn_up_exps, ffn_down_exps), a bias of the choice
        (exp_probs_b).  routing: _routing's.  What else a layer may have raises before (_unread)."""
        def plain(name):
            t = f.info(name)
            if t.type not in ("F32", "F16"):
                raise ValueError(f"{f.path()}: {name} is {t.type} (F32 and F16 are built)")
            return f.raw(name).view(np.float32 if t.type == "F32" else np.float16).reshape(t.shape).astype(np.float32)

        bias = next((plain(n) for n in (f"blk.{l}.exp_probs_b.bias", f"blk.{l}.exp_probs_b") if f.has_tensor(n)), None)
        weights = plain(f"blk.{l}.ffn_gate_inp.weight")
        if len(weights) != experts:
            raise ValueError(f"{f.path()}: a router of {len(weights)} experts in layer {l} of a model of {experts}")
        router = Router(weights, selection_bias=bias, **routing)
        parts = [f.tensor(f"blk.{l}.{n}.weight") for n in EXPERT_TENSORS[1:]]
        return Moe(router, *parts), {p.dtype().name for p in parts}

    @staticmethod
    def _rope(f: GgufFile, arch: str, head_dim: int, theta: float):
        """The rotary positions that the file asks for, None where they are the plain ones: a part of the head (rope.dimension_count), linear or YaRN scaling
        (rope.scaling.*), factors of the frequencies (rope_freqs.weight).  Of a kind that is not built, or of numbers that nothing can turn by: a warning, and the plain ones."""
        try:
            rot = f.integer(f"{arch}.rope.dimension_count", head_dim)
            kind = f.get(f"{arch}.rope.scaling.type") if f.has(f"{arch}.rope.scaling.type") else "none"
            factors = f.raw("rope_freqs.weight").view(np.float32) if f.has_tensor("rope_freqs.weight") else None
            magnitude = f.float_value(f"{arch}.rope.scaling.attn_factor", 0.0)
            if rot == head_dim and kind == "none" and factors is None and magnitude in (0.0, 1.0):
                return None
            interleaved = arch in INTERLEAVED_ROPE_ARCHS
            if kind not in ("none", "linear", "yarn") or rot > head_dim or rot % 2 or (rot < head_dim and not interleaved) or (factors is not None and factors.size != rot // 2):
                raise ValueError(f"rotary scaling {kind!r} of {rot} of {head_dim} values is not built")
            factor = f.float_value(f"{arch}.rope.scaling.factor", 1.0) or 1.0
            if magnitude and kind == "yarn":
                magnitude *= 0.1 * math.log(factor) + 1.0  # (the file's factor goes on top of the scaling's own)
            return Rope(rot, theta, interleaved, None if kind == "none" else kind, factor,
                        f.integer(f"{arch}.rope.scaling.original_context_length", f.integer(f"{arch}.context_length", 2048)),
                        f.float_value(f"{arch}.rope.scaling.yarn_beta_fast", 32.0), f.float_value(f"{arch}.rope.scaling.yarn_beta_slow", 1.0), magnitude, factors)
        except ValueError as e:
            warnings.warn(f"{arch}: the file's rotary positions are not built ({e}); the positions are the plain ones")
            return None

    def generate(self, prompt, max_new_tokens: int | None = None, on_text=None):
        """generate(prompt, max_new_tokens[, on_text]): the greedy (temperature 0) continuation of `prompt` as a string, at most
        `max_new_tokens` tokens, each piece of text going to `on_text` as it is produced (Llm.generate, Llm.java:74-82).
        generate(request): a GenerationRequest - sampling, stop sequences - to a GenerationResult (Llm.java:84-93)."""
        if isinstance(prompt, GenerationRequest):
            return self._generate_request(prompt)
        if max_new_tokens is None:
            raise TypeError("generate(prompt, max_new_tokens) or generate(GenerationRequest)")
        ids = self._tok.encode(prompt)
        if not ids:
            raise ValueError("the prompt has no tokens")
        stream = StreamDecoder(self._tok)
        pieces = []

        def on_token(token, _user):
            s = stream.push(token)
            if s:
                pieces.append(s)
                if on_text is not None:
                    on_text(s)

        self.generate_tokens(ids, max_new_tokens, on_token)
        tail = stream.flush()
        if tail:
            pieces.append(tail)
            if on_text is not None:
                on_text(tail)
        return "".join(pieces)

    def continuations(self, request: GenerationRequest, count: int, page_tokens: int = 64, cache_type: int = 1) -> list:
        """`count` GenerationResults for one request, decoded together: the prompt runs through the model once, its pages of the cache (ggml type F16 1 or F32 0)
        are shared and read once a pass, and every sequence draws with a generator of its own (seed, seed + 1, ...).  The request's on_token is for
        generate and has to be None."""
        if request.on_token is not None:
            raise ValueError("on_token is for one sequence: Llm.generate")
        return self._continue(request, count, page_tokens, cache_type, None)

    def _continue(self, rq: GenerationRequest, count: int, page_tokens: int, cache_type: int, emit) -> list:
        ids = self._tok.encode(rq.prompt)
        if not ids:
            raise ValueError("the prompt has no tokens")
        if count < 1:
            raise ValueError(f"{count} continuations")
        if len(ids) + rq.max_new_tokens > self._info.context:
            raise ValueError(f"{len(ids)} prompt tokens + {rq.max_new_tokens} new ones in a context of {self._info.context}")
        texts = [_Text(self._tok, rq, ids, None if rq.seed is None else rq.seed + i, emit) for i in range(count)]
        if rq.max_new_tokens > 0:
            drafts = min(rq.draft_tokens, rq.max_new_tokens - 1)
            # (a sequence's last pass may hold drafts behind its last position)
            run = SharedPrompt(self._dec, ids, count, len(ids) + rq.max_new_tokens + drafts, 1 + drafts, page_tokens, cache_type)
            greedy = rq.temperature <= 0.0 or rq.top_k == 1
            for t in texts:
                t.take(sample_token(run.prompt_logits, rq.temperature, rq.top_k, rq.top_p, t.rng))
            while True:
                live = [i for i, t in enumerate(texts) if t.reason is None]
                if not live:
                    break
                if not drafts:
                    logits = run.step(live, [[texts[i].known[-1]] for i in live])
                    for i, row in zip(live, logits):
                        texts[i].take(sample_token(row, rq.temperature, rq.top_k, rq.top_p, texts[i].rng))
                    continue
                tokens = [[texts[i].known[-1]] + look_up_draft(texts[i].known, drafts) for i in live]
                numbers = np.concatenate([texts[i].rng.random((len(ts), 2)) for i, ts in zip(live, tokens)])
                got = run.verify(live, tokens, [0.0 if greedy else rq.temperature] * len(live), numbers)
                for i, ts, (kept, token) in zip(live, tokens, got):
                    for t in ts[1:1 + kept] + [token]:
                        if texts[i].reason is None:
                            texts[i].take(t)
        return [t.result(len(ids)) for t in texts]

    def _generate_request(self, rq: GenerationRequest) -> GenerationResult:
        """The token loop on the host, for requests the library's greedy loop does not cover: the prompt in one pass
        (jitnn_hip_llama_prefill), then logits -> sample_token -> embedding row -> one decode step per token.  Drafted tokens go through a paged cache."""
        if rq.draft_tokens:
            return self._continue(rq, 1, 64, 0, rq.on_token)[0]
        ids = self._tok.encode(rq.prompt)
        if not ids:
            raise ValueError("the prompt has no tokens")
        if len(ids) + rq.max_new_tokens > self._info.context:
            raise ValueError(f"{len(ids)} prompt tokens + {rq.max_new_tokens} new ones in a context of {self._info.context}")
        eos = self._tok.eos if self._tok.eos is not None else -1
        rng = np.random.default_rng(rq.seed)
        stream, stops = StreamDecoder(self._tok), StopFilter(rq.stop)
        pieces, out, reason = [], [], "length"

        def emit(s):
            s, stopped = stops.push(s)
            if s:
                pieces.append(s)
                if rq.on_token is not None:
                    rq.on_token(s)
            return stopped

        if rq.max_new_tokens > 0:
            logits = self._dec.prefill(self._dec.embed(ids), 0)
            pos = len(ids)
            while True:
                token = sample_token(logits, rq.temperature, rq.top_k, rq.top_p, rng)
                if token == eos:
                    reason = "eos"
                    break
                out.append(token)
                if emit(stream.push(token)):
                    reason = "stop"
                    break
                if len(out) == rq.max_new_tokens:
                    break
                logits = self._dec.decode(self._dec.embed([token])[0], pos)
                pos += 1
        if reason != "stop":
            if emit(stream.flush()):
                reason = "stop"
            tail = stops.flush()
            if tail:
                pieces.append(tail)
                if rq.on_token is not None:
                    rq.on_token(tail)
        return GenerationResult("".join(pieces), out, len(ids), reason)

    def generate_tokens(self, prompt_ids, max_new_tokens: int, on_token=None, pos0: int = 0) -> list:
        """Token ids in, token ids out: the loop of jitnn_hip_llama_generate (stops at the file's end-of-sequence token)."""
        eos = self._tok.eos if self._tok.eos is not None else -1
        return self._dec.generate(prompt_ids, max_new_tokens, eos, on_token, pos0)

    def gguf(self) -> GgufFile:
        return self._gguf

    def tokenizer(self) -> Tokenizer:
        return self._tok

    def model(self) -> LlamaDecoder:
        return self._dec

    def info(self) -> ModelInfo:
        return self._info

    def close(self):
        self._dec.close()
        self._gguf.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
        return False
