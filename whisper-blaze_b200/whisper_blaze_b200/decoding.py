"""A decoder that generates from 8-bit key/value caches, batched, without a host
round trip per token.

`Kv8Cache` is the pages, scales, block table and lengths that ops.kv8_append and
ops.attention_kv8 work on. `Kv8Decoder` is a pre-norm decoder (causal
self-attention, cross-attention to encoder states, GELU MLP) of FP8 linears
whose two caches per layer are such pages and whose vocabulary logits go to
ops.sample. A prompt of any length is one pass; after it every token is one
replay of a CUDA graph that appends, attends, projects and samples.

    cfg = DecoderConfig(layers=2)
    decoder = Kv8Decoder(cfg, random_decoder_weights(cfg, "cuda:0"), "cuda:0")
    tokens, logprobs = decoder.generate(states, prompt, 64, temperature=0.7, top_p=0.9)

Takes the place of the decoder half of HF's WhisperForConditionalGeneration
.generate, which whisper_blaze/model.py runs with fp16 caches of torch tensors.
"""
from __future__ import annotations

import contextlib
import functools
import threading
from dataclasses import dataclass
from typing import Dict, List, Optional, Tuple

import torch

from . import ops


class Kv8Cache:
    """8-bit keys and values of `layers` layers for `batch` sequences of up to max_tokens tokens.

    All layers share the block table [batch, max_blocks] and the lengths [batch]
    (int32, on the device). Here sequence b owns the pages b * max_blocks onwards;
    a caller with a page allocator of its own writes the table instead."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, max_tokens: int, device, block: int = 64,
                 fmt: str = "e4m3") -> None:
        dev = torch.device(device)
        self.fmt, self.block, self.batch = fmt, block, batch
        width = -(-max_tokens // block)
        self.max_tokens = width * block
        pages = batch * width
        self.codes = torch.zeros(layers, 2, pages, kv_heads, block, head_dim, dtype=torch.uint8, device=dev)
        self.scales = torch.ones(layers, 2, pages, kv_heads, dtype=torch.float32, device=dev)
        self.block_table = torch.arange(pages, dtype=torch.int32, device=dev).view(batch, width)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)

    def _layer(self, layer: int) -> tuple:
        return (self.codes[layer, 0], self.codes[layer, 1], self.scales[layer, 0], self.scales[layer, 1], self.block_table)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, new_lens: Optional[torch.Tensor] = None) -> None:
        """Store k, v [B, Hkv, T, D] behind the tokens held; `advance` counts them, once for all layers."""
        ops.kv8_append(k, v, *self._layer(layer), self.lens, new_lens, fmt=self.fmt)

    def advance(self, count) -> None:
        """`count` tokens (a number or int32 [B]) per sequence were appended to every layer."""
        self.lens.add_(count)

    def attend(self, layer: int, q: torch.Tensor, seq_lens: torch.Tensor, q_lens: Optional[torch.Tensor] = None,
               causal: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(q k^T / sqrt(D)) v over the first seq_lens tokens of each sequence."""
        return ops.attention_kv8(q, *self._layer(layer), seq_lens, q_lens, causal=causal, fmt=self.fmt, out=out)


@dataclass(frozen=True)
class DecoderConfig:
    """Decoder dimensions; the defaults are large-v3's, the encoder stack's width and heads."""
    d_model: int = 1280
    heads: int = 20
    ffn: int = 5120
    layers: int = 32
    vocab: int = 51866
    max_tokens: int = 448
    source_tokens: int = 1500
    eps: float = 1e-5

    @property
    def head_dim(self) -> int:
        return self.d_model // self.heads


def random_decoder_weights(cfg: DecoderConfig, device, seed: int = 1234, std: float = 0.02) -> Dict[str, torch.Tensor]:
    """Random-init fp16 weights by name: linears [out, in] and biases ~ N(0, std), LayerNorm gamma 1 beta 0, drawn in
    order on `device` from one generator."""
    dev = torch.device(device)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    D, F = cfg.d_model, cfg.ffn

    def n(*shape):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * std).half()

    w = {"embed": n(cfg.vocab, D), "positions": n(cfg.max_tokens, D)}
    for i in range(cfg.layers):
        for name, out, inp in (("qkv", 3 * D, D), ("o", D, D), ("xq", D, D), ("xkv", 2 * D, D), ("xo", D, D),
                               ("fc1", F, D), ("fc2", D, F)):
            w[f"{i}.{name}.w"], w[f"{i}.{name}.b"] = n(out, inp), n(out)
        for name in ("ln1", "ln2", "ln3"):
            w[f"{i}.{name}.g"], w[f"{i}.{name}.b"] = torch.ones_like(w["embed"][0]), torch.zeros_like(w["embed"][0])
    w["ln.g"], w["ln.b"] = torch.ones_like(w["embed"][0]), torch.zeros_like(w["embed"][0])
    return w


_TURN = threading.RLock()
_LAST: Dict[int, tuple] = {}  # by device index: the stream of the last decoder call, an event behind it


@contextlib.contextmanager
def _turn(device: torch.device):
    """Work issued in here runs, on the GPU, after what was issued in here before it for that device, on whatever
    stream: the decoders of a device share the workspaces of its linears and of its attention, which calls that
    run at the same time must not, and their grid-wide linears need the SMs that another's could hold."""
    with _TURN, torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            yield
            return
        index, stream = torch.cuda.current_device(), torch.cuda.current_stream()
        stream_before, event = _LAST.get(index, (stream, None))
        if stream_before != stream:
            stream.wait_event(event)
        try:
            yield
        finally:
            event = torch.cuda.Event()
            event.record(stream)
            _LAST[index] = (stream, event)


def _in_turn(fn):
    @functools.wraps(fn)
    def call(self, *args, **kwargs):
        with _turn(self.device):
            return fn(self, *args, **kwargs)
    return call


class Kv8Decoder:
    """See the module's description. One instance runs one batch at a time, on one stream. Instances on one device take
    turns, whatever their streams and threads; other calls of ops.linear_fp8, gemm_fp8 and attention_kv8 that may run
    at the same time need workspaces of their own."""

    def __init__(self, cfg: DecoderConfig, weights: Dict[str, torch.Tensor], device, block: int = 64,
                 fmt: str = "e4m3") -> None:
        self.cfg, self.block, self.fmt = cfg, block, fmt
        self.device = torch.device(device)
        self.w = {k: t.to(self.device) for k, t in weights.items()}
        with _turn(self.device):
            # FP8 once; the fp16 originals of the linears are dropped, the embedding's stays for the lookup
            self.q = {k[:-2]: ops.quantise(t.contiguous()) for k, t in self.w.items() if k.endswith(".w")}
            self.q["vocab"] = ops.quantise(self.w["embed"].contiguous())
        self.w = {k: t for k, t in self.w.items() if not k.endswith(".w")}
        self.own: Optional[Kv8Cache] = None
        self.source: Optional[Kv8Cache] = None
        self._step: Optional[dict] = None
        self._most = 0  # tokens that the longest sequence holds, at most: the host's count, padding included

    def _make_room(self, T: int, new_lens: Optional[torch.Tensor]) -> None:
        """Raises if T tokens more, or new_lens of them, are more than the positions of a sequence. The lengths are on the
        device: they are looked at, and waited for, only where the host's count does not say. (What a caller's own graph
        of logits() appends in its replays is not counted.)"""
        if torch.cuda.is_current_stream_capturing():
            return
        if self._most + T > self.cfg.max_tokens:
            most = int((self.own.lens + (T if new_lens is None else new_lens)).max())
            if most > self.cfg.max_tokens:
                raise ValueError(f"{T} more tokens make a sequence of {most}; the decoder holds {self.cfg.max_tokens}")
            self._most = most
        else:
            self._most += T

    def _linear(self, name: str, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                epilogue: str = "none") -> torch.Tensor:
        codes, scale = self.q[name]
        return ops.linear_fp8(x, codes, scale, self.w.get(f"{name}.b"), residual,
                              "residual" if residual is not None else epilogue)[0]

    def _norm(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return ops.layernorm(x, None, self.w[f"{name}.g"], self.w[f"{name}.b"], self.cfg.eps)[0]

    def _heads(self, x: torch.Tensor, B: int, parts: int) -> List[torch.Tensor]:
        """The [B, H, T, D] views of a projection's output [B * T, parts * d_model]."""
        x = x.view(B, -1, parts, self.cfg.heads, self.cfg.head_dim)
        return [x[:, :, i].transpose(1, 2) for i in range(parts)]

    @_in_turn
    @torch.inference_mode()
    def start(self, states: torch.Tensor, state_lens: Optional[torch.Tensor] = None) -> None:
        """Project the encoder's states [B, S, d_model] fp16 into each layer's cross cache and empty the other.
        state_lens [B] int32: how many of the S are real (default: all)."""
        cfg = self.cfg
        B, S, _ = states.shape
        if S > cfg.source_tokens:
            raise ValueError(f"{S} encoder states; the decoder is made for {cfg.source_tokens}")
        if self.own is None or self.own.batch != B:
            self._step = None  # the captured step holds the addresses of the caches being replaced
            args = (cfg.layers, B, cfg.heads, cfg.head_dim)
            with torch.inference_mode(False):  # caches that a caller may write to outside it, too
                self.own = Kv8Cache(*args, cfg.max_tokens, self.device, self.block, self.fmt)
                self.source = Kv8Cache(*args, cfg.source_tokens, self.device, self.block, self.fmt)
        self.own.lens.zero_()
        self._most = 0
        self.source.lens.zero_()
        if state_lens is not None:
            state_lens = state_lens.clamp(0, S)  # as kv8_append takes them
        x = states.reshape(B * S, cfg.d_model)
        for i in range(cfg.layers):
            k, v = self._heads(self._linear(f"{i}.xkv", x), B, 2)
            self.source.append(i, k, v, state_lens)
        self.source.advance(S if state_lens is None else state_lens)

    @_in_turn
    @torch.inference_mode()
    def logits(self, tokens: torch.Tensor, new_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Run tokens [B, T] int64 behind those already held; fp16 logits [B, vocab] after each sequence's last.
        new_lens [B] int32: how many of the T are real (default: all). ValueError where a sequence would have more
        than max_tokens."""
        cfg, own, source = self.cfg, self.own, self.source
        B, T = tokens.shape
        if new_lens is not None:
            new_lens = new_lens.clamp(0, T)  # as kv8_append takes them
        self._make_room(T, new_lens)
        at = own.lens.long()[:, None] + torch.arange(T, device=self.device)
        h = (self.w["embed"][tokens] + self.w["positions"][at.clamp_(max=cfg.max_tokens - 1)]).view(B * T, cfg.d_model)
        held = own.lens + (T if new_lens is None else new_lens)
        attn = torch.empty(B, T, cfg.heads, cfg.head_dim, dtype=torch.float16, device=self.device)
        flat, out = attn.view(B * T, cfg.d_model), attn.transpose(1, 2)
        for i in range(cfg.layers):
            q, k, v = self._heads(self._linear(f"{i}.qkv", self._norm(f"{i}.ln1", h)), B, 3)
            own.append(i, k, v, new_lens)
            own.attend(i, q, held, new_lens, out=out)
            h = self._linear(f"{i}.o", flat, residual=h)
            q, = self._heads(self._linear(f"{i}.xq", self._norm(f"{i}.ln2", h)), B, 1)
            source.attend(i, q, source.lens, new_lens, causal=False, out=out)
            h = self._linear(f"{i}.xo", flat, residual=h)
            f = self._linear(f"{i}.fc1", self._norm(f"{i}.ln3", h), epilogue="gelu")
            h = self._linear(f"{i}.fc2", f, residual=h)
        own.advance(T if new_lens is None else new_lens)
        h = h.view(B, T, cfg.d_model)
        last = h[:, -1] if new_lens is None else h[torch.arange(B, device=self.device), (new_lens.long() - 1).clamp(min=0)]
        return self._linear("vocab", self._norm("ln", last.contiguous()))

    @_in_turn
    @torch.inference_mode()
    def step(self, tokens: torch.Tensor, new_lens: Optional[torch.Tensor] = None,
             **settings) -> Tuple[torch.Tensor, torch.Tensor]:
        """logits(), then ops.sample with fresh random numbers and the settings given: (next tokens, log-probabilities)."""
        x = self.logits(tokens, new_lens)
        return ops.sample(x, torch.empty_like(x, dtype=torch.float32).exponential_(), **settings)

    def _captured_step(self, settings: dict) -> dict:
        """The graph of one step. To be called between start() and the prompt: the step that is run before the capture
        writes at the start of empty sequences' first pages, which the prompt's append then starts afresh. (Behind a
        prompt it could raise a page's scale and re-code the prompt's tokens.)"""
        key = tuple(sorted((k, v.data_ptr() if isinstance(v, torch.Tensor) else v) for k, v in settings.items()))
        if self._step is None or self._step["key"] != key:
            B = self.own.batch
            token = torch.zeros(B, 1, dtype=torch.int64, device=self.device)
            draws = torch.cuda.get_rng_state(self.device)
            self.step(token, **settings)  # every first-time initialisation
            self.own.lens.zero_()
            self._most = 0
            torch.cuda.set_rng_state(draws, self.device)  # as if it had not been
            torch.cuda.synchronize(self.device)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                drawn, logprob = self.step(token, **settings)
                token.copy_(drawn.clamp(min=0)[:, None])
            # `settings` keeps the tensors alive that the graph reads
            self._step = {"key": key, "graph": graph, "token": token, "drawn": drawn, "logprob": logprob,
                          "settings": settings}
        return self._step

    @_in_turn
    @torch.inference_mode()
    def generate(self, states: torch.Tensor, prompt: torch.Tensor, count: int,
                 state_lens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                 **settings) -> Tuple[torch.Tensor, torch.Tensor]:
        """`count` tokens for each prompt [B, T] int64: (tokens int64 [B, count], log-probabilities fp32 [B, count]).

        settings: temperature, top_k, top_p, min_p as ops.sample takes them; draws
        come from the device's default generator."""
        T = prompt.shape[1]
        if count < 1 or T < 1 or T + count - 1 > self.cfg.max_tokens:
            raise ValueError(f"{T} prompt tokens and {count} new ones; the decoder holds {self.cfg.max_tokens}")
        self.start(states, state_lens)
        tokens = torch.empty(prompt.shape[0], count, dtype=torch.int64, device=self.device)
        logprobs = torch.empty(prompt.shape[0], count, dtype=torch.float32, device=self.device)
        s = self._captured_step(settings) if count > 1 else None
        drawn, lp = self.step(prompt, prompt_lens, **settings)
        tokens[:, 0], logprobs[:, 0] = drawn, lp
        if count > 1:
            s["token"].copy_(drawn.clamp(min=0)[:, None])
            self._most += count - 1
            for i in range(1, count):
                s["graph"].replay()
                tokens[:, i], logprobs[:, i] = s["drawn"], s["logprob"]
        return tokens, logprobs
