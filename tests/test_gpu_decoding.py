"""A decoder on 8-bit caches: the cache's operators, the FP8 linears and the sampler used together.

The reference is the same decoder in fp32 whose linears round both operands to
8 bits as the decoder's do (ops.quantise, tested by itself), with keys and
values that are not rounded. Tolerance on the logits' relative L2 error: an
e4m3 code is off by at most 2^-4 of its value, uniformly, so by 2^-4 / sqrt(3) =
0.036 rms at the worst mantissa and about 0.026 on average. A product of two
quantised operands is off by sqrt(2) * 0.026 = 0.037, and a residual branch with
two or three products in a row and the cache's own rounding in between by at
most 0.037 * sqrt(3) + 0.026 = 0.09 of itself. The residual stream is a sum of
such branches, so it is off by at most 0.09 of itself per layer: 0.09 * sqrt(2)
for two layers, with the vocabulary product 0.13. The gate is 0.2; a branch left
out or a token misplaced is off by a large part of 1.

(An unrounded fp32 decoder is further away than that: here the scores of the
attention have a standard deviation of several units, and the softmax passes an
error of a score on as a factor.)
"""
import pytest
import torch
import torch.nn.functional as F

from whisper_blaze_b200 import _lib, ops
from whisper_blaze_b200.decoding import DecoderConfig, Kv8Decoder, random_decoder_weights

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(d_model=256, heads=4, ffn=512, layers=2, vocab=1003, max_tokens=96, source_tokens=70)
GATE = 0.2


class Reference:
    """The decoder in fp32: logits() as Kv8Decoder's, keys and values per sequence in fp32."""

    def __init__(self, decoder, w, states, state_lens=None):
        self.cfg, self.w = decoder.cfg, {k: t.float() for k, t in w.items()}
        self.weights = {name: self._rounded(w["embed"] if name == "vocab" else w[f"{name}.w"]) for name in decoder.q}
        B, S, _ = states.shape
        self.real = state_lens or [S] * B
        self.cross = []
        for i in range(self.cfg.layers):
            self.cross.append(self._heads(self._linear(f"{i}.xkv", states), 2))
        self.own = [[[None, None] for _ in range(B)] for _ in range(self.cfg.layers)]
        self.lens = [0] * B

    @staticmethod
    def _rounded(x):
        codes, scale = ops.quantise(x.half().contiguous())
        return codes.view(torch.float8_e4m3fn).float() * scale

    def _linear(self, name, x):
        return F.linear(self._rounded(x), self.weights[name], self.w.get(f"{name}.b"))

    def _norm(self, name, x):
        return F.layer_norm(x, (self.cfg.d_model,), self.w[f"{name}.g"], self.w[f"{name}.b"], self.cfg.eps)

    def _heads(self, x, parts):
        x = x.view(x.shape[0], -1, parts, self.cfg.heads, self.cfg.head_dim)
        return [x[:, :, i].transpose(1, 2) for i in range(parts)]

    def logits(self, tokens, new_lens=None):
        cfg, w = self.cfg, self.w
        B, T = tokens.shape
        n = new_lens or [T] * B
        at = torch.tensor(self.lens, device=tokens.device)[:, None] + torch.arange(T, device=tokens.device)
        h = w["embed"][tokens] + w["positions"][at.clamp(max=cfg.max_tokens - 1)]
        for i in range(cfg.layers):
            q, k, v = self._heads(self._linear(f"{i}.qkv", self._norm(f"{i}.ln1", h)), 3)
            y = torch.zeros_like(q)
            for b in range(B):
                held = self.own[i][b]
                for j, x in enumerate((k, v)):
                    x = x[b, :, :n[b]]
                    held[j] = x if held[j] is None else torch.cat([held[j], x], 1)
                mask = torch.ones(n[b], held[0].shape[1], dtype=torch.bool, device=q.device).tril(held[0].shape[1] - n[b])
                y[b, :, :n[b]] = F.scaled_dot_product_attention(q[b, :, :n[b]], held[0], held[1], attn_mask=mask)
            h = h + self._linear(f"{i}.o", y.transpose(1, 2).reshape(B, T, -1))
            q, = self._heads(self._linear(f"{i}.xq", self._norm(f"{i}.ln2", h)), 1)
            y = torch.zeros_like(q)
            for b in range(B):
                k, v = (x[b, :, :self.real[b]] for x in self.cross[i])
                y[b, :, :n[b]] = F.scaled_dot_product_attention(q[b, :, :n[b]], k, v)
            h = h + self._linear(f"{i}.xo", y.transpose(1, 2).reshape(B, T, -1))
            h = h + self._linear(f"{i}.fc2", F.gelu(self._linear(f"{i}.fc1", self._norm(f"{i}.ln3", h))))
        self.lens = [a + b for a, b in zip(self.lens, n)]
        last = torch.stack([h[b, n[b] - 1] for b in range(B)])
        return self._linear("vocab", self._norm("ln", last))


@pytest.fixture
def setup(cuda_device):
    w = random_decoder_weights(CFG, cuda_device, std=0.1)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    states = torch.randn(3, CFG.source_tokens, CFG.d_model, generator=g, device=cuda_device).half()
    tokens = torch.randint(CFG.vocab, (3, 40), generator=g, device=cuda_device)
    return Kv8Decoder(CFG, w, cuda_device), w, states, tokens


def _error(x, ref):
    return ((x.float() - ref).norm() / ref.norm()).item()


def test_prompt_then_tokens_match_the_fp32_decoder(setup):
    decoder, w, states, tokens = setup
    reference = Reference(decoder, w, states)
    decoder.start(states)
    assert _error(decoder.logits(tokens[:, :33]), reference.logits(tokens[:, :33])) <= GATE
    for i in range(33, 40):
        assert _error(decoder.logits(tokens[:, i:i + 1]), reference.logits(tokens[:, i:i + 1])) <= GATE
    assert decoder.own.lens.tolist() == [40] * 3 and _lib.device_error() == 0


def test_ragged_prompts_and_states(setup):
    decoder, w, states, tokens = setup
    lens, real = [40, 7, 1], [70, 33, 64]
    i32 = dict(dtype=torch.int32, device=tokens.device)
    reference = Reference(decoder, w, states, real)
    decoder.start(states, torch.tensor(real, **i32))
    got, ref = decoder.logits(tokens, torch.tensor(lens, **i32)), reference.logits(tokens, lens)
    for b in range(3):
        assert _error(got[b], ref[b]) <= GATE
    assert decoder.own.lens.tolist() == lens and decoder.source.lens.tolist() == real
    got, ref = decoder.logits(tokens[:, :1]), reference.logits(tokens[:, :1])
    for b in range(3):
        assert _error(got[b], ref[b]) <= GATE


def test_generate_is_the_steps_it_replays(setup):
    """Greedy: the graph's tokens are those of steps made one at a time. Sampled: the same seed gives the same tokens,
    and another setting its own."""
    decoder, _, states, tokens = setup
    got, logprobs = decoder.generate(states, tokens[:, :5], 12, temperature=0.0)
    decoder.start(states)
    x = tokens[:, :5]
    for i in range(12):
        logits = decoder.logits(x)
        x = logits.argmax(-1, keepdim=True)
        assert torch.equal(got[:, i], x[:, 0])
        # the log-probability is the fp32 log-softmax of these logits: sums of 1003 terms, an approximate exponential
        want = torch.log_softmax(logits.double(), -1).gather(1, x)[:, 0]
        assert (logprobs[:, i].double() - want).abs().max() <= 1e-4
    torch.manual_seed(7)
    a, _ = decoder.generate(states, tokens[:, :5], 12, temperature=1.0, top_k=50)
    torch.manual_seed(7)
    decoder.start(states)
    first, _ = decoder.step(tokens[:, :5], temperature=1.0, top_k=50)
    assert torch.equal(a[:, 0], first) and int(a.min()) >= 0 and int(a.max()) < CFG.vocab
    torch.manual_seed(7)
    b, _ = decoder.generate(states, tokens[:, :5], 12, temperature=1.0, top_k=50)
    assert torch.equal(a, b)
    c, _ = decoder.generate(states, tokens[:, :5], 12, temperature=0.0)
    assert torch.equal(c, got)


def test_refuses_more_than_it_holds(setup):
    decoder, _, states, tokens = setup
    with pytest.raises(ValueError, match="holds 96"):
        decoder.generate(states, tokens, 60)
    with pytest.raises(ValueError, match="made for 70"):
        decoder.start(torch.cat([states, states], 1))


# ------------------------------------------------ calls, workspaces, give-ups

def _long(dev, queries, kv_heads=2, group=4, seed=3, blocks=60):
    g = torch.Generator(device=dev).manual_seed(seed)
    B, D = 4, 64
    codes = [torch.randint(0, 120, (B * blocks, kv_heads, 64, D), generator=g, device=dev).to(torch.uint8) for _ in "kv"]
    scales = [torch.full((B * blocks, kv_heads), 2.0 ** -7, device=dev) for _ in "kv"]
    table = torch.arange(B * blocks, dtype=torch.int32, device=dev).view(B, blocks)
    lens = torch.tensor([blocks * 64, 1000, 1, 2500], dtype=torch.int32, device=dev)
    q = torch.randn(B, kv_heads * group, queries, D, generator=g, device=dev).half()
    return q, *codes, *scales, table, lens


@pytest.mark.parametrize("queries,sites", [(1, range(41, 43)), (64, range(51, 56))])
def test_attention_gives_up_with_a_status_and_the_next_call_is_right(cuda_device, queries, sites):
    """Both kernels' bounded waits run out at a limit of 1 ns; what is in flight is waited for, the host reads the
    status, the shared workspace is zero again. (Long caches, and L2 flushed, so that the loads are behind.)"""
    flush = torch.empty(1 << 29, dtype=torch.uint8, device=cuda_device)
    args = _long(cuda_device, queries, kv_heads=8, blocks=1000)
    want = ops.attention_kv8(*args)
    assert _lib.device_error() == 0
    code = 0
    try:
        _lib.set_wait_timeout_ns(1)
        for _ in range(10):
            flush.zero_()
            ops.attention_kv8(*args)
            code = _lib.device_error()
            if code:
                break
    finally:
        _lib.set_wait_timeout_ns(0)
    assert code & 0xFF == _lib.WBK_ERR_DEVICE_TIMEOUT, f"no device timeout reported (word {code:#x})"
    assert (code >> 8) in sites, f"site {code >> 8}"
    assert int(ops.kv8_workspace(cuda_device.index or 0).count_nonzero().item()) == 0
    assert torch.equal(ops.attention_kv8(*args), want)
    assert _lib.device_error() == 0


def test_shared_workspace_stays_where_it_is(cuda_device):
    """A graph that holds its address stays right when a call that needs more follows."""
    args = _long(cuda_device, 1)
    want = ops.attention_kv8(*args)
    ws = ops.kv8_workspace(cuda_device.index or 0)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_kv8(*args, out=out)
    ops.attention_kv8(*_long(cuda_device, 64))
    graph.replay()
    assert torch.equal(out, want)
    assert ops.kv8_workspace(cuda_device.index or 0) is ws


def test_workspace_of_ones_own(cuda_device):
    args = _long(cuda_device, 64)
    need = _lib.lib().wbk_attention_kv8_ws_bytes(4, 8, 2, 64, 64)
    own = torch.zeros(need, dtype=torch.uint8, device=cuda_device)
    assert torch.equal(ops.attention_kv8(*args, workspace=own), ops.attention_kv8(*args))
    with pytest.raises((RuntimeError, ValueError), match="workspace"):
        ops.attention_kv8(*args, workspace=own[:need - 256])
    for scale in (-0.5, float("inf"), float("nan")):
        with pytest.raises((RuntimeError, ValueError), match="scale"):
            ops.attention_kv8(*args, scale=scale)


@pytest.mark.parametrize("queries", [1, 40])
def test_a_scale_of_zero_gives_the_mean(cuda_device, queries):
    q, kc, vc, ks, vs, table, lens = _long(cuda_device, queries)
    y = ops.attention_kv8(q, kc, vc, ks, vs, table, lens, causal=False, scale=0.0)
    v = vc.view(torch.float8_e4m3fn).double() * vs.double()[..., None, None]
    for b, n in enumerate(lens.tolist()):
        mean = v[table[b].long()].transpose(0, 1).reshape(2, -1, 64)[:, :n].mean(1)
        # equal weights are exact; fp32 sums of at most 3840 positive values, and the output rounded to 11 bits
        assert ((y[b].double() - mean.repeat_interleave(4, 0)[:, None]).abs() <= 2.0 ** -10 * mean.repeat_interleave(4, 0)[:, None]).all()


def test_the_short_call_path_and_the_checked_one_agree(cuda_device, monkeypatch):
    """Well-formed calls go through the extension module; the Python path, which makes the others' checks and errors,
    gives the same results."""
    g = torch.Generator(device=cuda_device).manual_seed(11)
    q, kc, vc, ks, vs, table, lens = _long(cuda_device, 2)
    kv = torch.randn(2, 4, 3, 2, 64, generator=g, device=cuda_device).half().transpose(2, 3)
    logits = torch.randn(5, 777, generator=g, device=cuda_device)
    noise = torch.empty_like(logits).exponential_(generator=g)
    few = torch.tensor([3, 0, 2, 1], dtype=torch.int32, device=cuda_device)

    def run():
        cache = [t.clone() for t in (kc, vc, ks, vs)]
        ops.kv8_append(kv[0], kv[1], *cache, table, (lens - 3).clamp(min=0), few)
        out = torch.empty(4, 2, 8, 64, dtype=torch.float16, device=cuda_device).transpose(1, 2)
        return [*cache, ops.attention_kv8(q, *cache, table, lens, causal=False, scale=0.1),
                ops.attention_kv8(q, *cache, table, lens, few.clamp(max=2), out=out), out,
                *ops.sample(logits, noise, 0.8, 40, 0.9), *ops.sample(logits.half(), noise, top_k=few[0].repeat(5))]

    assert ops._short() is not None
    short = run()
    monkeypatch.setattr(ops, "_SHORT", [None])
    checked = run()
    assert all(torch.equal(a, b) for a, b in zip(short, checked))
