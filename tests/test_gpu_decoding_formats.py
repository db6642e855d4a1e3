"""The decoder in both formats of the cache and all page sizes, against the reference of test_gpu_decoding.py with keys
and values rounded as the cache's definition says (oracle.decode, on the CPU).

The gate is test_gpu_decoding's, whose derivation allows for the cache's rounding; here that is in the reference,
and what remains are roundings to 16 bits and the 8-bit codes that these move to the next one.
"""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import decode, fp8
from test_gpu_decoding import CFG, GATE, Reference, _error
from whisper_blaze_b200 import _lib
from whisper_blaze_b200.decoding import Kv8Decoder, random_decoder_weights

pytestmark = pytest.mark.gpu


class Pages:
    """Keys or values of one layer and sequence, in pages."""

    def __init__(self, block, fmt, tokens):
        pages = -(-tokens // block)
        self.fmt, self.len = {"e4m3": fp8.E4M3, "e5m2": fp8.E5M2}[fmt], 0
        self.codes = np.zeros((pages, CFG.heads, block, CFG.head_dim), np.uint8)
        self.scales = np.ones((pages, CFG.heads), np.float32)

    def add(self, x):
        """Appends x [H, n, D]; all tokens held, as the codes have them."""
        decode.append_one(x.half().float().cpu().numpy(), self.codes, self.scales, np.arange(len(self.codes)), self.len, self.fmt)
        self.len += x.shape[1]
        values = fp8.decode(self.codes, self.fmt).astype(np.float32) * self.scales[..., None, None]
        held = values.transpose(1, 0, 2, 3).reshape(CFG.heads, -1, CFG.head_dim)[:, :self.len]
        return torch.from_numpy(np.ascontiguousarray(held)).to(x.device)


class Rounded(Reference):
    def __init__(self, decoder, w, states):
        super().__init__(decoder, w, states)
        B, (block, fmt) = states.shape[0], (decoder.block, decoder.fmt)
        self.cross = [[torch.stack([Pages(block, fmt, CFG.source_tokens).add(x[b]) for b in range(B)]) for x in kv]
                      for kv in self.cross]
        self.pages = [[[Pages(block, fmt, CFG.max_tokens) for _ in "kv"] for _ in range(B)] for _ in range(self.cfg.layers)]

    def logits(self, tokens):
        w, (B, T) = self.w, tokens.shape
        at = self.pages[0][0][0].len
        h = w["embed"][tokens] + w["positions"][at:at + T]
        for i in range(self.cfg.layers):
            q, k, v = self._heads(self._linear(f"{i}.qkv", self._norm(f"{i}.ln1", h)), 3)
            k, v = (torch.stack([self.pages[i][b][j].add(x[b]) for b in range(B)]) for j, x in enumerate((k, v)))
            mask = torch.ones(T, at + T, dtype=torch.bool, device=q.device).tril(at)
            y = F.scaled_dot_product_attention(q, k, v, attn_mask=mask)
            h = h + self._linear(f"{i}.o", y.transpose(1, 2).reshape(B, T, -1))
            q, = self._heads(self._linear(f"{i}.xq", self._norm(f"{i}.ln2", h)), 1)
            y = F.scaled_dot_product_attention(q, *self.cross[i])
            h = h + self._linear(f"{i}.xo", y.transpose(1, 2).reshape(B, T, -1))
            h = h + self._linear(f"{i}.fc2", F.gelu(self._linear(f"{i}.fc1", self._norm(f"{i}.ln3", h))))
        return self._linear("vocab", self._norm("ln", h[:, -1]))


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_prompt_then_tokens(cuda_device, fmt, block):
    w = random_decoder_weights(CFG, cuda_device, std=0.1)
    g = torch.Generator(device=cuda_device).manual_seed(15)
    states = torch.randn(3, CFG.source_tokens, CFG.d_model, generator=g, device=cuda_device).half()
    tokens = torch.randint(CFG.vocab, (3, 40), generator=g, device=cuda_device)
    decoder = Kv8Decoder(CFG, w, cuda_device, block, fmt)
    reference = Rounded(decoder, w, states)
    decoder.start(states)
    errors = [_error(decoder.logits(tokens[:, :33]), reference.logits(tokens[:, :33]))]
    for i in range(33, 40):
        errors.append(_error(decoder.logits(tokens[:, i:i + 1]), reference.logits(tokens[:, i:i + 1])))
    assert max(errors) <= GATE, errors
    assert _lib.device_error() == 0
