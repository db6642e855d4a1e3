"""The capture of a decoder's step leaves the caches, and with them the answer, as they are without it.

Everything compared here is computed by the same kernels from the same inputs, which give equal bits: no tolerance.
"""
import pytest
import torch

from whisper_blaze_b200.decoding import DecoderConfig, Kv8Decoder, random_decoder_weights

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(d_model=256, heads=4, ffn=512, layers=2, vocab=1003, max_tokens=96, source_tokens=70)


@pytest.fixture
def setup(cuda_device):
    """Weights with which token 0, and no other, has keys and values far above the others': only its embedding has
    anything in channel 7 of the first layer's input, whose weights are large."""
    w = random_decoder_weights(CFG, cuda_device, std=0.1)
    w["positions"] *= 0.01
    w["embed"][:, 7] = 0
    w["positions"][:, 7] = 0
    w["embed"][0] = 0
    w["embed"][0, 7] = 1
    w["0.qkv.w"][CFG.d_model:, 7] *= 30
    g = torch.Generator(device=cuda_device).manual_seed(6)
    states = torch.randn(3, CFG.source_tokens, CFG.d_model, generator=g, device=cuda_device).half()
    prompt = torch.randint(1, CFG.vocab, (3, 5), generator=g, device=cuda_device)
    return w, states, prompt


def _held(decoder, n):
    """Scales and codes of the first n tokens, which lie in each sequence's first page."""
    pages = decoder.own.block_table[:, 0].long()
    return decoder.own.scales[:, :, pages].clone(), decoder.own.codes[:, :, pages, :, :n].clone()


@pytest.mark.parametrize("block,fmt", [(64, "e4m3"), (16, "e5m2")])
def test_the_capturing_call_answers_as_the_others(setup, cuda_device, block, fmt):
    w, states, prompt = setup
    decoder = Kv8Decoder(CFG, w, cuda_device, block, fmt)
    count = 7  # the prompt and all of them lie in one page
    first, lp_first = decoder.generate(states, prompt, count, temperature=0.0)
    captured = _held(decoder, 5 + count - 1)
    again, lp_again = decoder.generate(states, prompt, count, temperature=0.0)
    replayed = _held(decoder, 5 + count - 1)
    decoder.start(states)
    x, steps = prompt, []
    for _ in range(count):
        x = decoder.logits(x).argmax(-1, keepdim=True)
        steps.append(x)
    stepped = _held(decoder, 5 + count - 1)
    assert int(first.min()) > 0, "token 0 was drawn: the inputs do not show anything"
    for got in (captured, replayed):
        assert torch.equal(got[0], stepped[0]), "page scales"
        assert torch.equal(got[1], stepped[1]), "codes"
    assert torch.equal(first, torch.cat(steps, 1)) and torch.equal(again, first) and torch.equal(lp_again, lp_first)
