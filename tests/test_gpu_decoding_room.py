"""A decoder's sequences hold max_tokens tokens: a call that would pass that is refused and changes nothing."""
import pytest
import torch

from whisper_blaze_b200.decoding import DecoderConfig, Kv8Decoder, random_decoder_weights

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(d_model=256, heads=4, ffn=512, layers=1, vocab=501, max_tokens=24, source_tokens=20)


@pytest.fixture
def setup(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(9)
    states = torch.randn(2, CFG.source_tokens, CFG.d_model, generator=g, device=cuda_device).half()
    tokens = torch.randint(CFG.vocab, (2, 40), generator=g, device=cuda_device)
    return Kv8Decoder(CFG, random_decoder_weights(CFG, cuda_device, std=0.1), cuda_device, block=16), states, tokens


def _i32(tokens, values):
    return torch.tensor(values, dtype=torch.int32, device=tokens.device)


def test_the_last_position_is_used_and_the_next_refused(setup):
    decoder, states, tokens = setup
    decoder.start(states)
    decoder.logits(tokens[:, :20])
    for i in range(20, 24):
        decoder.logits(tokens[:, i:i + 1])
    held = decoder.own.codes.clone()
    for call in (decoder.logits, decoder.step):
        with pytest.raises(ValueError, match="holds 24"):
            call(tokens[:, :1])
    assert decoder.own.lens.tolist() == [24, 24] and torch.equal(decoder.own.codes, held)
    decoder.start(states)
    with pytest.raises(ValueError, match="holds 24"):
        decoder.logits(tokens[:, :25])
    decoder.logits(tokens[:, :24])


def test_padding_does_not_count(setup):
    """The padded lengths pass the limit, the sequences do not; a padded call answers as an unpadded one."""
    decoder, states, tokens = setup
    decoder.start(states)
    decoder.logits(tokens, _i32(tokens, [20, 3]))  # 40 wide
    decoder.logits(tokens[:, :10], _i32(tokens, [4, 10]))
    assert decoder.own.lens.tolist() == [24, 13]
    with pytest.raises(ValueError, match="holds 24"):
        decoder.logits(tokens[:, :10], _i32(tokens, [1, 0]))
    decoder.logits(tokens[:, :1], _i32(tokens, [0, 1]))
    assert decoder.own.lens.tolist() == [24, 14]


def test_what_a_graph_appended_counts(setup):
    decoder, states, tokens = setup
    decoder.generate(states, tokens[:, :10], 15, temperature=0.0)  # the last token drawn is not stored
    assert decoder.own.lens.tolist() == [24, 24]
    with pytest.raises(ValueError, match="holds 24"):
        decoder.logits(tokens[:, :1])
    decoder.generate(states, tokens[:, :10], 10, temperature=0.0)
    decoder.logits(tokens[:, :5])
    with pytest.raises(ValueError, match="holds 24"):
        decoder.logits(tokens[:, :1])


def test_counts_beyond_what_is_given_are_all_of_it(setup):
    """As kv8_append takes them: more than T is T, less than none is none; the lengths say what the caches hold."""
    decoder, states, tokens = setup
    decoder.start(states[:, :15], _i32(tokens, [15, 0]))
    want = decoder.logits(tokens[:, :8], _i32(tokens, [8, 0]))
    then = decoder.logits(tokens[:, 8:9])
    decoder.start(states[:, :15], _i32(tokens, [20, -3]))
    assert decoder.source.lens.tolist() == [15, 0]
    got = decoder.logits(tokens[:, :8], _i32(tokens, [11, -2]))
    assert decoder.own.lens.tolist() == [8, 0]
    assert torch.equal(got, want) and torch.equal(decoder.logits(tokens[:, 8:9]), then)
