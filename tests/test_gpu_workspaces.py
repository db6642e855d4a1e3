"""Workspaces and captured graphs on the GPU: what a graph holds the address of stays its own."""
import pytest
import torch

from conftest import randn_f16
from whisper_blaze_b200 import _lib, ops
from whisper_blaze_b200.decoding import DecoderConfig, Kv8Decoder, random_decoder_weights

pytestmark = pytest.mark.gpu


def _linear(dev, M, N, K, seed):
    x = randn_f16((M, K), seed).to(dev)
    w, scale = ops.quantise(randn_f16((N, K), seed + 1, std=0.02).to(dev))
    return x, w, scale


def test_a_graph_of_linears_outlives_a_larger_call(cuda_device, monkeypatch):
    """Captured with the smallest shared workspace; a later call needs a larger one, and tensors that could have taken the
    first one's memory are neither read nor written by the replays."""
    for name in ("_SPLITK_WS", "_SPLITK_OUTGROWN"):
        monkeypatch.setattr(ops, name, {})
    args = _linear(cuda_device, 64, 1280, 1280, 60)
    need = int(_lib.lib().wbk_gemm_fp8_ws_bytes(64, 1280, 1280))
    want = ops.linear_fp8(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_fp8(*args)
    larger = _linear(cuda_device, 8, 1280, 5120, 70)
    assert int(_lib.lib().wbk_gemm_fp8_ws_bytes(8, 1280, 5120)) > need
    first = ops.linear_fp8(*larger)
    marks = [torch.full((need,), 0x5A, dtype=torch.uint8, device=cuda_device) for _ in range(64)]
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(bool((m == 0x5A).all()) for m in marks)
    assert all(torch.equal(a, b) for a, b in zip(ops.linear_fp8(*larger), first))
    assert _lib.device_error() == 0


# ------------------------------------------------------------ two decoders

CFG = DecoderConfig(d_model=256, heads=4, ffn=2048, layers=2, vocab=1003, max_tokens=200, source_tokens=70)


def _decoder(dev, seed, batch=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    decoder = Kv8Decoder(CFG, random_decoder_weights(CFG, dev, seed=seed, std=0.1), dev)
    states = torch.randn(batch, CFG.source_tokens, CFG.d_model, generator=g, device=dev).half()
    prompt = torch.randint(CFG.vocab, (batch, 40), generator=g, device=dev)
    return decoder, states, prompt


def test_two_decoders_on_two_streams(cuda_device):
    """Issued together they give what each gives alone."""
    both = [_decoder(cuda_device, 81), _decoder(cuda_device, 82, batch=2)]
    alone = [d.generate(s, p, 60, temperature=0.0) for d, s, p in both]
    streams = [torch.cuda.Stream(cuda_device) for _ in both]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for (d, s, p), stream in zip(both, streams):
            with torch.cuda.stream(stream):
                got.append(d.generate(s, p, 60, temperature=0.0))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert _lib.device_error() == 0
