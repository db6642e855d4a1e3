"""GPU parity of ops.sample against its definition in 64 bits (oracle.decode.sample_one).

Gates: tokens equal. The kernel's fp32 masses and scores are within 2^-20 or so of the 64-bit ones, so a token could
differ only where the two best scores, or a mass and its threshold at the winner, agree to that: the seeded inputs below
have no such row. logprob: |y - ref| <= 2^-20 (1 + |ref|): one fp32 subtraction, a logarithm, and a sum of fp32
exponentials whose rounding errors are below 2^-21 relative.
"""
import math

import numpy as np
import pytest
import torch

from conftest import seeded
from oracle import decode
from whisper_blaze_b200 import ops

pytestmark = pytest.mark.gpu


def _inputs(dev, rows, vocab, seed, dtype=torch.float16, std=2.0, likely=40):
    g = seeded(seed)
    x = torch.randn(rows, vocab, generator=g) * std
    for r in range(rows):
        x[r, torch.randperm(vocab, generator=g)[:min(likely, vocab // 2)]] += 7.0
    noise = torch.empty(rows, vocab).exponential_(generator=g)
    return x.to(dtype).to(dev), noise.to(dev)


def _check(logits, noise, temperature, top_k, top_p, min_p, tensors=True):
    dev, rows = logits.device, logits.shape[0]
    per = [np.broadcast_to(np.asarray(a), rows).tolist() for a in (temperature, top_k, top_p, min_p)]
    if tensors:
        args = [torch.tensor(a, dtype=d, device=dev)
                for a, d in zip(per, (torch.float32, torch.int32, torch.float32, torch.float32))]
    else:
        args = [a[0] for a in per]
    tok, lp = ops.sample(logits, noise, *args)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    x, e = logits.float().cpu().numpy(), noise.cpu().numpy()
    for r in range(rows):
        f32 = [np.float32(per[0][r]), per[1][r], np.float32(per[2][r]), np.float32(per[3][r])]
        t, l = decode.sample_one(x[r], e[r], float(f32[0]), f32[1], float(f32[2]), float(f32[3]))
        assert tok[r].item() == t, f"row {r}: token {tok[r].item()}, expected {t}"
        got = lp[r].item()
        assert got == l if math.isinf(l) else abs(got - l) <= 2.0 ** -20 * (1 + abs(l)), f"row {r}: logprob {got}, {l}"
    return tok, lp


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1000, 4097, 51866])
def test_settings(cuda_device, dtype, vocab):
    settings = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.3, 0, 0.95, 0.02), (0.2, 5, 1.0, 0.0), (1.0, 1, 1.0, 0.0),
                (0.0, 7, 0.5, 0.3), (1.0, 0, 0.3, 0.0), (2.0, 900, 0.99, 0.001), (1.0, 3, 1e-6, 0.0), (5.0, 2, 0.6, 1.0),
                (1.0, 10 ** 9, 0.9999, 0.0), (0.05, 0, 0.8, 0.5)]
    logits, noise = _inputs(cuda_device, len(settings), vocab, vocab, dtype)
    _check(logits, noise, *zip(*settings))


@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.05), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.7, 0.0)])
def test_numbers_for_every_row(cuda_device, settings):
    logits, noise = _inputs(cuda_device, 9, 1531, 3)
    _check(logits, noise, *settings, tensors=False)


@pytest.mark.parametrize("vocab", [64, 5000, 51866])
def test_ties(cuda_device, vocab):
    """Few distinct logits and constant noise: the order within ties decides every cut, at the lowest indexes."""
    g = seeded(vocab)
    logits = torch.randint(0, 4, (10, vocab), generator=g).half().to(cuda_device)
    logits[0] = 0.0
    logits[1] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0).half()  # +0 and -0 are one value
    noise = torch.empty(10, vocab).exponential_(generator=g).to(cuda_device)
    for k in (1, 2, 10, vocab // 2, vocab - 1):
        _check(logits, noise, 1.0, k, 1.0, 0.0)
        _check(logits, noise, 1.0, k, 0.5, 0.0)
    _check(logits, torch.ones_like(noise), 1.0, 0, 0.9, 0.0)
    _check(logits, torch.ones_like(noise), 0.0, 0, 0.9, 0.0)


def test_race_that_rejects_for_long(cuda_device):
    """Noise that makes the race order the reverse of the tokens' order, so that every round's winner is the last
    token left, with cuts that keep few."""
    vocab = 3000
    logits = torch.linspace(3, 0, vocab).repeat(4, 1).to(cuda_device)
    noise = torch.logspace(0, -30, vocab).repeat(4, 1).to(cuda_device)
    _check(logits, noise, 1.0, 0, [0.01, 0.5, 0.9, 0.999], 0.0)
    _check(logits, noise, 1.0, [3, 100, 2999, 1], [0.9, 0.01, 0.5, 0.5], 0.0)
    _check(torch.zeros_like(logits), noise, 1.0, 0, [0.01, 0.5, 0.9, 0.999], 0.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_special_values(cuda_device, dtype):
    vocab = 777
    logits, noise = _inputs(cuda_device, 8, vocab, 5, torch.float32)
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[1, 500] = -3.0
    logits[2, ::3] = math.nan
    logits[3, 44] = math.inf
    logits[3, 600] = math.inf
    logits[4] = math.nan
    logits[5, 1:] = torch.finfo(dtype).min
    logits[6, 5:] = -math.inf
    noise[7, ::2] = 0.0
    noise[6, 0] = 1e-45
    logits = logits.to(dtype)
    for settings in ((1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.5, 0.1)):
        tok, lp = _check(logits, noise, *settings)
        assert tok[0].item() == -1 and tok[4].item() == -1 and tok[1].item() == 500


def test_strided_rows_and_outputs(cuda_device):
    big, wide = _inputs(cuda_device, 6, 2003, 7)
    logits, noise = big[:, 1:1602], wide[:, 3:1604]
    tok, lp = _check(logits, noise, 0.9, 30, 0.95, 0.0)
    t2, l2 = torch.full_like(tok, -7), torch.full_like(lp, 9.0)
    got = ops.sample(logits, noise, 0.9, 30, 0.95, 0.0, tokens_out=t2, logprobs_out=l2)
    assert got[0] is t2 and got[1] is l2 and torch.equal(t2, tok) and torch.equal(l2, lp)


def test_many_rows_and_equal_bits(cuda_device):
    logits, noise = _inputs(cuda_device, 300, 2500, 8, torch.bfloat16)
    tok, lp = _check(logits, noise, 0.9, 100, 0.9, 0.01)
    for _ in range(3):
        t2, l2 = ops.sample(logits, noise, 0.9, 100, 0.9, 0.01)
        assert torch.equal(t2, tok) and torch.equal(l2, lp)


@pytest.mark.parametrize("vocab,dtype", [(131072, torch.float32), (200003, torch.float16), (600001, torch.float32)])
def test_large_vocabularies(cuda_device, vocab, dtype):
    logits, noise = _inputs(cuda_device, 3, vocab, 9, dtype)
    _check(logits, noise, [1.0, 0.8, 1.2], [0, 64, 5000], [0.9, 0.95, 1.0], 0.0)


def test_draws_follow_the_distribution(cuda_device):
    """20000 rows of one distribution: each kept token's share is within 5 standard deviations of its probability."""
    rows = 20000
    x = torch.tensor([1.0, 0.5, 2.0, -1.0, 0.0, 1.5, -math.inf, 0.25])
    noise = torch.empty(rows, 8).exponential_(generator=seeded(10)).to(cuda_device)
    tok, _ = ops.sample(x.repeat(rows, 1).to(cuda_device), noise, 0.8, 5, 0.9)
    order = torch.argsort(-x, stable=True)[:5]
    p = torch.softmax(x[order].double() / 0.8, 0)
    keep = (p.cumsum(0) - p) < 0.9
    p = torch.zeros(8, dtype=torch.float64).index_put((order[keep],), p[keep] / p[keep].sum())
    share = torch.bincount(tok.cpu(), minlength=8).double() / rows
    assert ((share - p).abs() <= 5 * (p * (1 - p) / rows).sqrt()).all()


def test_refusals(cuda_device):
    logits, noise = _inputs(cuda_device, 4, 100, 11)
    f = torch.ones(4, device=cuda_device)
    for args, match in (((logits.cpu(), noise), "CUDA"), ((logits.double(), noise), "fp16, bf16 or fp32"),
                        ((logits[0], noise), "2-D"), ((logits, noise.half()), "fp32"), ((logits, noise[:, :99]), "shape"),
                        ((logits.t(), noise.t()), "contiguous rows"), ((logits, noise, f.half()), "temperature"),
                        ((logits, noise, f, f), "top_k"), ((logits, noise, f, 0, f[:3]), "top_p"),
                        ((logits, noise, 1.0, 0, 1.0, f.cpu()), "min_p"), ((logits[:, :0], noise[:, :0]), "vocab = 0")):
        with pytest.raises(RuntimeError, match=match):
            ops.sample(*args)
    for args in ((-1.0,), (1.0, -2), (1.0, 0, -0.1), (1.0, 0, 1.0, -0.5), (float("nan"),)):
        with pytest.raises(ValueError, match="negative"):
            ops.sample(logits, noise, *args)
    with pytest.raises(RuntimeError, match="tokens_out"):
        ops.sample(logits, noise, tokens_out=torch.empty(4, dtype=torch.int32, device=cuda_device))
    tok, lp = ops.sample(logits[:0], noise[:0])
    assert tok.numel() == 0 and lp.numel() == 0
