"""Attention over the 8-bit cache where most tokens' weights are far below the largest but carry the output.

A weight is rounded to fp16 as 2^7 to 2^15 times what it is relative to the largest, so it is off by at most 2^-11 of
itself and by half of fp16's smallest step, 2^-25, over 2^7. With S = sum_j w_j / max w (at least 1) and A = sum_j p_j |v_j| an output is
off by r |ref| for its own rounding (r = 2^-11 fp16, 2^-8 bf16), (2^-11 + 2^-13) A for the weights' rounding and fp32
scores, sums and exponentials, and sum_j 2^-32 |v_j| / S.
"""
import numpy as np
import pytest
import torch

from conftest import seeded
from oracle import decode, fp8
from whisper_blaze_b200 import ops

pytestmark = pytest.mark.gpu

BLOCK = 128


@pytest.mark.parametrize("pages", [1, 2, 8192])
@pytest.mark.parametrize("T", [1, 130])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_small_weights_count(cuda_device, d, dtype, T, pages):
    """One token of each page has a weight about 2^26 times the others' and the value 0; the table names one page again
    and again (up to 2^20 tokens), so the answer is that of the page alone."""
    g = seeded(d + T)
    k = torch.randn(BLOCK, d, generator=g).double().numpy() * 0.02
    v = torch.rand(BLOCK, d, generator=g).double().numpy() * 8000 + 6000
    k[:, 0], k[5, 0], v[5] = 0.0, 1.0, 0.0
    codes = [decode.round_codes(k * 256, fp8.E4M3), decode.round_codes(v / 32, fp8.E4M3)]
    scales = [2.0 ** -8, 32.0]
    k, v = (fp8.decode(c, fp8.E4M3).astype(np.float64) * s for c, s in zip(codes, scales))
    q = torch.randn(1, 1, T, d, generator=g)
    q[..., 0] = 26.0 * np.log(2.0)
    q = q.to(dtype).to(cuda_device)
    gpu = [torch.from_numpy(c).view(1, 1, BLOCK, d).to(cuda_device) for c in codes]
    gpu += [torch.full((1, 1), s, device=cuda_device) for s in scales]
    table = torch.zeros(1, pages, dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([pages * BLOCK], dtype=torch.int32, device=cuda_device)
    got = ops.attention_kv8(q, *gpu, table, lens, causal=False, scale=1.0).double().cpu().numpy()[0, 0]
    qn = q.double().cpu().numpy()[0, 0]
    ref, weight = decode.attention_one(qn, k, v, T, False, 1.0)
    s = qn @ k.T
    total = np.exp(s - s.max(-1, keepdims=True)).sum(-1, keepdims=True)
    r = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    tol = r * np.abs(ref) + (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -32 * np.abs(v).sum(0) / total + 1e-12
    err = np.abs(got - ref)
    assert (err <= tol).all(), f"error {err.max():.3e} of {np.abs(ref).max():.3e}, {(err / tol).max():.2f} of the gate"
