"""Forms of the cache's calls that take a way of their own: repeated queries and more than 128 query heads per KV head (the
few-rows kernel with many blocks of rows), repeated keys and values, and scales at the ends of their range. Gates as in
test_gpu_kv8.py.
"""
import numpy as np
import pytest
import torch

from conftest import seeded
from oracle import decode
from test_gpu_kv8 import Cache, _append_and_check, _attention_check, _i32, _q
from whisper_blaze_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 3), (128, 4)])
@pytest.mark.parametrize("over", ["positions", "heads", "batch", "all"])
def test_repeated_queries(cuda_device, over, d, group, causal):
    """Strides of 0 with more than 32 rows per KV head, over short and long sequences."""
    lens, T = [41, 2500, 0, 130], 41
    shape = [len(lens), 2 * group, T, d]
    small = list(shape)
    for i, name in enumerate(("batch", "heads", "positions")):
        if over in (name, "all"):
            small[i] = 1
    c = Cache(cuda_device, len(lens), 2, d, 64, -(-max(lens) // 64), seed=60 + d)
    q = _q(cuda_device, 61, *small, dtype=torch.bfloat16 if d == 128 else torch.float16).expand(*shape)
    assert 0 in q.stride()
    gpu = c.to_gpu()
    y = _attention_check(cuda_device, c, q, lens, [T, T, T, 17], causal, gpu=gpu)
    for _ in range(2):
        assert torch.equal(ops.attention_kv8(q, *gpu, _i32(cuda_device, lens), _i32(cuda_device, [T, T, T, 17]), causal=causal), y)


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("d,dtype,fmt", [(64, torch.float16, "e4m3"), (128, torch.bfloat16, "e5m2")])
def test_more_query_heads_per_kv_head_than_a_tile(cuda_device, d, dtype, fmt, T):
    lens = [3000, 5, 0, 700]
    c = Cache(cuda_device, len(lens), 1, d, 128, -(-max(lens) // 128), fmt, seed=62)
    _attention_check(cuda_device, c, _q(cuda_device, 63, len(lens), 130, T, d, dtype=dtype), lens)


@pytest.mark.parametrize("over", [0, 1, 2])
def test_append_repeated_values(cuda_device, over):
    shape = [3, 4, 20, 64]
    small = list(shape)
    small[over] = 1
    c = Cache(cuda_device, 3, 4, 64, 16, 4, seed=64 + over)
    k, v = (_q(cuda_device, 65 + i, *small).expand(*shape) for i in range(2))
    _append_and_check(cuda_device, c, k, v, [0, 7, 30])


@pytest.mark.parametrize("T,d", [(1, 64), (1, 128), (150, 64), (150, 128)])
@pytest.mark.parametrize("exponents", [(-64,), (60,), (-64, 26), (-30, 60)])
def test_value_scales_at_the_ends_of_their_range(cuda_device, T, d, exponents):
    """One scale or two, at most 2^90 apart. A weight is off by 2^-32 of the row's largest product of weight and value scale, which
    is at most the largest weight times the largest scale."""
    c = Cache(cuda_device, 2, 2, d, 16, 24, seed=70)
    c.scales[1][:] = np.ldexp(1.0, np.random.RandomState(4).choice(exponents, c.scales[1].shape)).astype(np.float32)
    q = _q(cuda_device, 71, 2, 2, T, d, dtype=torch.bfloat16)
    lens = [384, 333]
    y = ops.attention_kv8(q, *c.to_gpu(), _i32(cuda_device, lens)).double().cpu().numpy()
    for b in range(2):
        for h in range(2):
            k, v = c.values(0, b, h, lens[b]), c.values(1, b, h, lens[b])
            ref, weight = decode.attention_one(q[b, h].double().cpu().numpy(), k, v, T, True, d ** -0.5)
            tol = 2.0 ** -8 * np.abs(ref) + (2.0 ** -11 + 2.0 ** -13) * weight + 384 * 2.0 ** -32 * np.abs(v).max()
            assert np.isfinite(y[b, h]).all() and (np.abs(y[b, h] - ref) <= tol).all()
