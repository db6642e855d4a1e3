"""Host checks of the cache and sampling entry points: bad arguments are refused before anything is launched, and the
Python layer refuses CPU tensors. Needs no GPU. Also pins the 64-bit oracle of these operators to hand-made cases."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import decode, fp8
from whisper_blaze_b200 import _lib, ops

FAKE = 0x10000  # never dereferenced: validation fails first


def _err(status):
    return status, _lib.lib().wbk_last_error().decode()


def _append(**change):
    a = dict(k=FAKE, v=FAKE, dtype=0, batch=2, kv_heads=2, tokens=1, head_dim=64,
             strides=(ctypes.c_int64 * 6)(128, 64, 128, 128, 64, 128), fmt=0, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, pages=4,
             block=16, table=FAKE, max_blocks=2, table_stride=2, lens=FAKE, fresh=None, stream=None) | change
    return _err(_lib.lib().wbk_kv8_append(*a.values()))


def _attend(**change):
    a = dict(q=FAKE, out=FAKE, dtype=0, batch=2, heads=4, kv_heads=2, queries=1, head_dim=64,
             strides=(ctypes.c_int64 * 6)(256, 64, 256, 256, 64, 256), fmt=0, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, pages=4,
             block=16, table=FAKE, max_blocks=2, table_stride=2, lens=FAKE, q_lens=None, causal=1, scale=1.0, ws=FAKE,
             ws_bytes=1 << 40, stream=None) | change
    return _err(_lib.lib().wbk_attention_kv8(*a.values()))


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("change,status,match", [
    ({"dtype": 2}, _lib.WBK_ERR_INVALID_ARG, "dtype"), ({"fmt": 3}, _lib.WBK_ERR_INVALID_ARG, "format"),
    ({"head_dim": 96}, _lib.WBK_ERR_UNSUPPORTED, "head_dim"), ({"block": 48}, _lib.WBK_ERR_UNSUPPORTED, "block"),
    ({"kc": None}, _lib.WBK_ERR_INVALID_ARG, "null"), ({"lens": None}, _lib.WBK_ERR_INVALID_ARG, "null"),
    ({"strides": None}, _lib.WBK_ERR_INVALID_ARG, "null"), ({"kc": FAKE + 8}, _lib.WBK_ERR_UNSUPPORTED, "aligned"),
    ({"vs": FAKE + 2}, _lib.WBK_ERR_INVALID_ARG, "misaligned"), ({"pages": 0}, _lib.WBK_ERR_INVALID_ARG, "cache size"),
    ({"table_stride": 1}, _lib.WBK_ERR_INVALID_ARG, "cache size"),
    ({"pages": 1 << 31}, _lib.WBK_ERR_UNSUPPORTED, "too large"), ({"batch": -1}, _lib.WBK_ERR_INVALID_ARG, "negative"),
    ({"batch": 40000}, _lib.WBK_ERR_UNSUPPORTED, "batch"),
    ({"strides": (ctypes.c_int64 * 6)(128, 60, 128, 128, 64, 128)}, _lib.WBK_ERR_UNSUPPORTED, "multiple of 8"),
    ({"strides": (ctypes.c_int64 * 6)(128, 64, 128, 128, -64, 128)}, _lib.WBK_ERR_UNSUPPORTED, "multiple of 8"),
])
def test_cache_calls_reject_bad_arguments_on_host(call, change, status, match):
    st, msg = call(**change)
    assert st == status and match in msg


def test_cache_calls_own_arguments():
    assert _append(k=FAKE + 2)[0] == _lib.WBK_ERR_UNSUPPORTED
    assert _append(fresh=FAKE + 1)[0] == _lib.WBK_ERR_INVALID_ARG
    st, msg = _attend(kv_heads=3)
    assert st == _lib.WBK_ERR_INVALID_ARG and "evenly" in msg
    assert _attend(out=FAKE + 8)[0] == _lib.WBK_ERR_UNSUPPORTED
    assert _attend(q_lens=FAKE + 2)[0] == _lib.WBK_ERR_INVALID_ARG
    assert _attend(heads=70000, kv_heads=1)[0] == _lib.WBK_ERR_UNSUPPORTED
    # nothing to do is no error
    for none in ({"batch": 0}, {"tokens": 0}, {"kv_heads": 0}):
        assert _append(k=None, v=None, **none)[0] == 0
    for none in ({"batch": 0}, {"queries": 0}, {"heads": 0}):
        assert _attend(q=None, out=None, **none)[0] == 0


def test_sample_rejects_bad_arguments_on_host():
    def call(**change):
        a = dict(logits=FAKE, dtype=0, rows=2, vocab=10, ls=10, noise=FAKE, ns=10, t=None, k=None, p=None, m=None, ta=1.0,
                 ka=0, pa=1.0, ma=0.0, tok=FAKE, lp=FAKE, stream=None) | change
        return _err(_lib.lib().wbk_sample(*a.values()))

    for change, match in (({"dtype": 5}, "dtype"), ({"vocab": 0}, "vocab = 0"), ({"rows": -1}, "negative"),
                          ({"logits": None}, "null"), ({"tok": None}, "null"), ({"ls": 9}, "stride"), ({"ns": 9}, "stride"),
                          ({"noise": FAKE + 2}, "misaligned"), ({"tok": FAKE + 4}, "misaligned")):
        st, msg = call(**change)
        assert st == _lib.WBK_ERR_INVALID_ARG and match in msg
    assert call(vocab=(1 << 30) + 1, ls=1 << 31, ns=1 << 31)[0] == _lib.WBK_ERR_UNSUPPORTED
    assert call(rows=0, logits=None)[0] == 0


def test_python_layer_refuses_cpu_tensors():
    x = torch.zeros(1, 2, 1, 64).half()
    cache = torch.zeros(2, 2, 16, 64, dtype=torch.uint8)
    scale = torch.ones(2, 2)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.kv8_append(x, x, cache, cache, scale, scale, table, lens)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.attention_kv8(x, cache, cache, scale, scale, table, lens)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.sample(torch.zeros(1, 5), torch.ones(1, 5))


def test_oracle_scales_and_codes():
    assert decode.scale_for(0.0, fp8.E4M3) == 2.0 ** -64
    for fmt, mx in ((fp8.E4M3, 448.0), (fp8.E5M2, 57344.0)):
        for e in (-30, -3, 0, 5):
            assert decode.scale_for(mx * 2.0 ** e, fmt) == 2.0 ** e
            assert decode.scale_for(mx * 2.0 ** e * (1 + 2.0 ** -11), fmt) == 2.0 ** (e + 1)
    codes = np.zeros((2, 1, 16, 64), np.uint8)
    scales = np.ones((2, 1), np.float32)
    decode.append_one(np.full((1, 17, 64), 3.5), codes, scales, np.array([1, 0]), 0, fp8.E4M3)
    assert (scales == 2.0 ** -7).all() and (fp8.decode(codes[1], fp8.E4M3) == 448).all()
    decode.append_one(np.full((1, 1, 64), 7.0), codes, scales, np.array([1, 0]), 17, fp8.E4M3)
    assert scales[0, 0] == 2.0 ** -6 and scales[1, 0] == 2.0 ** -7
    assert (fp8.decode(codes[0, 0, 0], fp8.E4M3) == 224).all() and (fp8.decode(codes[0, 0, 1], fp8.E4M3) == 448).all()


def test_oracle_sampling():
    x, e = np.log(np.array([0.1, 0.4, 0.3, 0.2])), np.array([1e-3, 1.0, 1.0, 1.0])
    assert decode.sample_one(x, e, 1.0, 0, 1.0, 0.0)[0] == 0
    assert decode.sample_one(x, e, 1.0, 3, 1.0, 0.0) == (1, pytest.approx(math.log(0.4)))
    assert decode.sample_one(x, np.array([1.0, 1.0, 1e-3, 1e-6]), 1.0, 3, 0.75, 0.0)[0] == 2  # before the third: 0.7 / 0.9
    assert decode.sample_one(x, np.array([1.0, 1.0, 1.0, 1e-6]), 1.0, 0, 1.0, 0.6)[0] == 1
    assert decode.sample_one(np.full(3, -np.inf), e[:3], 1.0, 0, 1.0, 0.0) == (-1, -math.inf)
