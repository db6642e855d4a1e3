"""GPU parity of the 8-bit key/value cache (append, attention) against 64-bit definitions (oracle.decode).

Gates. Append: codes and scales bit for bit (every operation on them is exact or one rounding to nearest even).
Attention, elementwise, with A = sum_j p_j |v_j|: r |ref| for the output's rounding (r = 2^-11 fp16, 2^-8 bf16:
half a unit in the last of 11 or 8 significant bits)
+ 2^-11 A for the softmax weights' rounding to fp16 + 2^-13 A for fp32 scores and exponentials (scores of some tens,
128 products) + L 2^-25 max|v| for weights below fp16's normal range.
"""
import numpy as np
import pytest
import torch

from conftest import seeded
from oracle import decode, fp8
from whisper_blaze_b200 import _lib, ops

FMT = {"e4m3": fp8.E4M3, "e5m2": fp8.E5M2}
pytestmark = pytest.mark.gpu


class Cache:
    """A cache of `pages` pages with random codes at random scales, on the GPU and as numpy."""

    def __init__(self, dev, batch, kvh, d, block, width, fmt="e4m3", seed=0, spare=3):
        g = seeded(seed)
        self.fmt, self.block, self.dev = fmt, block, dev
        pages = batch * width + spare
        top = 0x7E if fmt == "e4m3" else 0x7B
        self.codes, self.scales = [], []
        for _ in "kv":
            x = torch.randn(pages, kvh, block, d, generator=g).double().numpy()
            e = torch.randint(-9, -5, (pages, kvh), generator=g).numpy() - (0 if fmt == "e4m3" else 7)
            scale = np.ldexp(np.ones((pages, kvh)), e)
            codes = decode.round_codes(x / scale[..., None, None], FMT[fmt])
            assert (codes & 0x7F).max() <= top
            self.codes.append(codes)
            self.scales.append(scale.astype(np.float32))
        self.table = torch.randperm(pages, generator=g)[:batch * width].view(batch, width).numpy().astype(np.int32)

    def to_gpu(self):
        c = [torch.from_numpy(x.copy()).to(self.dev) for x in self.codes]
        s = [torch.from_numpy(x.copy()).to(self.dev) for x in self.scales]
        return c[0], c[1], s[0], s[1], torch.from_numpy(self.table.copy()).to(self.dev)

    def values(self, which, b, h, length):
        """The tokens' values [length, d] fp64 of one sequence and head; tokens of pages outside the pool left out."""
        got = []
        for j in range(length):
            page = self.table[b, j // self.block]
            if 0 <= page < len(self.codes[which]):
                got.append(fp8.decode(self.codes[which][page, h, j % self.block], FMT[self.fmt]).astype(np.float64)
                           * self.scales[which][page, h])
        return np.stack(got) if got else np.zeros((0, self.codes[which].shape[-1]))


def _i32(dev, values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------- append

def _append_and_check(dev, c, k, v, lens, fresh=None):
    kc, vc, ks, vs, table = c.to_gpu()
    n = fresh if fresh is not None else [k.shape[2]] * k.shape[0]
    ops.kv8_append(k, v, kc, vc, ks, vs, table, _i32(dev, lens), None if fresh is None else _i32(dev, fresh), fmt=c.fmt)
    for which, (x, got, gs) in enumerate(((k, kc, ks), (v, vc, vs))):
        xn = x.float().cpu().numpy()
        for b in range(k.shape[0]):
            decode.append_one(xn[b][:, :max(0, min(n[b], k.shape[2]))], c.codes[which], c.scales[which], c.table[b],
                              lens[b], FMT[c.fmt])
        assert np.array_equal(gs.cpu().numpy(), c.scales[which]), "scales"
        assert np.array_equal(got.cpu().numpy(), c.codes[which]), "codes"


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,block,T,lens", [(64, 16, 1, [0, 1, 15, 16, 17]), (64, 32, 5, [0, 30, 31, 32, 63]),
                                            (128, 64, 130, [0, 63, 64, 1, 100]), (128, 128, 257, [0, 127, 5, 128, 64]),
                                            (64, 128, 1, [127, 0, 129, 3, 255]), (64, 64, 1500, [0, 1, 0, 0, 36])])
def test_append_matches_definition(cuda_device, fmt, dtype, d, block, T, lens):
    B, H = len(lens), 3
    c = Cache(cuda_device, B, H, d, block, -(-(max(lens) + T) // block), fmt, seed=T)
    g = seeded(T + block)
    k, v = (torch.randn(B, H, T, d, generator=g).to(dtype).to(cuda_device) for _ in "kv")
    _append_and_check(cuda_device, c, k * 3, v, lens)


def test_append_ragged_strided_and_growing_scales(cuda_device):
    """The projection's [B, T, H * D] layout, ragged counts, and token after token 4 times larger, so that every
    append re-codes its page."""
    B, H, T, d, block = 4, 2, 9, 64, 16
    c = Cache(cuda_device, B, H, d, block, 4, seed=3)
    g = seeded(4)
    x = torch.randn(B, T, 2, H, d, generator=g).half()
    x = (x * torch.logspace(-4, 1, T).view(1, T, 1, 1, 1).half()).to(cuda_device)
    k, v = x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)
    _append_and_check(cuda_device, c, k, v, [0, 5, 14, 16], [9, 0, 4, 7])
    for i in range(T):
        _append_and_check(cuda_device, c, k[:, :, i:i + 1], v[:, :, i:i + 1], [30 + i] * B)


def test_append_special_values(cuda_device):
    """Zeros (the least scale), the format's exact maximum and one step above, subnormals, NaN and infinities."""
    H, d, block = 2, 64, 16
    rows = [0.0, 448.0, 448.25, 57344.0, 57376.0, 6e-8, 65504.0, float("inf"), float("nan"), -float("inf")]
    for fmt in ("e4m3", "e5m2"):
        c = Cache(cuda_device, len(rows), H, d, block, 2, fmt, seed=9)
        k = torch.zeros(len(rows), H, 3, d, dtype=torch.float16)
        k[:, 0, 1, 7] = torch.tensor(rows).half()
        k[:, 1, 0, ::5] = 1.5
        k[:, 1, 2, 3] = torch.tensor(rows).half()
        _append_and_check(cuda_device, c, k.to(cuda_device), -k.to(cuda_device), [0, 1, 2, 3, 15, 16, 14, 0, 1, 29])
    big = torch.zeros(2, H, 2, d, dtype=torch.bfloat16)
    big[0, :, :, 0] = 3.3e38
    big[1, :, :, 0] = 1e-30
    c = Cache(cuda_device, 2, H, d, block, 1, seed=10)
    _append_and_check(cuda_device, c, big.to(cuda_device), big.to(cuda_device), [0, 0])


def test_append_outside_the_table_or_pool_is_dropped(cuda_device):
    B, H, T, d, block = 3, 2, 20, 64, 16
    c = Cache(cuda_device, B, H, d, block, 3, seed=11)
    c.table[0, 1] = -1
    c.table[1, 1] = len(c.codes[0])
    g = seeded(12)
    k, v = (torch.randn(B, H, T, d, generator=g).half().to(cuda_device) for _ in "kv")
    _append_and_check(cuda_device, c, k, v, [10, 14, 40])


def test_append_nothing(cuda_device):
    c = Cache(cuda_device, 2, 2, 64, 16, 2, seed=13)
    k = torch.ones(2, 2, 4, 64, dtype=torch.float16, device=cuda_device)
    _append_and_check(cuda_device, c, k, k, [3, 5], [0, -1])
    kc, vc, ks, vs, table = c.to_gpu()
    ops.kv8_append(k[:, :, :0], k[:, :, :0], kc, vc, ks, vs, table, _i32(cuda_device, [3, 5]))
    assert np.array_equal(kc.cpu().numpy(), c.codes[0])


# ---------------------------------------------------------------- attention

def _attention_check(dev, c, q, lens, q_lens=None, causal=True, scale=None, out=None, gpu=None):
    B, Hq, T, D = q.shape
    kc, vc, ks, vs, table = c.to_gpu() if gpu is None else gpu
    y = ops.attention_kv8(q, kc, vc, ks, vs, table, _i32(dev, lens), None if q_lens is None else _i32(dev, q_lens),
                          causal=causal, scale=scale, fmt=c.fmt, out=out)
    assert y.shape == q.shape and y.dtype == q.dtype
    got = y.double().cpu().numpy()
    qn = q.double().cpu().numpy()
    group = Hq // c.codes[0].shape[1]
    r = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    for b in range(B):
        n = T if q_lens is None else q_lens[b]
        for kvh in range(Hq // group):
            k, v = c.values(0, b, kvh, lens[b]), c.values(1, b, kvh, lens[b])
            far = len(k) * 2.0 ** -25 * (np.abs(v).max() if len(v) else 0.0)
            for h in range(kvh * group, (kvh + 1) * group):
                ref, weight = decode.attention_one(qn[b, h], k, v, n, causal, scale if scale is not None else D ** -0.5)
                tol = r * np.abs(ref) + (2.0 ** -11 + 2.0 ** -13) * weight + far + 1e-12
                err = np.abs(got[b, h] - ref)
                assert (err <= tol).all(), f"b {b} h {h}: error {err.max():.3e}, {(err / tol).max():.2f} of the gate"
    return y


def _q(dev, seed, *shape, dtype=torch.float16, std=1.5):
    return (torch.randn(*shape, generator=seeded(seed)) * std).to(dtype).to(dev)


@pytest.mark.parametrize("dtype,fmt", [(torch.float16, "e4m3"), (torch.bfloat16, "e4m3"), (torch.float16, "e5m2"),
                                       (torch.bfloat16, "e5m2")])
@pytest.mark.parametrize("d,block", [(64, 16), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("group", [1, 4, 6])
def test_single_token_ragged(cuda_device, dtype, fmt, d, block, group):
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 300, 127, 128, 129]
    c = Cache(cuda_device, len(lens), 2, d, block, -(-300 // block), fmt, seed=d + block)
    _attention_check(cuda_device, c, _q(cuda_device, 5, len(lens), 2 * group, 1, d, dtype=dtype), lens)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,lens,q_lens", [(2, [2, 1, 700, 64], None), (5, [5, 3, 130, 64], [5, 3, 0, 2]),
                                           (17, [17, 400, 16, 33], None), (65, [65, 64, 1, 300], [65, 60, 1, 33]),
                                           (130, [130, 257, 129, 500], [130, 128, 64, 129]),
                                           (300, [300, 299, 301, 1000], None)])
@pytest.mark.parametrize("d,block,group", [(64, 16, 1), (128, 64, 4), (64, 128, 2), (128, 32, 1)])
def test_several_queries(cuda_device, causal, T, lens, q_lens, d, block, group):
    c = Cache(cuda_device, len(lens), 2, d, block, -(-max(lens) // block), seed=T)
    _attention_check(cuda_device, c, _q(cuda_device, 6, len(lens), 2 * group, T, d), lens, q_lens, causal)


@pytest.mark.parametrize("dtype,fmt", [(torch.bfloat16, "e4m3"), (torch.float16, "e5m2"), (torch.bfloat16, "e5m2")])
@pytest.mark.parametrize("d,T", [(64, 7), (128, 200)])
def test_several_queries_types(cuda_device, dtype, fmt, d, T):
    lens = [T, 333]
    c = Cache(cuda_device, 2, 2, d, 64, 6, fmt, seed=T)
    _attention_check(cuda_device, c, _q(cuda_device, 7, 2, 6, T, d, dtype=dtype), lens)


@pytest.mark.parametrize("T", [1, 3, 129])
def test_strided_queries_and_output(cuda_device, T):
    """q as a slice of a fused projection [B, T, H * 3 * D], the output written into [B, T, H * D]."""
    B, H, d = 3, 4, 64
    lens = [T, T + 70, T + 5]
    c = Cache(cuda_device, B, H, d, 32, 8, seed=21)
    big = _q(cuda_device, 22, B, T, 3 * H * d)
    q = big.view(B, T, 3, H, d)[:, :, 1].transpose(1, 2)
    out = torch.full((B, T, H * d), float("nan"), dtype=torch.float16, device=cuda_device)
    y = _attention_check(cuda_device, c, q, lens, out=out.view(B, T, H, d).transpose(1, 2))
    assert y.data_ptr() == out.data_ptr() and not out.isnan().any()


@pytest.mark.parametrize("T", [1, 140])
def test_what_lies_behind_the_length_is_not_used(cuda_device, T):
    """NaN and largest codes behind every length, stale scales that are NaN, table entries that name no page."""
    B, H, d, block = 3, 2, 64, 16
    lens = [T, T + 18, T + 40]
    width = -(-(T + 40) // block) + 2
    c = Cache(cuda_device, B, H, d, block, width, seed=23)
    used = set()
    for b in range(B):
        used |= {(int(c.table[b, j // block]), j % block) for j in range(lens[b])}
    for page in range(len(c.codes[0])):
        for slot in range(block):
            if (page, slot) not in used:
                for x in c.codes:
                    x[page, :, slot] = 0x7F if slot % 2 else 0x7E
        if not any(p == page for p, _ in used):
            for s in c.scales:
                s[page] = np.nan
    gpu = c.to_gpu()
    for b in range(B):
        gpu[4][b, -(-lens[b] // block):] = torch.tensor([-5, 1 << 30, -1, 7, 0, 1])[:width - -(-lens[b] // block)]
    _attention_check(cuda_device, c, _q(cuda_device, 24, B, 4, T, d), lens, gpu=gpu)
    _attention_check(cuda_device, c, _q(cuda_device, 25, B, 4, T, d), lens, causal=False, gpu=gpu)


@pytest.mark.parametrize("T", [1, 130])
def test_pages_outside_the_pool_are_left_out(cuda_device, T):
    c = Cache(cuda_device, 2, 2, 64, 32, 8, seed=26)
    c.table[0, 2] = -1
    c.table[1, 0] = 1000
    c.table[1, 3] = -7
    _attention_check(cuda_device, c, _q(cuda_device, 27, 2, 2, T, 64), [200, 256], causal=False)


@pytest.mark.parametrize("T,d", [(1, 64), (1, 128), (150, 64), (150, 128)])
def test_pages_of_very_different_scales(cuda_device, T, d):
    """Value scales from 2^-64 to 2^10 side by side, key scales likewise small, zero pages among them: the output's
    precision follows what the weights pick, not the largest scale."""
    c = Cache(cuda_device, 2, 2, d, 16, 24, seed=28)
    g = np.random.RandomState(3)
    c.scales[1][:] = np.ldexp(1.0, g.choice([-64, -30, -9, -8, 0], c.scales[1].shape)).astype(np.float32)
    c.codes[1][::5] = 0
    c.scales[1][::5] = np.float32(2.0 ** -64)
    c.scales[0][::3] = np.float32(2.0 ** -20)
    q = _q(cuda_device, 29, 2, 2, T, d)
    kc, vc, ks, vs, table = c.to_gpu()
    lens = [384, 333]
    y = ops.attention_kv8(q, kc, vc, ks, vs, table, _i32(cuda_device, lens)).double().cpu().numpy()
    for b in range(2):
        for h in range(2):
            k, v = c.values(0, b, h, lens[b]), c.values(1, b, h, lens[b])
            ref, weight = decode.attention_one(q[b, h].double().cpu().numpy(), k, v, T, True, d ** -0.5)
            # weights times values below 2^-24 of the largest such product are lost to fp16's range
            tol = 2.0 ** -11 * np.abs(ref) + (2.0 ** -11 + 2.0 ** -13) * weight + 384 * 2.0 ** -25 * np.abs(v).max() + 2.0 ** -25
            assert (np.abs(y[b, h] - ref) <= tol).all()


@pytest.mark.parametrize("T", [1, 130])
def test_rising_scores_and_custom_scale(cuda_device, T):
    """Scores that rise all along the cache, so the running maximum moves at every tile, and reach +-90."""
    c = Cache(cuda_device, 1, 1, 64, 64, 10, seed=30)
    n = 620
    for j in range(n):
        page = c.table[0, j // 64]
        c.codes[0][page, 0, j % 64, 0] = fp8.encode_rne_satfinite(np.float32([(j - 310) * 1.0]), fp8.E4M3)[0]
        c.scales[0][page, 0] = 2.0 ** -8
    q = _q(cuda_device, 31, 1, 1, T, 64, std=0.05)
    q[..., 0] = 70.0
    _attention_check(cuda_device, c, q, [n], scale=1.0, causal=False)
    _attention_check(cuda_device, c, -q, [n], scale=0.5, causal=False)


@pytest.mark.parametrize("T", [1, 4, 150])
def test_a_long_cache_and_equal_bits(cuda_device, T):
    c = Cache(cuda_device, 2, 2, 128, 128, 40, seed=32)
    q = _q(cuda_device, 33, 2, 8, T, 128, dtype=torch.bfloat16)
    gpu = c.to_gpu()
    lens = [5100, 2049]
    y = _attention_check(cuda_device, c, q, lens, gpu=gpu)
    args = (q, *gpu, _i32(cuda_device, lens))
    for _ in range(3):
        assert torch.equal(ops.attention_kv8(*args), y)


@pytest.mark.parametrize("d,T,group,dtype,fmt", [(64, 9, 4, torch.float16, "e4m3"), (128, 33, 1, torch.bfloat16, "e4m3"),
                                                 (64, 128, 1, torch.bfloat16, "e5m2"), (128, 15, 8, torch.float16, "e5m2")])
@pytest.mark.parametrize("causal", [True, False])
def test_33_to_128_rows(cuda_device, causal, d, T, group, dtype, fmt):
    """Two shares of the work per CTA: one long sequence in all of them, short ones of a tile or two, one with nothing."""
    lens, q_lens = [9000, 130, 0, T, 257, 700], [T, T, T, 5, 0, T - 1]
    c = Cache(cuda_device, len(lens), 2, d, 64, -(-max(lens) // 64), fmt, seed=T)
    q = _q(cuda_device, 50 + T, len(lens), 2 * group, T, d, dtype=dtype)
    gpu = c.to_gpu()
    y = _attention_check(cuda_device, c, q, lens, q_lens, causal, gpu=gpu)
    for _ in range(3):
        assert torch.equal(ops.attention_kv8(q, *gpu, _i32(cuda_device, lens), _i32(cuda_device, q_lens), causal=causal,
                                             fmt=fmt), y)


def test_many_items_of_one_tile(cuda_device):
    """More items than shares, each of one tile of 64 rows."""
    lens = [1 + i * 3 % 128 for i in range(96)]
    c = Cache(cuda_device, len(lens), 4, 64, 32, 4, seed=51)
    _attention_check(cuda_device, c, _q(cuda_device, 52, len(lens), 4, 64, 64), lens, causal=False)


def test_offsets_past_32_bits(cuda_device):
    """A pool whose last pages lie beyond 2^32 bytes, filled only where it is read."""
    pages, d, block = (1 << 32) // (128 * 128) + 40, 128, 128
    codes = torch.empty(2, pages, 1, block, d, dtype=torch.uint8, device=cuda_device)
    scales = torch.full((2, pages, 1), 2.0 ** -7, device=cuda_device)
    c = Cache(cuda_device, 1, 1, d, block, 30, seed=34)
    far = torch.arange(pages - 33, pages, device=cuda_device)
    for which in range(2):
        codes[which, far] = torch.from_numpy(c.codes[which]).to(cuda_device)
        scales[which, far] = torch.from_numpy(c.scales[which]).to(cuda_device)
    table = torch.from_numpy(c.table).to(cuda_device) + (pages - 33)
    lens = [3500]
    for T in (1, 140):
        _attention_check(cuda_device, c, _q(cuda_device, 35, 1, 4, T, d), lens,
                         gpu=(codes[0], codes[1], scales[0], scales[1], table))
    k, v = (_q(cuda_device, 36 + i, 1, 1, 60, d) for i in range(2))
    ops.kv8_append(k, v, codes[0], codes[1], scales[0], scales[1], table, _i32(cuda_device, lens))
    for which, x in enumerate((k, v)):
        decode.append_one(x[0].float().cpu().numpy(), c.codes[which], c.scales[which], c.table[0], lens[0], fp8.E4M3)
        assert np.array_equal(codes[which, far].cpu().numpy(), c.codes[which])


@pytest.mark.parametrize("T", [1, 130])
def test_append_then_attend_on_a_side_stream(cuda_device, T):
    """Token by token appends and attention on a stream of their own with a workspace of their own."""
    B, H, d, block = 2, 2, 64, 32
    c = Cache(cuda_device, B, H, d, block, 8, seed=40)
    kc, vc, ks, vs, table = c.to_gpu()
    side = torch.cuda.Stream()
    need = max(1, int(_lib.lib().wbk_attention_kv8_ws_bytes(B, 2 * H, H, T, d)))
    with torch.cuda.stream(side):
        ws = torch.zeros(need, dtype=torch.uint8, device=cuda_device)
        k, v = (torch.randn(B, H, T + 3, d, generator=seeded(41 + i)).half().to(cuda_device) for i in range(2))
        q = _q(cuda_device, 43, B, 2 * H, T, d)
        lens = torch.zeros(B, dtype=torch.int32, device=cuda_device)
        for i in range(3):
            ops.kv8_append(k[:, :, i:i + 1], v[:, :, i:i + 1], kc, vc, ks, vs, table, lens)
            lens += 1
        ops.kv8_append(k[:, :, 3:], v[:, :, 3:], kc, vc, ks, vs, table, lens)
        lens += T
        y = ops.attention_kv8(q, kc, vc, ks, vs, table, lens, workspace=ws)
    side.synchronize()
    for which, x in enumerate((k, v)):
        xn = x.float().cpu().numpy()
        for b in range(B):
            for i in range(3):
                decode.append_one(xn[b][:, i:i + 1], c.codes[which], c.scales[which], c.table[b], i, fp8.E4M3)
            decode.append_one(xn[b][:, 3:], c.codes[which], c.scales[which], c.table[b], 3, fp8.E4M3)
    assert torch.equal(y, _attention_check(cuda_device, c, q, [T + 3] * B))


def test_capture_into_a_graph(cuda_device):
    """One append + attention step captured once, replayed for three tokens."""
    B, H, d = 2, 2, 64
    c = Cache(cuda_device, B, H, d, 32, 4, seed=44)
    gpu = c.to_gpu()
    k, v, q = (torch.zeros(B, H, 1, d, dtype=torch.float16, device=cuda_device) for _ in range(3))
    before, after = _i32(cuda_device, [0, 20]), _i32(cuda_device, [1, 21])
    out = torch.empty_like(q)

    def step():
        ops.kv8_append(k, v, *gpu, before)
        ops.attention_kv8(q, *gpu, after, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    gpu[0].copy_(torch.from_numpy(c.codes[0]))
    gpu[1].copy_(torch.from_numpy(c.codes[1]))
    gpu[2].copy_(torch.from_numpy(c.scales[0]))
    gpu[3].copy_(torch.from_numpy(c.scales[1]))
    for i in range(3):
        for t, s in ((k, 50), (v, 60), (q, 70)):
            t.copy_(_q(cuda_device, s + i, B, H, 1, d))
        graph.replay()
        torch.cuda.synchronize()
        for which, x in enumerate((k, v)):
            for b, n in enumerate((i, 20 + i)):
                decode.append_one(x[b].float().cpu().numpy(), c.codes[which], c.scales[which], c.table[b], n, fp8.E4M3)
        assert torch.equal(out, _attention_check(cuda_device, c, q, [1 + i, 21 + i], gpu=gpu))
        before += 1
        after += 1


def test_refusals(cuda_device):
    c = Cache(cuda_device, 2, 2, 64, 16, 2, seed=45)
    kc, vc, ks, vs, table = c.to_gpu()
    lens = _i32(cuda_device, [3, 4])
    q = _q(cuda_device, 46, 2, 4, 1, 64)
    kv = _q(cuda_device, 47, 2, 2, 1, 64)

    def attend(**change):
        a = dict(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, block_table=table, seq_lens=lens) | change
        return ops.attention_kv8(**a)

    def append(**change):
        a = dict(k=kv, v=kv, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, block_table=table, seq_lens=lens) | change
        return ops.kv8_append(**a)

    for call in (attend, append):
        for change, match in (({"k_cache": kc.cpu()}, "CUDA"), ({"k_cache": kc.float()}, "codes"),
                              ({"v_cache": vc[:, :, :8].contiguous()}, "same shape"), ({"k_scale": ks.half()}, "fp32"),
                              ({"k_scale": ks[:1]}, "shape"), ({"block_table": table.long()}, "int32"),
                              ({"block_table": table[:1]}, "block_table"), ({"seq_lens": lens.long()}, "int32"),
                              ({"seq_lens": lens[:1]}, "seq_lens"), ({"fmt": "int8"}, "format"),
                              ({"k_cache": kc.view(torch.float8_e5m2)}, "codes"),
                              ({"k_cache": kc[:, :, :, ::2]}, "contiguous")):
            with pytest.raises((RuntimeError, ValueError), match=match):
                call(**change)
    odd = _q(cuda_device, 48, 2, 4, 1, 68)[..., :64]
    for change, match in (({"q": q.float()}, "fp16 or bf16"), ({"q": q[0]}, "4D"), ({"q": q[:, :3]}, "evenly"),
                          ({"q": odd}, "multiple of 8"), ({"out": torch.empty_like(q).bfloat16()}, "out"),
                          ({"q_lens": lens.float()}, "q_lens"), ({"q": _q(cuda_device, 1, 2, 4, 1, 32)}, "heads of"),
                          ({"q": torch.empty(2 * 4 * 64 + 1, dtype=torch.float16, device=cuda_device)[1:].view(2, 4, 1, 64)},
                           "aligned")):
        with pytest.raises(RuntimeError, match=match):
            attend(**change)
    for change, match in (({"k": kv.float()}, "fp16 or bf16"), ({"v": kv.bfloat16()}, "same shape and dtype"),
                          ({"k": kv[:, :1], "v": kv[:, :1]}, "heads of"), ({"new_lens": lens[:1]}, "new_lens")):
        with pytest.raises(RuntimeError, match=match):
            append(**change)
    small = torch.zeros(4, 2, 8, 64, dtype=torch.uint8, device=cuda_device)
    with pytest.raises(RuntimeError, match="block 8"):
        attend(k_cache=small, v_cache=small, k_scale=ks[:4].contiguous(), v_scale=vs[:4].contiguous())
    empty = ops.attention_kv8(q[:, :, :0], kc, vc, ks, vs, table, lens)
    assert empty.shape == (2, 4, 0, 64)


def test_no_device_error(cuda_device):
    assert _lib.device_error() == 0
