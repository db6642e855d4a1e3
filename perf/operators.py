"""Cases and plain forms of the decoder-step operators: a key/value cache held in 8 bits, attention over it, sampling.

With `own` false, run() computes an operator from elementary torch operations in 32 bits; with `own` true it makes the
calls a user makes: ops.kv8_append, ops.attention_kv8 and ops.sample.

A cache page holds `block` tokens of one KV head: codes [pages, kv_heads, block, head_dim] (8-bit floats) and one
power-of-two scale per page and head. A block table [batch, max_blocks] names each sequence's pages in order.
"""
import math
import os
import sys

import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "whisper-blaze_b200")

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
MIN_EXP = -64  # smallest scale exponent


# ------------------------------------------------------------------ cases

def _attn(name, b, kvh, g, d, t, n, block, fmt="e4m3", dtype="float16", causal=True, ragged=0.5):
    """t queries per sequence over caches of up to n tokens; lengths lie between (1 - ragged) * n and n."""
    return {"name": name, "op": "attention", "b": b, "kvh": kvh, "g": g, "d": d, "t": t, "n": n, "block": block,
            "fmt": fmt, "dtype": dtype, "causal": causal, "ragged": ragged}


def _append(name, b, kvh, d, t, n, block, fmt="e4m3", dtype="float16", ragged=0.5):
    """t new tokens per sequence (ragged below that) behind caches of up to n tokens."""
    return {"name": name, "op": "append", "b": b, "kvh": kvh, "d": d, "t": t, "n": n, "block": block, "fmt": fmt,
            "dtype": dtype, "ragged": ragged}


def _sample(name, b, v, dtype="float16", mode="mixed"):
    """One token for each of b rows of v logits; mode: which filters are on."""
    return {"name": name, "op": "sample", "b": b, "v": v, "dtype": dtype, "mode": mode}


def listed():
    return [
        # decoder self-attention of one stream, mid-transcript: 20 heads of 64, at most 448 positions; latency only
        _attn("self step 1", 1, 20, 1, 64, 1, 224, 64, ragged=0.0),
        # the same step for a batch of 64 streams of different lengths
        _attn("self step 64", 64, 20, 1, 64, 1, 448, 32, ragged=0.9),
        # cross-attention of that step: every stream reads the 1500 encoder positions of its 30 s window
        _attn("cross step 64", 64, 20, 1, 64, 1, 1500, 64, causal=False, ragged=0.0),
        # grouped heads of 128 over long ragged caches, the generic serving step
        _attn("grouped long step", 16, 8, 4, 128, 1, 32768, 64, dtype="bfloat16", ragged=0.7),
        # prompt of 223 previous-text tokens before the first step
        _attn("prompt 223", 8, 20, 1, 64, 223, 223, 16, ragged=0.0),
        # a chunk of a long prompt behind what is cached already
        _attn("long prompt chunk", 1, 8, 4, 128, 2011, 16000, 128, ragged=0.0),
        # a step writes one token per stream
        _append("append step 64", 64, 20, 64, 1, 447, 32, ragged=0.9),
        # the encoder's keys and values of 64 windows enter the cross-attention cache
        _append("append cross 64", 64, 20, 64, 1500, 0, 64, ragged=0.0),
        # ragged prompts behind partly filled pages, the wider-range format
        _append("append prompts", 16, 8, 128, 1021, 2000, 128, fmt="e5m2", dtype="bfloat16", ragged=0.8),
        # one stream's next token from the 51866-entry vocabulary
        _sample("sample 1", 1, 51866),
        # the batch of 64 streams, each with its own settings
        _sample("sample 64", 64, 51866),
        # many rows of a large vocabulary in 32 bits
        _sample("sample 256 wide", 256, 131072, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "sample"])
    if op == "sample":
        v = _log_int(rng, 1000, 131072)
        b = _log_int(rng, 1, max(1, min(256, (256 * 131072) // v)))
        c = _sample("", b, v, rng.choice(["float16", "bfloat16", "float32"]), rng.choice(["mixed", "mixed", "plain"]))
        del c["name"]
        return c
    d = rng.choice([64, 128])
    block = rng.choice([16, 32, 64, 128])
    fmt = rng.choice(["e4m3", "e4m3", "e5m2"])
    dtype = rng.choice(["float16", "bfloat16"])
    ragged = rng.choice([0.0, 0.5, 0.9])
    kvh = rng.choice([1, 2, 4, 8, 20])
    if op == "append":
        t = _log_int(rng, 1, 1500)
        n = _log_int(rng, 1, 4096)
        b = _log_int(rng, 1, max(1, min(64, (64 * 1500 * 20 * 64) // (kvh * d * (t + n)))))
        c = _append("", b, kvh, d, t, n, block, fmt, dtype, ragged)
    else:
        g = rng.choice([1, 1, 2, 4, 6, 8])
        t = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
        n = max(t, _log_int(rng, 1, 32768))
        most_bytes = (16 * 8 * 128 * 32768) // (kvh * d * n)  # what the largest listed step reads
        most_pairs = (32 * 2011 * 16000) // (kvh * g * t * n)  # what the longest listed prompt computes
        b = _log_int(rng, 1, max(1, min(64, most_bytes, most_pairs)))
        t = max(1, min(t, (32 * 2011 * 16000) // (kvh * g * n)))
        c = _attn("", b, kvh, g, d, t, n, block, fmt, dtype, rng.choice([True, True, False]), ragged)
    del c["name"]
    return c


def _lengths(count, hi, ragged, lo=0):
    """`count` lengths spread evenly over [(1 - ragged) * hi, hi], none below lo; their sum does not depend on a seed."""
    low = int(hi * (1.0 - ragged))
    return [max(lo, hi - int((hi - low) * ((i * 0.618033988749895) % 1.0))) for i in range(count)]


def work(case):
    if case["op"] == "attention":
        t, heads = case["t"], case["kvh"] * case["g"]
        lens = _lengths(case["b"], case["n"], case["ragged"], lo=min(t, case["n"]))
        tokens, pages = sum(lens), sum(-(-n // case["block"]) for n in lens)
        pairs = sum(t * n - (t * (t - 1) // 2 if case["causal"] else 0) for n in lens)
        rows = case["b"] * t * heads
        return {"bytes": 2 * tokens * case["kvh"] * case["d"] + 8 * pages * case["kvh"] + 4 * rows * case["d"],
                "flops": 4 * pairs * heads * case["d"]}
    if case["op"] == "append":
        fresh = sum(_lengths(case["b"], case["t"], case["ragged"], lo=1))
        return {"bytes": 2 * fresh * case["kvh"] * case["d"] * 3, "flops": 2 * fresh * case["kvh"] * case["d"] * 3}
    item = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["b"] * case["v"] * (item + 4), "flops": case["b"] * case["v"] * 6}


# ----------------------------------------------------------------- inputs

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _kv_values(gen, heads, *shape):
    """Keys or values as a projection gives them: unit normal with a gain per head and channel and a channel offset.
    shape: (..., heads, tokens, d)."""
    d = shape[-1]
    gain = torch.exp(0.5 * _randn(gen, heads, 1, d))
    return _randn(gen, *shape) * gain + 0.3 * _randn(gen, heads, 1, d)


def _lens_tensor(gen, lengths):
    order = torch.randperm(len(lengths), generator=gen, device="cuda")
    return torch.tensor(lengths, dtype=torch.int32, device="cuda")[order]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    b = case["b"]
    dtype = DT[case["dtype"]]
    if case["op"] == "sample":
        v = case["v"]
        # a language model's logits: a broad bulk, a few hundred likelier tokens, some suppressed ones
        logits = 2.0 * _randn(gen, b, v)
        count = max(1, min(300, v // 8))
        likely = torch.randint(0, v // count, (b, count), generator=gen, device="cuda")
        likely += torch.arange(count, device="cuda") * (v // count)
        logits.scatter_(1, likely, 9.0 + 2.0 * _randn(gen, *likely.shape))
        suppressed = torch.randint(0, v, (b, max(1, v // 64)), generator=gen, device="cuda")
        logits.scatter_(1, suppressed, -math.inf)
        noise = torch.empty(b, v, device="cuda").exponential_(generator=gen)

        def pick(values, dt):
            i = torch.randint(0, len(values), (b,), generator=gen, device="cuda")
            return torch.tensor(values, dtype=dt, device="cuda")[i]

        s = {"case": case, "logits": logits.to(dtype), "noise": noise}
        if case["mode"] == "mixed":
            s |= {"temperature": pick([0.0, 0.2, 0.7, 1.0, 1.3], torch.float32),
                  "top_k": pick([0, 1, 40, 1000], torch.int32), "top_p": pick([0.5, 0.9, 0.95, 1.0], torch.float32),
                  "min_p": pick([0.0, 0.0, 0.05], torch.float32)}
        else:
            one = torch.ones(b, device="cuda")
            s |= {"temperature": one, "top_k": torch.zeros(b, dtype=torch.int32, device="cuda"), "top_p": one,
                  "min_p": torch.zeros(b, device="cuda")}
        return s

    kvh, d, t, block = case["kvh"], case["d"], case["t"], case["block"]
    grown = case["op"] == "append"
    lens = _lens_tensor(gen, _lengths(b, case["n"], case["ragged"], lo=0 if grown else min(t, case["n"])))
    fresh = _lens_tensor(gen, _lengths(b, t, case["ragged"], lo=1)) if grown else None
    width = max(1, -(-(case["n"] + (t if grown else 0)) // block))
    pages = b * width + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[: b * width].to(torch.int32).view(b, width)
    s = {"case": case, "lens": lens, "table": table}
    for kind in ("k", "v"):
        # what earlier appends left: pages of values at the page's own power-of-two scale
        scale = torch.exp2(torch.randint(-7, -4, (pages, kvh), generator=gen, device="cuda").float())
        if case["fmt"] == "e5m2":
            scale = scale / 128.0
        x = _kv_values(gen, kvh, pages, kvh, block, d) / scale[:, :, None, None]
        s[kind + "_cache"] = x.clamp(-F8_MAX[case["fmt"]], F8_MAX[case["fmt"]]).to(F8[case["fmt"]])
        s[kind + "_scale"] = scale
        del x
        if grown:  # the projection's output [b, t, heads * d], seen as [b, heads, t, d]
            x = _kv_values(gen, kvh, b, kvh, t, d).to(dtype).transpose(1, 2).contiguous()
            s[kind] = x.view(b, t, kvh, d).transpose(1, 2)
    if grown:
        s["fresh"] = fresh
    else:
        heads = kvh * case["g"]
        s["q"] = (1.5 * _randn(gen, b, t, heads, d)).to(dtype).transpose(1, 2)
    return s


# -------------------------------------------------------------- plain forms

def _plain_attention(case, s):
    q, lens = s["q"], s["lens"].long()
    b, heads, t, d = q.shape
    kvh, block = case["kvh"], case["block"]
    table = s["table"].long()
    n = table.shape[1] * block

    def whole(kind):
        x = s[kind + "_cache"][table].float() * s[kind + "_scale"][table][..., None, None]  # [b, blocks, kvh, block, d]
        x = torch.where(inside, x, 0.0)
        return x.transpose(1, 2).reshape(b, kvh, n, d)

    at = torch.arange(n, device=q.device)
    inside = (at[None] < lens[:, None]).view(b, -1, 1, block, 1)
    scores = q.float().reshape(b, kvh, heads // kvh * t, d) @ whole("k").transpose(2, 3)
    scores = scores.view(b, heads, t, n) * d ** -0.5
    last = lens[:, None].expand(b, t)
    if case["causal"]:
        last = last - t + 1 + torch.arange(t, device=q.device)
    hidden = (at >= last[..., None])[:, None]
    scores = scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(b, kvh, -1, n) @ whole("v")).view(b, heads, t, d)
    return torch.where(total > 0, out / total, 0.0).to(q.dtype)


def _scale_of(amax, fmt):
    """The least power of two 2^E, E >= MIN_EXP, with amax <= max_fp8 * 2^E (max_fp8 is 1.75 * 2^8 or 1.75 * 2^15)."""
    m, e = torch.frexp(amax)
    exp = e - (9 if fmt == "e4m3" else 16) + (m > 0.875).int()
    exp = torch.where(amax > 0, exp, MIN_EXP).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), exp)


def _plain_append(case, s):
    b, kvh, t, d = s["k"].shape
    block, fmt = case["block"], case["fmt"]
    lens, fresh, table = s["lens"].long(), s["fresh"].long(), s["table"].long()
    first = lens // block
    old = lens % block  # tokens already in the first touched page
    width = (t + block - 2) // block + 1
    blocks = first[:, None] + torch.arange(width, device="cuda")
    touched = torch.arange(width, device="cuda") * block < (old + fresh)[:, None]
    pages = table.gather(1, blocks.clamp(max=table.shape[1] - 1))[touched]  # [touched pages]
    at = torch.arange(width * block, device="cuda")
    src = at - old[:, None]  # the new token at each place of the touched pages
    new = ((src >= 0) & (src < fresh[:, None])).view(b, width, 1, block, 1)
    keep = (src < 0).view(b, width, 1, block, 1)
    src = src.clamp(0, t - 1)
    most = F8_MAX[fmt]

    def one(kind):
        cache, scales = s[kind + "_cache"], s[kind + "_scale"]
        x = s[kind].float().gather(2, src[:, None, :, None].expand(b, kvh, width * block, d))
        x = x.view(b, kvh, width, block, d).transpose(1, 2)
        x = torch.where(new, x, 0.0)[touched]
        amax = torch.where(x.isfinite(), x.abs(), 0.0).amax((-1, -2))
        was, left = scales[pages], keep[touched]
        scale = _scale_of(amax, fmt)
        scale = torch.where(left.any(dim=(-1, -2, -3))[:, None], torch.maximum(scale, was), scale)
        x = torch.where(x.isnan(), -math.inf, x) / scale[..., None, None]
        held = cache[pages].float()
        again = held * (was / scale)[..., None, None]
        x = torch.where(new[touched], x, torch.where(left, again, held)).clamp(-most, most)
        cache.view(torch.uint8)[pages] = x.to(F8[fmt]).view(torch.uint8)
        scales[pages] = scale
        return cache, scales

    return one("k") + one("v")


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    b, v = x.shape
    temperature = s["temperature"][:, None]
    top = x.amax(-1, keepdim=True)
    empty = top == -math.inf
    gap = x - torch.where(empty, 0.0, top)
    greedy = temperature <= 0
    p = torch.exp(gap / torch.where(greedy, 1.0, temperature))
    ordered, order = torch.sort(x, dim=-1, descending=True, stable=True)
    ps = p.gather(1, order)
    rank = torch.arange(v, device=x.device)
    k = s["top_k"].long()[:, None]
    in_k = rank < torch.where(k > 0, k, v)
    ps = torch.where(in_k, ps, 0.0)
    upto = torch.cumsum(ps, -1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], -1)
    top_p = s["top_p"][:, None]
    in_p = (before < top_p * upto[:, -1:]) | (rank == 0) | (top_p >= 1)
    keep = in_k & in_p & (ps >= s["min_p"][:, None]) & (ordered > -math.inf)
    score = torch.where(keep, ps / s["noise"].gather(1, order).clamp(min=1.1754944e-38), -1.0)
    score = torch.empty_like(score).scatter_(1, order, score)
    token = torch.where(greedy[:, 0], x.argmax(-1), score.argmax(-1))
    logprob = gap.gather(1, token[:, None]) - torch.log(torch.exp(gap).sum(-1, keepdim=True))
    token = torch.where(empty[:, 0], -1, token)
    return token, torch.where(empty[:, 0], -math.inf, logprob[:, 0])


def run(s):
    case = s["case"]
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(0, PACKAGE)
        from whisper_blaze_b200 import ops
        if case["op"] == "attention":
            return ops.attention_kv8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                     s["lens"], causal=case["causal"], fmt=case["fmt"])
        if case["op"] == "append":
            ops.kv8_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                           s["lens"], s["fresh"], fmt=case["fmt"])
            return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]
        return ops.sample(s["logits"], s["noise"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if case["op"] == "attention":
        return _plain_attention(case, s)
    if case["op"] == "append":
        return _plain_append(case, s)
    return _plain_sample(s)


# ------------------------------------------------------- definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    block = case.get("block")
    if case["op"] == "attention":  # sequence by sequence and KV head by KV head, one dense softmax
        q = s["q"].double()
        b, heads, t, d = q.shape
        out = torch.zeros_like(q)
        g = case["g"]
        for i, length in enumerate(s["lens"].tolist()):
            pages = s["table"][i, : -(-length // block)].long()
            for h in range(case["kvh"] if length else 0):
                k, v = ((s[n + "_cache"][pages, h].double() * s[n + "_scale"][pages, h].double()[:, None, None])
                        .reshape(-1, d)[:length] for n in "kv")
                x = torch.einsum("gtd,nd->gtn", q[i, h * g:(h + 1) * g], k) / math.sqrt(d)
                if case["causal"]:
                    late = torch.ones(t, length, dtype=torch.bool, device=q.device).triu(length - t + 1)
                    x = x.masked_fill(late, -math.inf)
                out[i, h * g:(h + 1) * g] = torch.softmax(x, -1).nan_to_num(0.0) @ v
        return out

    if case["op"] == "append":  # page by page of each sequence, all heads of it at once
        fmt, most = case["fmt"], F8_MAX[case["fmt"]]
        small = 2.0 ** (-9 if fmt == "e4m3" else -16)  # spacing of the format's smallest values
        bits = 3 if fmt == "e4m3" else 2
        if case["b"] * (case["t"] // block + 2) > 8000:
            return None  # tens of thousands of small steps

        def rounded(y):  # to the nearest value of the format, ties to even
            y = y.clamp(-most, most)
            _, e = torch.frexp(y)
            step = torch.ldexp(torch.ones_like(y), e - 1 - bits).clamp(min=small)
            return torch.round(y / step) * step

        result = []
        for kind in "kv":
            codes, scales = s[kind + "_cache"].double(), s[kind + "_scale"].double()
            for i, (length, fresh) in enumerate(zip(s["lens"].tolist(), s["fresh"].tolist())):
                done = 0
                while done < fresh:
                    page, slot = int(s["table"][i, (length + done) // block]), (length + done) % block
                    count = min(block - slot, fresh - done)
                    x = s[kind][i, :, done:done + count].double()
                    peak = x.abs().amax((1, 2))
                    scale = torch.exp2(torch.ceil(torch.log2(peak / most)).clamp(min=MIN_EXP))
                    scale = torch.where((peak <= most * scale / 2) & (scale > 2.0 ** MIN_EXP), scale / 2, scale)
                    if slot:
                        scale = torch.maximum(scale, scales[page])
                        codes[page, :, :slot] = rounded(codes[page, :, :slot] * (scales[page] / scale)[:, None, None])
                    codes[page, :, slot:slot + count] = rounded(x / scale[:, None, None])
                    scales[page] = scale
                    done += count
            result += [codes, scales]
        return tuple(result)

    # sampling, row by row: the kept prefix of the sorted tokens, then the race among them
    tokens, logprobs = [], []
    settings = zip(*(s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p")))
    for row, (temperature, top_k, top_p, min_p) in enumerate(settings):
        x, noise = s["logits"][row].double(), s["noise"][row].double()
        v = x.numel()
        if temperature <= 0:
            tokens.append(int(torch.nonzero(x == x.max())[0]))
        else:
            p = torch.exp((x - x.max()) / temperature)
            order = torch.argsort(-x, stable=True)[: top_k if 0 < top_k < v else v]
            mass = p[order].cumsum(0)
            kept = order if top_p >= 1 else order[: 1 + int((mass[:-1] < top_p * mass[-1]).sum())]
            kept = torch.sort(kept[p[kept] >= min_p]).values
            tokens.append(int(kept[torch.argmax(p[kept] / noise[kept])]))
        logprobs.append(float(x[tokens[-1]] - torch.logsumexp(x, 0)))
    return torch.tensor(tokens, device="cuda"), torch.tensor(logprobs, dtype=torch.float64, device="cuda")
