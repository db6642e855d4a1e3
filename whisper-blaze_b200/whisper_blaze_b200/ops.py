"""Tensor-level wrappers over libwbk.so for torch callers.

Every op runs on torch's current stream of its input's device, under a device
guard, and never synchronises unless it must hand a value back to the host.
Scales can stay on the device (1-element fp32 tensors), so a chain of
quantise -> GEMM -> norm -> quantise issues no host round trip.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence, Union

import torch

from . import _lib
from ._lib import (DT_BF16, DT_F16, DT_F32, EPI_BIAS_MAXKEY, EPI_GELU, EPI_NONE, EPI_RESIDUAL, EPI_RESIDUAL_CLAMP,
                   FMT_E4M3, FMT_E5M2, check, lib, ptr, stream_of)

Scale = Union[float, torch.Tensor]

# Number of libwbk kernels launched by this process (quantise() launches the
# amax and the quantise kernel, 2; every other op launches 1).
LAUNCHES = [0]


def _count(n: int = 1) -> None:
    LAUNCHES[0] += n


_FMT_BY_NAME = {"e4m3": FMT_E4M3, "e5m2": FMT_E5M2, FMT_E4M3: FMT_E4M3, FMT_E5M2: FMT_E5M2}
_EPI_BY_NAME = {"none": EPI_NONE, "bias": EPI_NONE, "gelu": EPI_GELU, "residual": EPI_RESIDUAL,
                "residual_clamp": EPI_RESIDUAL_CLAMP, "bias_maxkey": EPI_BIAS_MAXKEY, EPI_NONE: EPI_NONE,
                EPI_GELU: EPI_GELU, EPI_RESIDUAL: EPI_RESIDUAL, EPI_RESIDUAL_CLAMP: EPI_RESIDUAL_CLAMP,
                EPI_BIAS_MAXKEY: EPI_BIAS_MAXKEY}
_BYTE_DTYPES = {torch.uint8, torch.int8, torch.float8_e4m3fn, torch.float8_e5m2}


def fmt_code(fmt) -> int:
    try:
        return _FMT_BY_NAME[fmt]
    except KeyError:
        raise ValueError(f"unknown fp8 format {fmt!r}; expected 'e4m3' or 'e5m2'") from None


def require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")


def require_contig(t: torch.Tensor, name: str) -> None:
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def require_input(t: torch.Tensor, name: str) -> None:
    require_cuda(t, name)
    require_contig(t, name)


def require_fp16(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.float16:
        raise RuntimeError(f"{name} must be fp16")


def require_bytes(t: torch.Tensor, name: str) -> None:
    if t.dtype not in _BYTE_DTYPES:
        raise RuntimeError(f"{name} must hold fp8 codes (uint8 or a float8 dtype), got {t.dtype}")


def require_same_device(*ts: Optional[torch.Tensor]) -> None:
    devs = {t.device for t in ts if t is not None}
    if len(devs) > 1:
        raise RuntimeError(f"tensors are on different devices: {sorted(map(str, devs))}")


def new_amax_ws(device) -> torch.Tensor:
    """A zeroed device uint32 accumulator (held as int32) for the fused amax."""
    return torch.zeros(1, dtype=torch.int32, device=device)


# ---------------------------------------------------------------- quantiser

def amax_accumulate(x: torch.Tensor, amax_ws: torch.Tensor) -> torch.Tensor:
    require_input(x, "x")
    require_fp16(x, "x")
    require_same_device(x, amax_ws)
    with torch.cuda.device(x.device):
        check(lib().wbk_amax_f16(x.data_ptr(), x.numel(), amax_ws.data_ptr(), stream_of(x)), "amax")
    _count()
    return amax_ws


def quantise_from_amax(x: torch.Tensor, amax_ws: torch.Tensor, fmt="e4m3", q_out: Optional[torch.Tensor] = None,
                       scale_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantise x with the scale implied by an already accumulated amax."""
    require_input(x, "x")
    require_fp16(x, "x")
    f = fmt_code(fmt)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device) if q_out is None else q_out
    s = torch.empty(1, dtype=torch.float32, device=x.device) if scale_out is None else scale_out
    require_same_device(x, amax_ws, q, s)
    with torch.cuda.device(x.device):
        check(lib().wbk_quantise_from_amax_f16(x.data_ptr(), x.numel(), f, amax_ws.data_ptr(), q.data_ptr(),
                                               s.data_ptr(), stream_of(x)), "quantise")
    _count()
    return q, s


# Tensors of RESIDENT_QUANT_MIN to RESIDENT_QUANT_MAX elements (a multiple of 8,
# 16-byte aligned) are quantised by the one-launch resident kernel
# (wbk_quantise_f16_resident); the library applies the same bounds.
RESIDENT_QUANT_MIN = 1 << 22
RESIDENT_QUANT_MAX = 88 << 20
_RESIDENT_SYNC_OFFSET = 32  # bytes: words 8..11 of the device's shared workspace (the GEMM's use 0..3)


def quantise(x: torch.Tensor, fmt="e4m3", q_out: Optional[torch.Tensor] = None,
             scale_out: Optional[torch.Tensor] = None,
             amax_ws: Optional[torch.Tensor] = None,
             sync_ws: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-tensor quantise; returns (codes uint8, device fp32 scale [1]). No host sync.

    Large tensors (RESIDENT_QUANT_MIN to RESIDENT_QUANT_MAX elements) take one cooperative
    launch that reads x from HBM about once; its grid-wide arrival uses 16 bytes
    of sync words, by default in the device's shared workspace, so such calls
    must not run concurrently on different streams: pass `sync_ws` (a zeroed
    device tensor of 16 bytes, left zeroed by each call) to give a stream its
    own. Codes, scale and amax are the same on either path."""
    require_input(x, "x")
    require_fp16(x, "x")
    f = fmt_code(fmt)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device) if q_out is None else q_out
    s = torch.empty(1, dtype=torch.float32, device=x.device) if scale_out is None else scale_out
    ws = torch.empty(1, dtype=torch.int32, device=x.device) if amax_ws is None else amax_ws
    require_same_device(x, q, s, ws, sync_ws)
    n = x.numel()
    with torch.cuda.device(x.device):
        if (RESIDENT_QUANT_MIN <= n <= RESIDENT_QUANT_MAX and n % 8 == 0 and x.data_ptr() % 16 == 0
                and q.data_ptr() % 8 == 0):
            if sync_ws is None:
                sync_ptr = splitk_workspace(x.device, 256).data_ptr() + _RESIDENT_SYNC_OFFSET
            else:
                if sync_ws.numel() * sync_ws.element_size() < 16 or sync_ws.data_ptr() % 16 != 0:
                    raise ValueError("sync_ws must hold 16 bytes at a 16-byte aligned address")
                sync_ptr = sync_ws.data_ptr()
            check(lib().wbk_quantise_f16_resident(x.data_ptr(), n, f, q.data_ptr(), s.data_ptr(), ws.data_ptr(),
                                                  sync_ptr, stream_of(x)), "quantise")
            _count(1)
        else:
            check(lib().wbk_quantise_f16(x.data_ptr(), n, f, q.data_ptr(), s.data_ptr(), ws.data_ptr(),
                                         stream_of(x)), "quantise")
            _count(2)
    return q, s


def quantise_gelu(y: torch.Tensor, ymax_key: Optional[torch.Tensor] = None, fmt="e4m3",
                  q_out: Optional[torch.Tensor] = None, scale_out: Optional[torch.Tensor] = None,
                  amax_ws: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantise fp16(gelu(y)) per tensor without storing the GELU output.

    ymax_key: the max-key word written by a GEMM with the 'bias_maxkey'
    epilogue over y (lets the amax come from y's maximum), or None."""
    require_input(y, "y")
    require_fp16(y, "y")
    f = fmt_code(fmt)
    q = torch.empty(y.shape, dtype=torch.uint8, device=y.device) if q_out is None else q_out
    s = torch.empty(1, dtype=torch.float32, device=y.device) if scale_out is None else scale_out
    ws = torch.empty(1, dtype=torch.int32, device=y.device) if amax_ws is None else amax_ws
    require_same_device(y, ymax_key, q, s, ws)
    with torch.cuda.device(y.device):
        check(lib().wbk_quantise_gelu_f16(y.data_ptr(), y.numel(), f, ptr(ymax_key), q.data_ptr(), s.data_ptr(),
                                          ws.data_ptr(), stream_of(y)), "quantise_gelu")
    _count(2)
    return q, s


def dequantise(q: torch.Tensor, scale: float, shape: Sequence[int], fmt="e4m3") -> torch.Tensor:
    require_input(q, "fp8")
    require_bytes(q, "fp8")
    f = fmt_code(fmt)
    shape = [int(d) for d in shape]
    out = torch.empty(shape, dtype=torch.float16, device=q.device)
    if out.numel() != q.numel():
        raise RuntimeError(f"shape {shape} holds {out.numel()} elements but fp8 has {q.numel()}")
    with torch.cuda.device(q.device):
        check(lib().wbk_dequantise_f16(q.data_ptr(), q.numel(), f, float(scale), out.data_ptr(), stream_of(q)),
              "dequantise")
    _count()
    return out


# -------------------------------------------------------------------- norms

def layernorm(x: torch.Tensor, residual: Optional[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor,
              eps: float = 1e-5, want_sum: bool = False, out: Optional[torch.Tensor] = None,
              sum_out: Optional[torch.Tensor] = None,
              out_amax: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    require_input(x, "x")
    require_input(gamma, "gamma")
    require_input(beta, "beta")
    require_fp16(x, "x")
    require_fp16(gamma, "gamma")
    require_fp16(beta, "beta")
    if residual is not None:
        require_input(residual, "residual")
        require_fp16(residual, "residual")
        if residual.shape != x.shape:
            raise RuntimeError("residual must have the same shape as x")
    if x.dim() == 0:
        raise RuntimeError("x must have at least one dimension")
    D = x.shape[-1]
    if gamma.numel() != D or beta.numel() != D:
        raise RuntimeError(f"gamma and beta must have {D} elements")
    rows = x.numel() // D if D else 0
    o = torch.empty_like(x) if out is None else out
    s = (torch.empty_like(x) if sum_out is None else sum_out) if want_sum else None
    require_same_device(x, residual, gamma, beta, o, s, out_amax)
    with torch.cuda.device(x.device):
        check(lib().wbk_layernorm_f16(x.data_ptr(), ptr(residual), gamma.data_ptr(), beta.data_ptr(), o.data_ptr(),
                                      ptr(s), rows, D, float(eps), ptr(out_amax), stream_of(x)), "layernorm_fused")
    _count()
    return o, s


def layernorm_quantise_ws(rows: int, device) -> torch.Tensor:
    """Workspace for layernorm_quantise: per-row statistics + the (scale, 1/scale) pair."""
    return torch.empty(int(lib().wbk_layernorm_quantise_ws_bytes(int(rows))), dtype=torch.uint8, device=device)


def layernorm_quantise(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5, fmt="e4m3",
                       q_out: Optional[torch.Tensor] = None, scale_out: Optional[torch.Tensor] = None,
                       ws: Optional[torch.Tensor] = None,
                       amax_ws: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """fp8 codes of LayerNorm(x) (no residual), bit-identical to layernorm() then quantise(),
    without writing the fp16 LayerNorm output."""
    require_input(x, "x")
    require_input(gamma, "gamma")
    require_input(beta, "beta")
    require_fp16(x, "x")
    require_fp16(gamma, "gamma")
    require_fp16(beta, "beta")
    D = x.shape[-1]
    if gamma.numel() != D or beta.numel() != D:
        raise RuntimeError(f"gamma and beta must have {D} elements")
    rows = x.numel() // D if D else 0
    f = fmt_code(fmt)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device) if q_out is None else q_out
    s = torch.empty(1, dtype=torch.float32, device=x.device) if scale_out is None else scale_out
    w = layernorm_quantise_ws(rows, x.device) if ws is None else ws
    a = torch.empty(1, dtype=torch.int32, device=x.device) if amax_ws is None else amax_ws
    if w.numel() < lib().wbk_layernorm_quantise_ws_bytes(rows):
        raise RuntimeError("layernorm_quantise workspace too small")
    require_same_device(x, gamma, beta, q, s, w, a)
    with torch.cuda.device(x.device):
        check(lib().wbk_layernorm_quantise_f16(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), rows, D, float(eps), f,
                                               q.data_ptr(), s.data_ptr(), w.data_ptr(), a.data_ptr(), stream_of(x)),
              "layernorm_quantise")
    _count(2)
    return q, s


def rmsnorm(x: torch.Tensor, residual: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    require_input(x, "x")
    require_input(residual, "residual")
    require_input(gamma, "gamma")
    require_fp16(x, "x")
    require_fp16(residual, "residual")
    require_fp16(gamma, "gamma")
    if residual.shape != x.shape:
        raise RuntimeError("residual must have the same shape as x")
    D = x.shape[-1]
    if gamma.numel() != D:
        raise RuntimeError(f"gamma must have {D} elements")
    out = torch.empty_like(x)
    require_same_device(x, residual, gamma)
    with torch.cuda.device(x.device):
        check(lib().wbk_rmsnorm_f16(x.data_ptr(), residual.data_ptr(), gamma.data_ptr(), out.data_ptr(),
                                    x.numel() // D, D, float(eps), stream_of(x)), "rmsnorm_fused")
    _count()
    return out


# --------------------------------------------------------------------- GEMM

def _scale_arg(scale: Scale, name: str, device) -> tuple[float, Optional[int]]:
    if isinstance(scale, torch.Tensor):
        if scale.numel() != 1 or scale.dtype != torch.float32 or not scale.is_cuda:
            raise RuntimeError(f"{name} must be a Python float or a 1-element fp32 CUDA tensor")
        if scale.device != device:
            raise RuntimeError(f"{name} is on {scale.device}, expected {device}")
        return 1.0, scale.data_ptr()
    return float(scale), None


_SPLITK_WS: dict = {}
_SPLITK_OUTGROWN: dict = {}  # device: workspaces that were too small for a later call
_KV8_WS: list = []  # by device index


@_lib.on_device_timeout
def _zero_shared_workspaces(device_index: int) -> None:
    """After a device-side timeout a kernel may have left the sync words or split-K tickets of
    the device's shared workspaces non-zero; zero them again so the next call starts clean.
    (Workspaces passed by the caller are the caller's to zero, as wbk.h states.)"""
    shared = _KV8_WS[device_index] if device_index < len(_KV8_WS) else None
    dev = torch.device("cuda", device_index)
    for ws in (_SPLITK_WS.get(dev), shared, *_SPLITK_OUTGROWN.get(dev, ())):
        if ws is not None:
            ws.zero_()


def _zeros(nbytes: int, device: torch.device) -> torch.Tensor:
    with torch.inference_mode(False):  # a tensor made in inference mode could not be zeroed again outside it
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)


def splitk_workspace(device, nbytes: int) -> Optional[torch.Tensor]:
    """The per-device split-K workspace (zero-filled once, grown on demand).

    One that was outgrown is kept: a captured graph may hold its address. Each is at least twice the one before. A call
    in a capture that needs a larger one gets it for itself: it lies in the graph's memory, and only the replays zero it.
    Shared by every short-M GEMM on the device, so such GEMMs must not run
    concurrently on different streams; pass `workspace=` to gemm_fp8 to give a
    stream its own."""
    if nbytes <= 0:
        return None
    dev = torch.device(device)
    ws = _SPLITK_WS.get(dev)
    if ws is None or ws.numel() < nbytes:
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            return _zeros(nbytes, dev)
        if ws is not None:
            nbytes = max(nbytes, 2 * ws.numel())
        new = _zeros(nbytes, dev)
        if ws is not None:
            _SPLITK_OUTGROWN.setdefault(dev, []).append(ws)
        ws = _SPLITK_WS[dev] = new
    return ws


def _check_epilogue_args(epilogue, M: int, N: int, out_shape, bias, residual, out_amax) -> int:
    epi = _EPI_BY_NAME.get(epilogue)
    if epi is None:
        raise ValueError(f"unknown epilogue {epilogue!r}")
    if bias is not None:
        require_input(bias, "bias")
        require_fp16(bias, "bias")
        if bias.numel() != N:
            raise RuntimeError(f"bias must have {N} elements")
    if residual is not None:
        require_input(residual, "residual")
        require_fp16(residual, "residual")
        if residual.numel() != M * N:
            raise RuntimeError(f"residual must have shape {out_shape}")
    if epi in (EPI_RESIDUAL, EPI_RESIDUAL_CLAMP) and residual is None:
        raise RuntimeError("residual epilogue requires a residual tensor")
    if epi == EPI_BIAS_MAXKEY and out_amax is None:
        raise RuntimeError("the bias_maxkey epilogue requires out_amax")
    return epi


def gemm_fp8(a: torch.Tensor, a_scale: Scale, w: torch.Tensor, w_scale: Scale,
             bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, epilogue="none",
             a_format="e4m3", w_format="e4m3", out: Optional[torch.Tensor] = None,
             out_amax: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
             split_k: bool = True) -> torch.Tensor:
    """out[..., N] = epilogue(dq(a)[..., K] @ dq(w)[N, K]^T + bias); fp16 output.

    a: fp8 codes [..., K]; w: fp8 codes [N, K] (nn.Linear layout); scales as
    Python floats or 1-element fp32 CUDA tensors; epilogue one of
    'none' | 'gelu' | 'residual' | 'residual_clamp' | 'bias_maxkey' (bias only, and
    out_amax receives the order key of the largest output, for quantise_gelu).
    Short-M shapes (M <= 128) split K over more SMs (split_k=True) using
    `workspace` (a zero-filled uint8 CUDA tensor of at least
    wbk_gemm_fp8_ws_bytes bytes) or the device's shared one.
    """
    require_input(a, "a_fp8")
    require_input(w, "w_fp8")
    require_bytes(a, "a_fp8")
    require_bytes(w, "w_fp8")
    if w.dim() != 2:
        raise RuntimeError("w_fp8 must be 2-D [N, K]")
    N, K = w.shape
    if a.dim() < 1 or a.shape[-1] != K:
        raise RuntimeError(f"a_fp8 last dimension {a.shape[-1] if a.dim() else None} != K={K}")
    M = a.numel() // K if K else 0
    out_shape = tuple(a.shape[:-1]) + (N,)
    epi = _check_epilogue_args(epilogue, M, N, out_shape, bias, residual, out_amax)
    alpha_a, pa = _scale_arg(a_scale, "a_scale", a.device)
    alpha_w, pw = _scale_arg(w_scale, "w_scale", a.device)
    alpha = float(torch.tensor(alpha_a, dtype=torch.float32) * torch.tensor(alpha_w, dtype=torch.float32))
    o = torch.empty(out_shape, dtype=torch.float16, device=a.device) if out is None else out
    require_same_device(a, w, bias, residual, o, out_amax, workspace)
    with torch.cuda.device(a.device):
        ws = None
        if split_k and 0 < M <= 128:
            need = lib().wbk_gemm_fp8_ws_bytes(M, N, K)
            ws = workspace if workspace is not None else splitk_workspace(a.device, need)
        check(lib().wbk_gemm_fp8_ws(a.data_ptr(), w.data_ptr(), M, N, K, fmt_code(a_format), fmt_code(w_format),
                                    alpha, pa, pw, ptr(bias), ptr(residual), o.data_ptr(), epi, ptr(out_amax),
                                    ptr(ws), 0 if ws is None else ws.numel(), stream_of(a)),
              "gemm_fp8")
    _count()
    return o


def linear_fp8(x: torch.Tensor, w: torch.Tensor, w_scale: Scale, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, epilogue="none", a_format="e4m3", w_format="e4m3",
               out: Optional[torch.Tensor] = None, out_amax: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, scale_out: Optional[torch.Tensor] = None,
               amax_ws: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """FP8 linear on an fp16 activation: quantise(x) then gemm_fp8, as one call.

    x: fp16 [..., K]; w: fp8 codes [N, K]. Returns (out fp16 [..., N], x's codes
    uint8 [..., K], x's scale fp32 [1]) -- the codes and scale are exactly what
    quantise(x) returns, the output exactly gemm_fp8 of them. For M <= 128 rows
    this is one kernel (the GEMM quantises x itself) using `workspace` or the
    device's shared one; otherwise the quantiser kernel and the GEMM.
    """
    require_input(x, "x")
    require_fp16(x, "x")
    require_input(w, "w_fp8")
    require_bytes(w, "w_fp8")
    if w.dim() != 2:
        raise RuntimeError("w_fp8 must be 2-D [N, K]")
    N, K = w.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise RuntimeError(f"x last dimension {x.shape[-1] if x.dim() else None} != K={K}")
    M = x.numel() // K if K else 0
    out_shape = tuple(x.shape[:-1]) + (N,)
    epi = _check_epilogue_args(epilogue, M, N, out_shape, bias, residual, out_amax)
    alpha, pw = _scale_arg(w_scale, "w_scale", x.device)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device) if q_out is None else q_out
    sc = torch.empty(1, dtype=torch.float32, device=x.device) if scale_out is None else scale_out
    aws = torch.empty(1, dtype=torch.int32, device=x.device) if amax_ws is None else amax_ws
    o = torch.empty(out_shape, dtype=torch.float16, device=x.device) if out is None else out
    require_same_device(x, w, bias, residual, o, out_amax, q, sc, aws, workspace)
    with torch.cuda.device(x.device):
        ws = None
        if 0 < M <= 128:
            need = lib().wbk_gemm_fp8_ws_bytes(M, N, K)
            ws = workspace if workspace is not None else splitk_workspace(x.device, need)
        check(lib().wbk_linear_fp8_f16(x.data_ptr(), M, N, K, fmt_code(a_format), q.data_ptr(), sc.data_ptr(),
                                       aws.data_ptr(), w.data_ptr(), fmt_code(w_format), pw, alpha, ptr(bias),
                                       ptr(residual), o.data_ptr(), epi, ptr(out_amax), ptr(ws),
                                       0 if ws is None else ws.numel(), stream_of(x)),
              "linear_fp8")
    _count(1 if 0 < M <= 128 else 2)
    return o, q, sc


# ---------------------------------------------------------------- attention

def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor] = None,
              scale: Optional[float] = None, out_amax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Non-causal attention, head dim 64: softmax(q k^T * scale) v.

    q [B, H, Sq, 64], k and v [B, H, Sk, 64] fp16 CUDA views (any strides that
    are multiples of 8 elements, last dimension contiguous), e.g. the q/k/v
    slices of a fused QKV projection; `out` likewise (default: a new contiguous
    [B, H, Sq, 64] tensor). scale defaults to 1/sqrt(64). out_amax (optional, an
    amax workspace) max-accumulates max|out|.
    """
    for t, name in ((q, "Q"), (k, "K"), (v, "V")):
        require_cuda(t, name)
        require_fp16(t, name)
        if t.dim() != 4:
            raise RuntimeError(f"{name} must be 4D: [B, H, S, D]")
        if t.stride(-1) != 1:
            raise RuntimeError(f"{name} must have a contiguous last dimension")
    B, H, Sq, D = q.shape
    if k.shape[:2] != (B, H) or v.shape[:2] != (B, H) or k.shape[-1] != D or v.shape[-1] != D:
        raise RuntimeError("Q, K and V must agree in batch, heads and head dim")
    if k.shape[2] != v.shape[2]:
        raise RuntimeError("K and V must have the same sequence length")
    Sk = k.shape[2]
    o = torch.empty((B, H, Sq, D), dtype=torch.float16, device=q.device) if out is None else out
    if o.shape != (B, H, Sq, D) or o.dtype != torch.float16 or o.stride(-1) != 1:
        raise RuntimeError(f"out must be an fp16 [B, H, Sq, D] = {(B, H, Sq, D)} view with a contiguous last dimension")
    require_same_device(q, k, v, o, out_amax)
    strides = (ctypes.c_int64 * 12)(*(list(q.stride()[:3]) + list(k.stride()[:3]) + list(v.stride()[:3]) +
                                      list(o.stride()[:3])))
    sc = float(scale) if scale is not None else D ** -0.5
    with torch.cuda.device(q.device):
        check(lib().wbk_attention_f16(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B, H, Sq, Sk, D,
                                      strides, sc, ptr(out_amax), stream_of(q)), "attention")
    _count()
    return o


# ------------------------------------------------------ 8-bit key/value cache

# The calls below are made once per layer and token, so what they do on the host is kept short. Each first offers its
# arguments to the extension module of csrc/wbk_calls.cpp, which makes the call if they are all as the entry point needs
# them; what it hands back (None) goes through the checks here, which say what is wrong, or make the call.

_SHORT: list = []  # [the module, or None]


def _short():
    if not _SHORT:
        _SHORT.append(_lib.calls())
    return _SHORT[0]


_DT16 = {torch.float16: DT_F16, torch.bfloat16: DT_BF16}
_F8_DTYPE = {FMT_E4M3: torch.float8_e4m3fn, FMT_E5M2: torch.float8_e5m2}


_I64X6 = ctypes.c_int64 * 6
_BYTES8 = (torch.uint8, torch.int8)


def _launch(fn, args: tuple, index: int, what: str) -> None:
    """fn(*args, stream) on the current stream of CUDA device `index`."""
    if torch.cuda.current_device() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        check(status, what)
    LAUNCHES[0] += 1


def _require_on(index: int, t: torch.Tensor, name: str) -> None:
    """t is a contiguous tensor on CUDA device `index`."""
    if t.get_device() != index:
        require_cuda(t, name)
        raise RuntimeError(f"{name} is on {t.device}, expected cuda:{index}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _require_int32(index: int, t: torch.Tensor, name: str, numel: int) -> None:
    _require_on(index, t, name)
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != numel:
        raise RuntimeError(f"{name} must be int32 with shape [{numel}]")


def _require_bhsd(t: torch.Tensor, name: str) -> tuple:
    """(dtype number, device index, shape, strides) of a [B, H, S, D] fp16 or bf16 CUDA view with a contiguous last
    dimension; the stride of a dimension of one entry, which says nothing, is 0."""
    index = t.get_device()
    if index < 0:
        require_cuda(t, name)
    dt = _DT16.get(t.dtype)
    if dt is None:
        raise RuntimeError(f"{name} must be fp16 or bf16, got {t.dtype}")
    shape = t.shape
    if len(shape) != 4:
        raise RuntimeError(f"{name} must be 4D: [B, H, S, D]")
    sb, sh, ss, sd = t.stride()
    if sd != 1:
        raise RuntimeError(f"{name} must have a contiguous last dimension")
    b, h, s, _ = shape
    return dt, index, shape, (sb if b > 1 else 0, sh if h > 1 else 0, ss if s > 1 else 0)


def _require_cache(index, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, batch, kv_heads, head_dim, fmt):
    """Checks a cache against the batch that uses it; (format, pages, heads, block, max_blocks, table stride)."""
    f = fmt_code(fmt)
    shape = k_cache.shape
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _require_on(index, t, name)
        dtype = t.dtype
        if dtype is not _F8_DTYPE[f] and dtype not in _BYTES8:
            raise RuntimeError(f"{name} must hold {fmt} codes (uint8, int8 or {_F8_DTYPE[f]}), got {dtype}")
        if len(shape) != 4:
            raise RuntimeError(f"{name} must be 4D: [pages, kv_heads, block, head_dim]")
    if shape != v_cache.shape:
        raise RuntimeError("k_cache and v_cache must have the same shape")
    pages, heads, block, d = shape
    if d != head_dim or (kv_heads is not None and heads != kv_heads):
        raise RuntimeError(f"the cache holds {heads} heads of {d}; the call has {kv_heads or heads} of {head_dim}")
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        _require_on(index, t, name)
        if t.dtype is not torch.float32 or t.shape != (pages, heads):
            raise RuntimeError(f"{name} must be fp32 with shape {(pages, heads)}")
    if block_table.get_device() != index:
        _require_on(index, block_table, "block_table")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch:
        raise RuntimeError(f"block_table must be int32 with shape [{batch}, max_blocks]")
    width = block_table.shape[1]
    stride, inner = block_table.stride()
    if width > 1 and inner != 1:
        raise RuntimeError("block_table must have contiguous rows")
    _require_int32(index, seq_lens, "seq_lens", batch)
    return f, pages, heads, block, width, stride if batch > 1 else width


@functools.lru_cache(maxsize=4096)
def _kv8_ws_bytes(index: int, batch: int, heads: int, kv_heads: int, queries: int, head_dim: int) -> int:
    with torch.cuda.device(index):
        return int(lib().wbk_attention_kv8_ws_bytes(batch, heads, kv_heads, queries, head_dim))


def kv8_workspace(index: int) -> torch.Tensor:
    """The workspace of attention_kv8 on CUDA device `index`, shared by its calls there: calls that may run at the
    same time need workspaces of their own. Made on first use (outside a capture, whose replays alone would zero it),
    of the size that the largest call needs, and kept, so that captured graphs can hold its address."""
    while len(_KV8_WS) <= index:
        _KV8_WS.append(None)
    if _KV8_WS[index] is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first attention_kv8 on a device must run before a capture, or be given a workspace")
        nbytes = max(_kv8_ws_bytes(index, 1, 1, 1, rows, 128) for rows in (8, 1024))
        _KV8_WS[index] = _zeros(nbytes, torch.device("cuda", index))
    return _KV8_WS[index]


def kv8_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               new_lens: Optional[torch.Tensor] = None, fmt="e4m3") -> None:
    """Write new tokens' keys and values into the pages of an 8-bit cache, in place.

    k, v [B, Hkv, T, D] fp16 or bf16 CUDA views (strides multiples of 8 elements,
    last dimension contiguous); k_cache, v_cache [pages, Hkv, block, D] fp8 codes
    (uint8 or the float8 dtype of `fmt`), block 16 / 32 / 64 / 128, D 64 / 128;
    k_scale, v_scale [pages, Hkv] fp32; block_table [B, max_blocks] int32;
    seq_lens [B] int32: tokens each sequence holds BEFORE this call; new_lens [B]
    int32: how many of the T tokens are real (default: all).
    A page and head share one power-of-two scale; where a new token needs a larger
    one, the page's older codes are rescaled. Tokens past the table, or whose page
    is outside the pool, are not stored. seq_lens is not changed.
    """
    short = _short()
    if short is not None:
        status = short.kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens, fmt)
        if status is not None:
            check(status, "kv8_append")
            LAUNCHES[0] += 1
            return
    dt, index, shape, ks3 = _require_bhsd(k, "k")
    vdt, vindex, vshape, vs3 = _require_bhsd(v, "v")
    if vdt != dt or vshape != shape or vindex != index:
        raise RuntimeError("k and v must have the same shape and dtype, on one device")
    B, H, T, D = shape
    f, pages, _, block, width, ts = _require_cache(index, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, B, H,
                                                   D, fmt)
    if new_lens is not None:
        _require_int32(index, new_lens, "new_lens", B)
    _launch(lib().wbk_kv8_append,
            (k.data_ptr(), v.data_ptr(), dt, B, H, T, D, _I64X6(*ks3, *vs3), f, k_cache.data_ptr(), v_cache.data_ptr(),
             k_scale.data_ptr(), v_scale.data_ptr(), pages, block, block_table.data_ptr(), width, ts,
             seq_lens.data_ptr(), None if new_lens is None else new_lens.data_ptr()), index, "kv8_append")


def attention_kv8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  q_lens: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None,
                  fmt="e4m3", out: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q k^T * scale) v over the pages of an 8-bit cache.

    q [B, Hq, T, D] fp16 or bf16 CUDA view, Hq a multiple of the cache's heads; the
    cache, block_table as for kv8_append; seq_lens [B] int32: tokens each sequence
    holds now (the T queries' own included where causal); q_lens [B] int32: how
    many of the T rows are real (default: all). Causal row i of n sees the first
    seq_len - n + i + 1 tokens, otherwise all seq_len; a row that sees none, and a
    padding row, is 0. scale defaults to 1/sqrt(D). `out` (default: a new
    contiguous [B, Hq, T, D] tensor) takes the output in q's dtype.
    Long caches are split over the SMs through `workspace` (a zero-filled uint8
    CUDA tensor of at least wbk_attention_kv8_ws_bytes bytes) or the device's
    shared one, so such calls must not run concurrently on different streams
    without a workspace of their own.
    """
    short = _short()
    if short is not None:
        got = short.attention_kv8(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, q_lens, causal, scale, fmt,
                                  out, workspace, _KV8_WS)
        if got is not None:
            if type(got) is int:
                check(got, "attention_kv8")
            LAUNCHES[0] += 1
            return got
    dt, index, shape, qs3 = _require_bhsd(q, "q")
    B, H, T, D = shape
    f, pages, kv_heads, block, width, ts = _require_cache(index, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                                                          B, None, D, fmt)
    if kv_heads == 0 or H % kv_heads != 0:
        raise RuntimeError(f"{H} query heads do not share {kv_heads} KV heads evenly")
    if q_lens is not None:
        _require_int32(index, q_lens, "q_lens", B)
    if out is None:
        o = torch.empty(shape, dtype=q.dtype, device=q.device)
        os3 = (H * T * D, T * D, D)
    else:
        o = out
        odt, oindex, oshape, os3 = _require_bhsd(o, "out")
        if odt != dt or oindex != index or oshape != shape:
            raise RuntimeError(f"out must be a {q.dtype} view of shape {tuple(shape)} on {q.device}")
    if workspace is None:
        workspace = kv8_workspace(index)
    else:
        _require_on(index, workspace, "workspace")
    _launch(lib().wbk_attention_kv8,
            (q.data_ptr(), o.data_ptr(), dt, B, H, kv_heads, T, D, _I64X6(*qs3, *os3), f, k_cache.data_ptr(),
             v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, block, block_table.data_ptr(), width, ts,
             seq_lens.data_ptr(), None if q_lens is None else q_lens.data_ptr(), 1 if causal else 0,
             D ** -0.5 if scale is None else float(scale), workspace.data_ptr(),
             workspace.numel() * workspace.element_size()), index, "attention_kv8")
    return o


# ----------------------------------------------------------------- sampling

_DT_LOGITS = {torch.float16: DT_F16, torch.bfloat16: DT_BF16, torch.float32: DT_F32}


def _per_row(index: int, value, name: str, dtype: torch.dtype, rows: int):
    """(number for every row, address of a device array or None)."""
    if isinstance(value, torch.Tensor):
        _require_on(index, value, name)
        if value.dtype is not dtype or value.dim() != 1 or value.shape[0] != rows:
            raise RuntimeError(f"{name} must be a number or a {dtype} tensor of shape [{rows}]")
        return 0, value.data_ptr()
    if not value >= 0:
        raise ValueError(f"{name} must not be negative, got {value}")
    return value, None


def _require_rows(index: int, t: torch.Tensor, name: str) -> int:
    """The row stride of a [B, V] tensor on CUDA device `index` whose rows are contiguous."""
    if t.get_device() != index:
        _require_on(index, t, name)
    (rows, width), (stride, inner) = t.shape, t.stride()
    if width > 1 and inner != 1:
        raise RuntimeError(f"{name} must have contiguous rows")
    return stride if rows > 1 else width


def sample(logits: torch.Tensor, noise: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           tokens_out: Optional[torch.Tensor] = None,
           logprobs_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Draw one token per row of logits; (tokens int64 [B], logprobs fp32 [B]).

    logits [B, V] fp16, bf16 or fp32; noise [B, V] fp32 of independent Exp(1)
    numbers (torch.Tensor.exponential_), both with contiguous rows. temperature,
    top_p, min_p: a number or an fp32 CUDA tensor [B]; top_k: a number or an int32
    CUDA tensor [B]. Filters apply in the order temperature, top_k, top_p (of what
    top_k left), min_p (relative to the largest probability); temperature 0 is
    greedy, top_k 0, top_p 1 and min_p 0 filter nothing. Ties go to the lowest
    index; equal inputs give equal tokens. logprobs is the token's log-probability
    under the unfiltered softmax of the logits as given. A row with no logit above
    -inf gives token -1 and logprob -inf.
    """
    short = _short()
    if short is not None and tokens_out is None and logprobs_out is None:
        got = short.sample(logits, noise, temperature, top_k, top_p, min_p)
        if got is not None:
            if type(got) is int:
                check(got, "sample")
            LAUNCHES[0] += 1
            return got
    index = logits.get_device()
    if index < 0:
        require_cuda(logits, "logits")
    dt = _DT_LOGITS.get(logits.dtype)
    if dt is None:
        raise RuntimeError(f"logits must be fp16, bf16 or fp32, got {logits.dtype}")
    if logits.dim() != 2:
        raise RuntimeError("logits must be 2-D [B, V]")
    B, V = logits.shape
    if noise.dtype is not torch.float32 or noise.shape != logits.shape:
        raise RuntimeError(f"noise must be fp32 with shape {(B, V)}")
    ls, ns = _require_rows(index, logits, "logits"), _require_rows(index, noise, "noise")
    t_all, t_row = _per_row(index, temperature, "temperature", torch.float32, B)
    k_all, k_row = _per_row(index, top_k, "top_k", torch.int32, B)
    p_all, p_row = _per_row(index, top_p, "top_p", torch.float32, B)
    m_all, m_row = _per_row(index, min_p, "min_p", torch.float32, B)
    if tokens_out is None:
        tokens_out = torch.empty(B, dtype=torch.int64, device=logits.device)
    elif tokens_out.dtype is not torch.int64 or tokens_out.shape != (B,):
        raise RuntimeError(f"tokens_out must be int64 with shape [{B}]")
    else:
        _require_on(index, tokens_out, "tokens_out")
    if logprobs_out is None:
        logprobs_out = torch.empty(B, dtype=torch.float32, device=logits.device)
    elif logprobs_out.dtype is not torch.float32 or logprobs_out.shape != (B,):
        raise RuntimeError(f"logprobs_out must be fp32 with shape [{B}]")
    else:
        _require_on(index, logprobs_out, "logprobs_out")
    _launch(lib().wbk_sample,
            (logits.data_ptr(), dt, B, V, ls, noise.data_ptr(), ns, t_row, k_row, p_row, m_row, t_all,
             min(int(k_all), 2 ** 31 - 1), p_all, m_all, tokens_out.data_ptr(), logprobs_out.data_ptr()),
            index, "sample")
    return tokens_out, logprobs_out
