"""On-device FP8 / NVFP4 weight quantisation (fa_quantize_fp8_rows / fa_quantize_nvfp4 in
include/flashact.h) and the product with NVFP4 weights (fa_nvfp4_linear): the codes and scales Pi05ActionExpert(wfmt="fp8" | "nvfp4") takes, computed
on the GPU from bf16 / fp16 / fp32 weights. The reference quantises on the host inside
HybridPi05._pack_weights (src/pi05/hybrid_model.py:105-110). No CPU fallback."""
from __future__ import annotations

import ctypes

import torch

from . import _capi as C
from .pi05 import _DT, _stream_ptr, on_stream


def _prep(w: torch.Tensor):
    if not w.is_cuda:
        raise C.FlashActError(C.FA_ERR_INVALID, "the weights must be a CUDA tensor")
    if w.dtype not in _DT:
        w = w.float()
    w = w.contiguous()
    w3 = w.view(-1, w.shape[-2], w.shape[-1]) if w.dim() >= 2 else w.view(1, 1, -1)
    return w, w3.shape


def _check(lib, st):
    if st != C.FA_OK:
        raise C.FlashActError(st, lib.fa_last_error(None).decode(errors="replace"))


def quantize_fp8_rows(w: torch.Tensor):
    """w [..., rows, K] -> (codes uint8 [..., rows, K], scale fp32 [..., rows]); per-row E4M3
    with scale max(amax, 1e-8) / 448."""
    lib = C.load_library()
    w, (L, R, K) = _prep(w)
    with torch.cuda.device(w.device):
        codes = torch.empty(w.shape, dtype=torch.uint8, device=w.device)
        scale = torch.empty(w.shape[:-1], dtype=torch.float32, device=w.device)
        _check(lib, lib.fa_quantize_fp8_rows(ctypes.c_void_p(w.data_ptr()), _DT[w.dtype], L, R, K,
                                             ctypes.c_void_p(codes.data_ptr()), ctypes.c_void_p(scale.data_ptr()),
                                             _stream_ptr()))
    return codes, scale


def quantize_nvfp4(w: torch.Tensor):
    """w [L, rows, K] (K % 16 == 0) -> (packed E2M1 codes uint8 [L, rows, K/2], E4M3 block scales
    as uint8 [L, rows, K/16], fp32 tensor scale [L])."""
    lib = C.load_library()
    if w.dim() != 3:
        raise C.FlashActError(C.FA_ERR_INVALID, "nvfp4 quantisation takes [L, rows, K]")
    w, (L, R, K) = _prep(w)
    with torch.cuda.device(w.device):
        packed = torch.empty(L, R, K // 2, dtype=torch.uint8, device=w.device)
        bscale = torch.empty(L, R, K // 16, dtype=torch.uint8, device=w.device)
        tscale = torch.empty(L, dtype=torch.float32, device=w.device)
        _check(lib, lib.fa_quantize_nvfp4(ctypes.c_void_p(w.data_ptr()), _DT[w.dtype], L, R, K,
                                          ctypes.c_void_p(packed.data_ptr()), ctypes.c_void_p(bscale.data_ptr()),
                                          ctypes.c_void_p(tscale.data_ptr()), _stream_ptr()))
    return packed, bscale, tscale


def nvfp4_linear(x: torch.Tensor, packed: torch.Tensor, block_scale: torch.Tensor, tensor_scale: torch.Tensor, *,
                 bias: torch.Tensor | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """x W^T * tensor_scale (+ bias) for x [..., K] (bf16 or fp16) of up to 16 rows and one layer's matrix as
    quantize_nvfp4 gives it: packed uint8 [N, K/2], block_scale uint8 [N, K/16], tensor_scale fp32 of one element;
    bias fp32 [N]. Returns [..., N] in x's type; `out` may not overlap x."""
    dt, shape, index = _DT.get(x.dtype), x.shape, x.get_device()
    if dt is None or not shape or index < 0:
        raise C.FlashActError(C.FA_ERR_INVALID, "x must be a CUDA tensor [..., K]")
    if stream is not None or torch._C._cuda_getDevice() != index:
        with on_stream(stream, index, x, packed, block_scale, tensor_scale, bias, out):
            return nvfp4_linear(x, packed, block_scale, tensor_scale, bias=bias, out=out)
    K, pshape = shape[-1], packed.shape
    N = pshape[0] if len(pshape) == 2 else 0
    if (pshape != (N, K // 2) or packed.dtype != torch.uint8 or packed.get_device() != index or not packed.is_contiguous()
            or block_scale.shape != (N, K // 16) or block_scale.dtype != torch.uint8 or block_scale.get_device() != index
            or not block_scale.is_contiguous() or tensor_scale.numel() != 1 or tensor_scale.dtype != torch.float32
            or tensor_scale.get_device() != index or bias is not None
            and (bias.shape != (N,) or bias.dtype != torch.float32 or bias.get_device() != index or not bias.is_contiguous())):
        _bad_operand(x, ("packed", packed, (N, K // 2), torch.uint8), ("block_scale", block_scale, (N, K // 16), torch.uint8),
                     ("tensor_scale", tensor_scale, None, torch.float32), ("bias", bias, (N,), torch.float32))
    if out is None:
        out = x.new_empty((*shape[:-1], N))
    elif out.shape != (*shape[:-1], N) or out.dtype != x.dtype or out.get_device() != index or not out.is_contiguous():
        raise C.FlashActError(C.FA_ERR_INVALID, f"'out' must be a contiguous {x.dtype} tensor {(*shape[:-1], N)} on {x.device}")
    if not x.is_contiguous():
        x = x.contiguous()
    p = x.data_ptr()
    if p % 16:
        x = x.clone()
        p = x.data_ptr()
    lib = C.load_library()
    st = lib.fa_nvfp4_linear(p, dt, x.numel() // K if K else 0, K, K, packed.data_ptr(), block_scale.data_ptr(), tensor_scale.data_ptr(),
                             None if bias is None else bias.data_ptr(), N, out.data_ptr(), N,
                             torch._C._cuda_getCurrentRawStream(index))
    if st != C.FA_OK:
        _check(lib, st)
    return out


def _bad_operand(x, *operands):
    for name, t, shape, dtype in operands:
        if t is not None and ((t.numel() != 1 if shape is None else t.shape != shape) or t.dtype != dtype or t.device != x.device
                              or not t.is_contiguous()):
            raise C.FlashActError(C.FA_ERR_INVALID, f"'{name}' must be a contiguous {dtype} tensor {shape or '(one element)'} on "
                                                    f"{x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
