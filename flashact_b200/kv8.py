"""A prefix KV cache in 8 bits (fa_kv8_* in include/flashact.h): E4M3 codes with a power-of-two scale for each
block of tokens and head, half the bytes of the bf16 prefix that the action experts bind. Tokens are appended on
the GPU, queries attend to them as they are, and bind_prefix_cache / bind_context_cache of the engines take the
values. No CPU fallback."""
from __future__ import annotations

import ctypes

import torch

from . import _capi as C
from .pi05 import _DT, on_stream

_byref = ctypes.byref
_current_device = torch._C._cuda_getDevice


# the raw current stream of a device: torch.cuda.current_stream(index).cuda_stream without the object
_current_stream = torch._C._cuda_getCurrentRawStream


def _bad(msg):
    return C.FlashActError(C.FA_ERR_INVALID, msg)


class Kv8Cache:
    """K and V of `batch` observations, `layers` layers and `heads` key heads, up to `capacity` tokens (rounded up to
    whole blocks). `lens` (int32 [batch], on the device) counts the tokens of each observation; it is changed by
    advance() and by the caller, not by append(), so that every layer of a step appends at the same place."""

    def __init__(self, batch: int, layers: int, heads: int, head_dim: int, capacity: int, *, block: int = 64,
                 device: int | str | torch.device = 0):
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        cap = -(-capacity // block) * block if block > 0 else capacity
        shape = (batch, layers, heads)
        if min(shape) < 1 or cap < 1:
            raise _bad(f"a cache of batch, layers, heads = {shape} and {capacity} tokens")
        self._own(torch.zeros(*shape, cap, head_dim, dtype=torch.uint8, device=dev),
                  torch.zeros(*shape, head_dim, cap, dtype=torch.uint8, device=dev),
                  torch.full((*shape, cap // block), 2.0 ** -96, device=dev),
                  torch.full((*shape, cap // block), 2.0 ** -96, device=dev),
                  torch.zeros(batch, dtype=torch.int32, device=dev))

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale, *, lens=None):
        """A cache over tensors that the caller owns, in the layout of fa_kv8: k uint8 [batch][layers][heads][capacity]
        [head_dim], v uint8 [batch][layers][heads][head_dim][capacity], scales fp32 [batch][layers][heads][blocks],
        lens int32 [batch]; contiguous, on one GPU."""
        self = cls.__new__(cls)
        if lens is None and k.dim():
            lens = torch.zeros(k.shape[0], dtype=torch.int32, device=k.device)
        self._own(k, v, k_scale, v_scale, lens)
        return self

    def _own(self, k, v, k_scale, v_scale, lens):
        if k.dim() != 5 or v.dim() != 5 or k_scale.dim() != 4:
            raise _bad("k and v have five dimensions, the scales four")
        b, layers, heads, cap, d = k.shape
        blocks = k_scale.shape[3]
        if not blocks or cap % blocks:
            raise _bad(f"{blocks} blocks for a capacity of {cap}")
        for name, t, shape, dt in (("k", k, (b, layers, heads, cap, d), torch.uint8), ("v", v, (b, layers, heads, d, cap), torch.uint8),
                                   ("k_scale", k_scale, (b, layers, heads, blocks), torch.float32),
                                   ("v_scale", v_scale, (b, layers, heads, blocks), torch.float32),
                                   ("lens", lens, (b,), torch.int32)):
            if tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous() or t.device != k.device or not t.is_cuda:
                raise _bad(f"'{name}' must be a contiguous {dt} CUDA tensor of shape {shape} on k's device, "
                           f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        self.k, self.v, self.k_scale, self.v_scale, self._lens_tensor = k, v, k_scale, v_scale, lens
        self.batch, self.layers, self.heads, self.capacity, self.head_dim = b, layers, heads, cap, d
        self.block = cap // blocks
        self.device = k.device
        self.lib = C.load_library()
        self._c = C.FaKv8(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), b, layers, heads, d, cap,
                          self.block)
        self._ref = ctypes.byref(self._c)
        self._ws = {}  # workspace bytes of the last shapes asked for
        self._index, self._lens, self._scale = self.device.index, lens.data_ptr(), d ** -0.5
        self._append, self._attention = self.lib.fa_kv8_append, self.lib.fa_kv8_attention

    @property
    def lens(self):
        return self._lens_tensor

    @lens.setter
    def lens(self, t):
        if t is None:
            raise _bad("'lens' must be a tensor")
        self._lens, self._lens_tensor = self._ints("lens", t), t

    def tensors(self):
        """The memory that the cache is: k, v, k_scale, v_scale, lens."""
        return self.k, self.v, self.k_scale, self.v_scale, self._lens_tensor

    def _check(self, st):
        if st != C.FA_OK:
            C.check(self.lib, None, st)

    def _rows(self, name, t, heads):
        shape = t.shape
        if len(shape) != 4 or shape[0] != self.batch or shape[2] != heads or shape[3] != self.head_dim:
            raise _bad(f"'{name}' must be [{self.batch}][tokens][{heads}][{self.head_dim}], got {tuple(shape)}")
        if t.get_device() != self._index:
            raise _bad(f"'{name}' is on {t.device}, the cache on {self.device}")
        st = t.stride()
        if st[3] != 1:
            t = t.contiguous()
            st = t.stride()
        return t, C.FaRows(t.data_ptr(), st[0], st[1], st[2])

    def _ints(self, name, t):
        if t is None:
            return None
        if t.dtype != torch.int32 or t.shape != self._lens_tensor.shape or not t.is_contiguous() or t.get_device() != self._index:
            raise _bad(f"'{name}' must be a contiguous int32 tensor [{self.batch}] on {self.device}")
        return t.data_ptr()

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, *, count: torch.Tensor | None = None,
               start: torch.Tensor | None = None, stream=None):
        """Quantises k, v [batch][tokens][heads][head_dim] (fp32, bf16 or fp16, any strides) into `layer` behind `start`
        (default: lens). count (int32 [batch]) gives each observation's number of real rows in a padded batch."""
        if stream is not None or _current_device() != self._index:
            with on_stream(stream, self._index, k, v, count, start, *self.tensors()):
                return self.append(layer, k, v, count=count, start=start)
        dt = _DT.get(k.dtype)
        if dt is None or v.dtype != k.dtype:
            raise _bad(f"k and v must share fp32, bf16 or fp16, got {k.dtype} and {v.dtype}")
        k, kr = self._rows("k", k, self.heads)
        v, vr = self._rows("v", v, self.heads)
        rows = k.shape[1]
        if v.shape[1] != rows:
            raise _bad(f"{rows} rows of k and {v.shape[1]} of v")
        self._check(self._append(self._ref, layer, rows, _byref(kr), _byref(vr), dt,
                                 self._lens if start is None else self._ints("start", start), self._ints("count", count),
                                 _current_stream(self._index)))

    def advance(self, n, *, stream=None):
        """lens += n (a number, or a tensor [batch]) after every layer has appended, on the stream of the appends: those on `stream` that
        have not run yet still read the lengths."""
        with on_stream(stream, self._index, self._lens_tensor, n if isinstance(n, torch.Tensor) else None):
            self._lens_tensor += n

    def attend(self, layer: int, q: torch.Tensor, *, scale: float | None = None, causal: bool = True,
               prefix: torch.Tensor | None = None, q_lens: torch.Tensor | None = None, lens: torch.Tensor | None = None,
               max_len: int = 0, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """softmax(scale q K^T + mask) V for q [batch][tokens][q_heads][head_dim] (bf16 or fp16, any strides); scale
        defaults to head_dim ** -0.5. lens (default: the cache's) counts the cached tokens, the queries' own among
        them. causal: token i of an observation's q_lens (default: tokens) stands at lens - q_lens + i and sees the
        keys up to there, and all below prefix; not causal: every key. max_len: an upper bound of lens that the host knows
        (default: the capacity). `out` may be q itself, but may not overlap it in another way. Its rows behind
        q_lens are left as they were (zero in a new tensor)."""
        if stream is not None or _current_device() != self._index:
            with on_stream(stream, self._index, q, prefix, q_lens, lens, out, *self.tensors()):
                return self.attend(layer, q, scale=scale, causal=causal, prefix=prefix, q_lens=q_lens, lens=lens,
                                   max_len=max_len, out=out)
        dt, shape = _DT.get(q.dtype), q.shape
        if dt is None or len(shape) != 4:
            raise _bad(f"q must be a bf16 or fp16 tensor of four dimensions, got {q.dtype} {tuple(shape)}")
        tokens, q_heads = shape[1], shape[2]
        q, qr = self._rows("q", q, q_heads)
        if out is None:  # contiguous like q, or of its own where q is not
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
            if q_lens is not None:
                out.zero_()
        elif out.shape != shape or out.dtype != q.dtype or out.device != self.device or (out.numel() and out.stride(3) != 1):
            raise _bad(f"'out' must be like q ({q.dtype} {tuple(shape)}) with a contiguous last dimension")
        st = out.stride()
        orow = C.FaRows(out.data_ptr(), st[0], st[1], st[2])
        need = self._ws.get((tokens, q_heads, max_len))
        if need is None:
            n = ctypes.c_size_t()
            self._check(self.lib.fa_kv8_attention_workspace(self._ref, tokens, q_heads, max_len, _byref(n)))
            if len(self._ws) >= 64:  # a caller whose max_len follows each step
                self._ws.clear()
            need = self._ws[tokens, q_heads, max_len] = n.value
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._check(self._attention(
            self._ref, layer, tokens, q_heads, _byref(qr), dt, self._lens if lens is None else self._ints("lens", lens),
            self._ints("q_lens", q_lens), self._ints("prefix", prefix), causal, self._scale if scale is None else scale, max_len,
            _byref(orow), ws.data_ptr() if need else None, need, _current_stream(self._index)))
        return out

    def read(self, rows: int, *, dtype=torch.bfloat16, lens: torch.Tensor | None = None, stream=None):
        """(K, V) as values [batch][layers][rows][heads * head_dim], zero at and behind each length."""
        if stream is not None or _current_device() != self._index:
            with on_stream(stream, self._index, lens, *self.tensors()):
                return self.read(rows, dtype=dtype, lens=lens)
        if dtype not in _DT:
            raise _bad(f"values are fp32, bf16 or fp16, not {dtype}")
        if rows < 0:
            raise _bad(f"rows={rows}")
        shape = (self.batch, self.layers, rows, self.heads * self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._check(self.lib.fa_kv8_read(self._ref, self._lens if lens is None else self._ints("lens", lens), rows, k.data_ptr(),
                                         v.data_ptr(), _DT[dtype], _current_stream(self._index)))
        return k, v
