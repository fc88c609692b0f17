"""Block-scaled FP8: the linear for layers that four bits hurt (output heads, sensitive projections), at half the bytes of bf16.

    activations   E4M3 codes and one fp32 scale for every row and 128 columns
    weights       E4M3 codes and one fp32 scale for every 128 x 128 tile
    scale         the block's largest magnitude / 448 (1 where that is zero); code = e4m3(fp32(value / scale))
    y[m, n]     = sum over blocks b of (sx[m, b] * sw[n // 128, b]) * (sum of code products in b), in fp32, rounded once

The two scales are multiplied first, in fp32: blocks whose product of scales leaves its range do so too (largest magnitude of x times
that of the weight above 6.8e43; below 2.4e-33 it loses bits).  A bias is added to the rounded y, in y's type, as `mixfp4_linear` does.

The reference keeps such layers in bf16 (project_quant/modeling.py:65-68 leaves output heads out of the walk); there is no
counterpart of this format in it.  Inputs that are not finite make their block's scale, and the results that read it, NaN.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch
from torch import nn

from . import _native as nat
from .linear import _status_word

FP8_BLOCK = 128


def _blocks(size: int) -> int:
    return -(-size // FP8_BLOCK)


def _addressable(codes: torch.Tensor) -> bool:
    """Rows that a tensor map can address: unit stride along K, each on 16 bytes."""
    return codes.stride(1) == 1 and codes.stride(0) >= codes.shape[1] and codes.stride(0) % 16 == 0 and codes.data_ptr() % 16 == 0


def _codes_for_kernels(codes: torch.Tensor) -> torch.Tensor:
    """The codes with rows that a tensor map can address (16-byte aligned); themselves where they are so already."""
    rows, k = codes.shape
    if _addressable(codes):
        return codes
    held = torch.empty((rows, _blocks(k) * FP8_BLOCK), dtype=codes.dtype, device=codes.device)[:, :k]
    held.copy_(codes)
    return held


def _check_parts(codes: torch.Tensor, scales: torch.Tensor, rows_per_scale: int) -> torch.Tensor:
    if codes.dtype == torch.uint8:
        codes = codes.view(torch.float8_e4m3fn)
    if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
        raise TypeError("codes must be float8_e4m3fn (or its bytes), scales float32")
    if codes.ndim != 2 or codes.shape[1] == 0 or codes.shape[0] == 0 and rows_per_scale > 1:
        raise ValueError("codes must be a matrix with at least one row and column")
    want = (-(-codes.shape[0] // rows_per_scale), _blocks(codes.shape[1]))
    if tuple(scales.shape) != want:
        raise ValueError(f"scales must have the shape {want}, one for each block of the codes, not {tuple(scales.shape)}")
    if codes.device != scales.device:
        raise ValueError("codes and scales must be on the same device")
    return codes


@dataclass
class FP8Weight:
    """A quantized [n, k] weight: codes float8_e4m3fn [n, k] with 16-byte aligned rows, scales float32 [ceil(n/128), ceil(k/128)],
    contiguous.  (`from_tensors` takes any strides and brings them there.)"""

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        self.codes = _check_parts(self.codes, self.scales, FP8_BLOCK)
        if not _addressable(self.codes) or not self.scales.is_contiguous():
            raise ValueError("a weight's code rows are 16-byte aligned and its scales contiguous: FP8Weight.from_tensors makes them so")
        self.n, self.k = self.codes.shape

    @classmethod
    def _made(cls, codes, scales) -> "FP8Weight":
        """Parts that this module made itself: nothing to check."""
        w = object.__new__(cls)
        w.codes, w.scales = codes, scales
        w.n, w.k = codes.shape
        return w

    @classmethod
    def from_tensors(cls, codes: torch.Tensor, scales: torch.Tensor) -> "FP8Weight":
        """Codes (float8_e4m3fn or their bytes) and scales of a checkpoint; copied only where their rows are not aligned."""
        codes = _check_parts(codes, scales, FP8_BLOCK)
        return cls(_codes_for_kernels(codes), scales.contiguous())

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.n * self.k + self.scales.numel() * 4

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize_fp8(self, dtype)

    def to(self, device) -> "FP8Weight":
        return FP8Weight.from_tensors(self.codes.to(device), self.scales.to(device))


@dataclass
class FP8Activations:
    """Quantized rows: codes float8_e4m3fn [m, k]; scales float32 [m, ceil(k/128)], a view whose columns are contiguous and
    padded to 128 rows (what the product fetches).  `shape` and `dtype` are the source's.  (`from_tensors` takes any strides
    and brings them there.)"""

    codes: torch.Tensor
    scales: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    def __post_init__(self):
        codes, scales = _check_parts(self.codes, self.scales, 1), self.scales
        m, k = codes.shape
        room, ld = _blocks(m) * FP8_BLOCK, scales.stride(1)
        held = scales.untyped_storage().nbytes() // 4 - scales.storage_offset()
        if (not _addressable(codes) or m > 1 and scales.stride(0) != 1 or m and (ld < room or ld % 4 != 0 or scales.data_ptr() % 16 != 0
                                                                                or held < (scales.shape[1] - 1) * ld + room)):
            raise ValueError("code rows are 16-byte aligned, and columns of scales have room for 128 rows: FP8Activations.from_tensors "
                             "makes them so")
        if self.shape[-1] != k or math.prod(self.shape[:-1]) != m:
            raise ValueError(f"codes {tuple(codes.shape)} are not rows of a tensor of shape {tuple(self.shape)}")
        self.codes = codes

    @classmethod
    def _made(cls, codes, scales, shape, dtype) -> "FP8Activations":
        """Parts that this module made itself: nothing to check."""
        q = object.__new__(cls)
        q.codes, q.scales, q.shape, q.dtype = codes, scales, shape, dtype
        return q

    @classmethod
    def from_tensors(cls, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> "FP8Activations":
        codes = _check_parts(codes, scales, 1)
        held = _scale_room(codes.shape[0], codes.shape[1], codes.device)
        held.copy_(scales)
        return cls(_codes_for_kernels(codes), held, codes.shape, dtype)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        return dequantize_fp8(self, self.dtype if dtype is None else dtype).reshape(self.shape)


def _scale_room(m: int, k: int, device) -> torch.Tensor:
    room, blocks = _blocks(m) * FP8_BLOCK, _blocks(k)
    held = torch.empty_strided((room, blocks), (1, room), dtype=torch.float32, device=device)
    return held if m == room else held.as_strided((m, blocks), (1, room))      # a microsecond less than a slice


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """[..., K] as rows with unit stride along K and a row stride of at least K."""
    nat.require_cuda(x, what)
    if x.dtype not in nat.DTYPE_CODE:
        raise TypeError(f"{what} must be bfloat16, float16 or float32")
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"{what} must have at least one column")
    x2 = x if len(shape) == 2 else x.reshape(-1, shape[-1])
    ld, step = x2.stride()
    if ld >= shape[-1] and step == 1:
        return x2
    x2 = x2.reshape(1, -1) if x2.shape[0] == 1 and step == 1 else x2.contiguous()
    if x2.stride(0) < shape[-1]:                         # a single row, whose stride can be any number
        x2 = x2.as_strided(x2.shape, (shape[-1], 1))
    return x2


def quantize_fp8_weight(w: torch.Tensor) -> FP8Weight:
    """A dense [n, k] weight (bf16, f16 or fp32, on the GPU) to codes and a scale for every 128 x 128 tile, in one pass."""
    if w.ndim != 2 or 0 in w.shape:
        raise ValueError("the weight must be a matrix with at least one row and column")
    w = _rows(w, "the weight")
    (n, k), device = w.shape, w.device
    blocks = _blocks(k)
    ld = blocks * FP8_BLOCK
    codes = torch.empty_strided((n, ld), (ld, 1), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty_strided((_blocks(n), blocks), (blocks, 1), dtype=torch.float32, device=device)
    with nat.on_device(device):
        st = nat.lib().mixfp4_fp8_quantize_tiles(w.data_ptr(), nat.DTYPE_CODE[w.dtype], n, k, w.stride(0), codes.data_ptr(), ld,
                                                 scales.data_ptr(), nat.stream_ptr(device))
    nat.check("mixfp4_fp8_quantize_tiles", st)
    return FP8Weight._made(codes if ld == k else codes.as_strided((n, k), (ld, 1)), scales)


def quantize_fp8_activations(x: torch.Tensor) -> FP8Activations:
    """Rows [..., K] to codes and a scale for every row and 128 columns: once for all the weights that read them."""
    x2 = _rows(x, "x")
    (m, k), device = x2.shape, x.device
    ld = _blocks(k) * FP8_BLOCK
    codes = torch.empty_strided((m, ld), (ld, 1), dtype=torch.float8_e4m3fn, device=device)      # a microsecond less than torch.empty
    scales = _scale_room(m, k, device)
    if m:
        with nat.on_device(device):
            st = nat.lib().mixfp4_fp8_quantize_rows(x2.data_ptr(), nat.DTYPE_CODE[x.dtype], m, k, x2.stride(0), codes.data_ptr(), ld,
                                                    scales.data_ptr(), _blocks(m) * FP8_BLOCK, nat.stream_ptr(device))
        nat.check("mixfp4_fp8_quantize_rows", st)
    return FP8Activations._made(codes if ld == k else codes.as_strided((m, k), (ld, 1)), scales, x.shape, x.dtype)


def dequantize_fp8(q: FP8Weight | FP8Activations, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """code * scale as a dense matrix, rounded once."""
    if dtype not in nat.DTYPE_CODE:
        raise TypeError("dtype must be bfloat16, float16 or float32")
    nat.require_cuda(q.codes, "codes")
    rows, k = q.codes.shape
    out = torch.empty((rows, k), dtype=dtype, device=q.device)
    if rows:
        with nat.on_device(q.device):
            st = nat.lib().mixfp4_fp8_dequant(q.codes.data_ptr(), q.codes.stride(0), q.scales.data_ptr(), q.scales.stride(0),
                                              q.scales.stride(1), FP8_BLOCK if isinstance(q, FP8Weight) else 1, rows, k,
                                              out.data_ptr(), nat.DTYPE_CODE[dtype], k, nat.stream_ptr(q.device))
        nat.check("mixfp4_fp8_dequant", st)
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(m: int, k: int) -> int:
    """The library's answer, a function of the sizes alone: half a microsecond less than asking again."""
    return nat.lib().mixfp4_fp8_workspace_bytes(m, k)


def fp8_linear(x: torch.Tensor | FP8Activations, weight: FP8Weight, *, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = x @ W^T (+ bias) on block-scaled FP8 operands.  x: a dense tensor [..., K] (bf16, f16 or fp32), quantized within
    the call, or what `quantize_fp8_activations` made of one.  out_dtype: bf16, f16 or fp32 (default: x's dtype).  bias [n]: rounded
    to that type and added to the rounded product, so a biased result is rounded twice (out_dtype=torch.float32 leaves the
    rounding to the caller).  A product whose device-side waits run out reports through `gemm_status()`, like the other GEMMs."""
    codes, n, k = weight.codes, weight.n, weight.k
    device, shape = codes.device, x.shape
    out_dtype = x.dtype if out_dtype is None else out_dtype
    out_code = nat.DTYPE_CODE.get(out_dtype)
    if out_code is None:
        raise TypeError("out_dtype must be bfloat16, float16 or float32")
    if shape[-1] != k:
        raise ValueError(f"x has K={shape[-1]}, the weight K={k}")
    if x.device != device:
        raise ValueError(f"x is on {x.device}, the weight on {device}")
    nat.require_cuda(codes, "the weight")
    quantized = isinstance(x, FP8Activations)
    x2 = x.codes if quantized else _rows(x, "x")
    m = x2.shape[0]
    y = torch.empty_strided((m, n), (n, 1), dtype=out_dtype, device=device)      # a microsecond less than torch.empty
    if m:
        lib = nat.lib()
        with nat.on_device(device):
            stream = nat.stream_ptr(device)
            if quantized:
                st = lib.mixfp4_fp8_gemm(x2.data_ptr(), x2.stride(0), x.scales.data_ptr(), x.scales.stride(1), codes.data_ptr(),
                                         codes.stride(0), weight.scales.data_ptr(), m, n, k, y.data_ptr(), out_code, n,
                                         _status_word(device).data_ptr(), stream)
                nat.check("mixfp4_fp8_gemm", st)
            else:
                nbytes = _workspace_bytes(m, k)
                work = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None      # a captured graph's own
                st = lib.mixfp4_fp8_linear(x2.data_ptr(), nat.DTYPE_CODE[x2.dtype], m, x2.stride(0), codes.data_ptr(),
                                           codes.stride(0), weight.scales.data_ptr(), n, k, y.data_ptr(), out_code, n,
                                           nat.ptr(work), nbytes, _status_word(device).data_ptr(), stream)
                nat.check("mixfp4_fp8_linear", st)
    if bias is not None:
        y += bias.to(y.dtype)
    return y if len(shape) == 2 else y.reshape(*shape[:-1], n)


class FP8Linear(nn.Module):
    """nn.Linear whose weight is held in block-scaled FP8; inference only, like MixFP4Linear."""

    def __init__(self, weight: FP8Weight, bias: torch.Tensor | None = None):
        super().__init__()
        self.in_features, self.out_features = weight.k, weight.n
        self._weight = None
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone(), requires_grad=False)

    def _apply(self, fn, recurse=True):
        """Moves between devices; a change of type (`model.half()`) reaches the bias alone: codes and scales are the format's."""
        held = self.weight_fp8
        super()._apply(fn, recurse)
        moved = held if self.codes.device == held.device else held.to(self.codes.device)
        self.codes, self.scales = moved.codes, moved.scales
        return self

    @property
    def weight_fp8(self) -> FP8Weight:
        """The layer's buffers as a weight; checked again when they are others (`load_state_dict(assign=True)`)."""
        held, now = self._weight, self._buffers
        if held is None or held.codes is not now["codes"] or held.scales is not now["scales"]:
            held = self._weight = FP8Weight.from_tensors(now["codes"], now["scales"])
            self.codes, self.scales = held.codes, held.scales
        return held

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear, *, device=None) -> "FP8Linear":
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        w = linear.weight.detach().to(device)
        bias = None if linear.bias is None else linear.bias.detach().to(device)
        return cls(quantize_fp8_weight(w if w.dtype in nat.DTYPE_CODE else w.to(torch.bfloat16)), bias)

    def forward(self, x: torch.Tensor | FP8Activations, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        return fp8_linear(x, self.weight_fp8, bias=self.bias, out_dtype=out_dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"
