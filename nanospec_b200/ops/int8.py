"""Products in 8-bit integers: rows quantised with a float32 scale each (tokens of activations, output channels of weights) and
their matrix product with an exact integer sum (csrc/quantize_rows.cu, csrc/gemm_i8.cu)."""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _on_current_device, _ptr, _stream, _tc, dtype_code, lib, sm_count
from .lib import KernelError

I8_MAX_K = 131072  # 127 * 127 * K stays within 32 bits


@dataclass
class RowsI8:
    """A matrix in 8-bit integers: `q` [R, K] int8 (rows on 16-byte boundaries) and `scale` [R] float32; row r stands for q[r] * scale[r]."""

    q: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    def values(self) -> torch.Tensor:
        """float32, for inspection."""
        return self.q.float() * self.scale[:, None]


def _aligned_rows(q: torch.Tensor) -> bool:
    return q.stride(1) == 1 and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


def _check_rows(r: RowsI8, name: str) -> None:
    q, scale = r.q, r.scale
    if q.dtype != torch.int8 or q.dim() != 2 or scale.dtype != torch.float32 or scale.shape != q.shape[:1] or not scale.is_contiguous():
        raise KernelError(f"linear_i8: {name} must be int8 [R, K] with one contiguous float32 scale per row")
    if q.shape[0] and not _aligned_rows(q):
        raise KernelError(f"linear_i8: the rows of {name} must start on 16-byte boundaries with unit inner stride (quantize_rows makes them so)")


def quantize_rows(x: torch.Tensor) -> RowsI8:
    """x [R, K] (float32 or bfloat16, unit inner stride) in 8-bit integers: scale[r] = float32(max |x[r]| / 127) and q[r] the integers
    nearest to x[r] / scale[r] (ties to even).  A row that holds an infinity or a NaN gets NaN for its scale and zeros; a row whose scale
    would be below 2^-120 gets 0 and zeros.  Weights go through it once, an output channel a row; `linear_i8` takes activations as they are
    or quantised."""
    _on_current_device(x)
    if x.dim() != 2 or x.stride(1) != 1 or not 1 <= x.shape[1] <= I8_MAX_K:
        raise KernelError(f"quantize_rows: a matrix with unit inner stride and 1 to {I8_MAX_K} columns is needed, not {tuple(x.shape)} with strides {x.stride()}")
    rows, K = x.shape
    code = dtype_code(x.dtype)
    q = torch.empty((rows, -(-K // 16) * 16), dtype=torch.int8, device=x.device)[:, :K]
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    lib.call("ns_quantize_rows", x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(), rows, K, code, _stream())
    return RowsI8(q, scale)


@functools.lru_cache(maxsize=4096)
def i8_tiles(M: int, N: int, K: int, sms: int) -> tuple[int, int, int]:
    """(tokens of a tile, features of a tile, blocks or pairs that divide k) of the product."""
    k_blocks = -(-K // 128)
    if M > 128:
        tiles = -(-M // 256) * -(-N // 256)
        splits = 1
        while splits < 4 and tiles * splits * 2 <= sms // 2 and splits * 2 <= k_blocks:
            splits *= 2
        return 256, 256, splits
    tile = 16 if M <= 16 else 32 if M <= 32 else 64 if M <= 64 else 128
    tiles = -(-N // 128)
    resident = sms * (2 if tile <= 64 else 1)
    splits = 1
    while splits < 8 and tiles * splits * 2 <= resident and splits * 2 <= k_blocks:
        splits *= 2
    return tile, 128, splits


def linear_i8(x: torch.Tensor | RowsI8, w: RowsI8, out: torch.Tensor, bias: torch.Tensor | None = None,
              tiles: tuple[int, int, int] | None = None) -> torch.Tensor:
    """out[n, f] = (sum_k xq[n, k] wq[f, k]) * xs[n] * ws[f] (+ bias[f], float32), the sum exact in 32-bit integers.  `x` [N, K] is quantised by
    rows on the way (`quantize_rows`) unless it comes so, for several products of the same activations; `out` [N, F] is float32 or bfloat16
    with unit inner stride."""
    ready = isinstance(x, RowsI8)
    held, wq = x.q if ready else x, w.q
    _on_current_device(held, wq, w.scale, out, bias, x.scale if ready else None)
    _check_rows(w, "w")
    if ready:
        _check_rows(x, "x")
    N, (F, K) = held.shape[0], wq.shape
    if held.dim() != 2 or held.shape[1] != K or not 1 <= K <= I8_MAX_K or (N and held.stride(1) != 1):
        raise KernelError(f"linear_i8: x {tuple(held.shape)} with unit inner stride and w {tuple(wq.shape)} must agree on K, which is {I8_MAX_K} at most")
    if out.shape != (N, F) or (N and F and out.stride(1) != 1):
        raise KernelError(f"linear_i8: out must be [{N}, {F}] with unit inner stride, not {tuple(out.shape)} with strides {out.stride()}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (F,) or not bias.is_contiguous()):
        raise KernelError("linear_i8: the bias is one contiguous float32 number per output feature")
    code, sms = dtype_code(out.dtype), sm_count()
    tiles = tiles or i8_tiles(N, F, K, sms)
    if ready:
        lib.call("ns_gemm_i8", held.data_ptr(), held.stride(0), x.scale.data_ptr(), wq.data_ptr(), wq.stride(0), w.scale.data_ptr(), _ptr(bias),
                 out.data_ptr(), out.stride(0), N, F, K, code, *tiles, 0, sms, _tc(out.device).error.data_ptr(), _stream())
    else:
        scratch = torch.empty(N * (-(-K // 16) * 16 + 4), dtype=torch.int8, device=out.device)
        lib.call("ns_linear_i8", held.data_ptr(), held.stride(0), dtype_code(held.dtype), scratch.data_ptr(), wq.data_ptr(), wq.stride(0),
                 w.scale.data_ptr(), _ptr(bias), out.data_ptr(), out.stride(0), N, F, K, code, *tiles, sms, _tc(out.device).error.data_ptr(), _stream())
    return out
