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
    """A matrix in 8-bit integers from -127 to 127 (not -128, with which the sum over the largest K could leave 32 bits): `q` [R, K] int8 (rows on 16-byte boundaries) and `scale` [R] float32; row r stands for q[r] * scale[r]."""

    q: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    def values(self) -> torch.Tensor:
        """float32, for inspection."""
        return self.q.float() * self.scale[:, None]


def _check_rows(r: RowsI8, name: str) -> int:
    """Elements from one row to the next."""
    q, scale = r.q, r.scale
    shape = q.shape
    if q.dtype is not torch.int8 or len(shape) != 2 or scale.dtype is not torch.float32 or scale.shape != shape[:1] or not scale.is_contiguous():
        raise KernelError(f"linear_i8: {name} must be int8 [R, K] with one contiguous float32 scale per row")
    step, inner = q.stride()
    if shape[0] and (inner != 1 or step & 15 or not step or q.data_ptr() & 15):
        raise KernelError(f"linear_i8: the rows of {name} must start on 16-byte boundaries with unit inner stride (quantize_rows makes them so)")
    return step


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


# us that a pair of SMs takes for 128 of k of a tile of 256 tokens x so many features
I8_WIDE_US = {64: 0.172, 128: 0.209, 192: 0.256, 256: 0.336}


@functools.lru_cache(maxsize=4096)
def i8_tiles(M: int, N: int, K: int, sms: int) -> tuple[int, int, int]:
    """(tokens of a tile, features of a tile, blocks or pairs that divide k) of the product.

    Up to 64 tokens, and up to 128 while the tiles of 128 features fit the SMs: one tile of tokens, k divided over up to eight blocks until every SM
    has one, and beyond that while a block keeps eight of its 128-wide pieces (us on a B200, 32 x 4096 x 4096, one, two, four and eight blocks: 16.4, 14.3, 12.3,
    14.3; 8 x 14336 x 4096: 32.8, 24.6, 22.5, 20.5; 77 x 2051 x 1003: eight 10.2, four 12.3; 128 x 4096 x 28672: 53 so, 43 in wide tiles).
    More tokens: the wide tiles of least cost, `I8_WIDE_US` for every piece of k and round over the pairs of SMs; two pairs to a tile only while all
    clusters of four blocks run at once (32 of them), for about 4 us (512 x 14336 x 4096: 256 features and two pairs 36.9, one 49.2; 200 x 4096 x 4096: 64
    features 16.4, 256 20.5; four pairs took 47 where two took 31: clusters of eight such blocks do not all find a place)."""
    k_blocks, tiles = -(-K // 128), -(-N // 128)
    if M <= 64 or (M <= 128 and tiles <= sms):
        tile = 16 if M <= 16 else 32 if M <= 32 else 64 if M <= 64 else 128
        resident, splits = sms * (2 if tile <= 64 else 1), 1
        while splits < 8 and splits * 2 <= k_blocks and (tiles * splits * 2 <= sms or (tiles * splits * 2 <= resident and k_blocks >= 16 * splits)):
            splits *= 2
        return tile, 128, splits
    best = None
    for features, us in I8_WIDE_US.items():
        tiles = -(-M // 256) * -(-N // features)
        for splits in (1, 2):
            if splits > 1 and (tiles > 32 or k_blocks < 16):
                continue
            cost = -(-tiles // (sms // 2)) * -(-k_blocks // splits) * us + (4 if splits > 1 else 0)
            if best is None or cost < best[0]:
                best = (cost, features, splits)
    return 256, *best[1:]


def linear_i8(x: torch.Tensor | RowsI8, w: RowsI8, out: torch.Tensor, bias: torch.Tensor | None = None,
              tiles: tuple[int, int, int] | None = None) -> torch.Tensor:
    """out[n, f] = (sum_k xq[n, k] wq[f, k]) * xs[n] * ws[f] (+ bias[f], float32), the sum exact in 32-bit integers.  `x` [N, K] is quantised by
    rows on the way (`quantize_rows`) unless it comes so, for several products of the same activations; `out` [N, F] is float32 or bfloat16
    with unit inner stride.  `tiles` (tokens and features of a tile, blocks or pairs that divide k): `i8_tiles`' choice when None; an output's
    bits are the same in all of them."""
    ready = isinstance(x, RowsI8)
    held, wq, ws = x.q if ready else x, w.q, w.scale
    if ready:
        _on_current_device(held, x.scale, wq, ws, out, bias)
        ldx = _check_rows(x, "x")
    else:
        _on_current_device(held, wq, ws, out, bias)
        ldx = 0
    ldw = _check_rows(w, "w")
    F, K = wq.shape
    shape, steps, ldo = held.shape, held.stride(), out.stride()
    if len(shape) != 2 or shape[1] != K or not 1 <= K <= I8_MAX_K or (steps[1] != 1 and shape[0]):
        raise KernelError(f"linear_i8: x {tuple(shape)} with unit inner stride and w {tuple(wq.shape)} must agree on K, which is {I8_MAX_K} at most")
    N = shape[0]
    if out.shape != (N, F) or (ldo[1] != 1 and N and F):
        raise KernelError(f"linear_i8: out must be [{N}, {F}] with unit inner stride, not {tuple(out.shape)} with strides {ldo}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (F,) or not bias.is_contiguous()):
        raise KernelError("linear_i8: the bias is one contiguous float32 number per output feature")
    code, sms, dev = dtype_code(out.dtype), sm_count(), out.device
    tile, features, splits = tiles or i8_tiles(N, F, K, sms)
    if ready:
        lib.call("ns_gemm_i8", held.data_ptr(), ldx, x.scale.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), _ptr(bias), out.data_ptr(), ldo[0], N, F, K,
                 code, tile, features, splits, 0, sms, _tc(dev).error.data_ptr(), _stream())
    else:
        scratch = torch.empty(N * (((K + 15) & -16) + 4), dtype=torch.int8, device=dev)
        lib.call("ns_linear_i8", held.data_ptr(), steps[0], dtype_code(held.dtype), scratch.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), _ptr(bias),
                 out.data_ptr(), ldo[0], N, F, K, code, tile, features, splits, sms, _tc(dev).error.data_ptr(), _stream())
    return out
