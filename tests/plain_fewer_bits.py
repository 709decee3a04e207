"""Plain statements of serving in fewer bits, in 64 bits: rows in 8-bit integers, the cache in 4 bits, attention over it; and steps to run them on."""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

F64 = torch.float64
TINY = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def to_bf16(x: torch.Tensor) -> torch.Tensor:
    """float64 to the nearest bfloat16 in one rounding, ties to even, as float64."""
    m, e = torch.frexp(x)
    return torch.where(torch.isfinite(x), torch.ldexp(torch.round(m * 256.0), e - 8), x)


def rows_i8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(integers, scales) as float64 and float32."""
    x = x.double()
    top = x.abs().amax(1)
    scale = (top / torch.full_like(top, 127.0)).float()
    scale = torch.where(scale < 2.0 ** -120, torch.zeros_like(scale), scale)
    bad = ~torch.isfinite(x).all(1)
    scale[bad] = math.nan
    q = torch.round(x / scale.double()[:, None])
    q[bad | (scale == 0)] = 0
    return q, scale


def held4(x: torch.Tensor) -> torch.Tensor:
    """What 4 bits make of finite x [..., D] (float64)."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    spread = (hi - lo) * 16.0 / 15.0
    S = torch.where(spread < 2.0 ** -100, torch.zeros_like(spread), to_bf16(spread))
    B = to_bf16(lo - S)
    code = torch.where(S > 0, torch.round(16.0 * (g - B) / S - 16.0).clamp(0, 15), torch.zeros_like(g))
    return to_bf16(B + S * (1.0 + code / 16.0)).reshape(x.shape)


def rotated(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor | None) -> torch.Tensor:
    """x [N, heads, D] in float64; pairs (j, j + D / 2)."""
    x = x.double()
    if inv_freq is None:
        return x
    half, n = x.shape[-1] // 2, inv_freq.numel()
    a = positions.double()[:, None, None] * inv_freq.double()
    y = x.clone()
    y[..., :n] = x[..., :n] * torch.cos(a) - x[..., half: half + n] * torch.sin(a)
    y[..., half: half + n] = x[..., half: half + n] * torch.cos(a) + x[..., :n] * torch.sin(a)
    return y


def in_type(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return to_bf16(x) if dtype == torch.bfloat16 else x.float().double()


def step(lens: list[tuple[int, int]], page: int, nkv: int, dim: int, dtype=torch.bfloat16, nq: int = 1, seed: int = 0, padding: int = 0, device="cuda"):
    """(context, lane, qkv) of a step: lens are (positions held before, tokens brought); `padding` rows behind the last request."""
    from nanospec_b200 import ops

    g = torch.Generator().manual_seed(seed)
    blocks = [-(-(a + n) // page) for a, n in lens]
    order = (torch.randperm(sum(blocks), generator=g) + 1).int()
    table = torch.full((len(lens), max(blocks) + 1), -1, dtype=torch.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at: at + b]
        at += b
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    q_lens, kv_lens = [n for _, n in lens], [a + n for a, n in lens]
    ctx = SimpleNamespace(
        n_tokens=sum(q_lens) + padding, n_requests=len(lens), q_lens=q_lens, kv_lens=kv_lens, max_q_len=max(q_lens), max_kv_len=max(kv_lens),
        positions=i32([p for a, n in lens for p in range(a, a + n)] + [0] * padding),
        token_req=i32([i for i, (_, n) in enumerate(lens) for _ in range(n)] + [-1] * padding),
        qo_indptr=i32([sum(q_lens[:i]) for i in range(len(lens) + 1)]), kv_len=i32(kv_lens), device=torch.device(device), extras={})
    lane = SimpleNamespace(k=ops.kv4_pages(sum(blocks) + 1, nkv, page, dim, device), v=ops.kv4_pages(sum(blocks) + 1, nkv, page, dim, device),
                           block_table=table.to(device), page_size=page, window=0, state=None)
    qkv = torch.randn((ctx.n_tokens, (nq + 2 * nkv) * dim), generator=g).to(dtype).to(device)
    return ctx, lane, qkv


def everything(ctx):
    """The same requests with all of their positions as the step's tokens."""
    out = SimpleNamespace(**vars(ctx))
    out.q_lens = list(ctx.kv_lens)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=ctx.device)  # noqa: E731
    out.positions = i32([p for n in ctx.kv_lens for p in range(n)])
    out.token_req = i32([i for i, n in enumerate(ctx.kv_lens) for _ in range(n)])
    out.n_tokens, out.extras = sum(ctx.kv_lens), {}
    return out


def fill(ctx, lane, nq: int, nkv: int, dim: int, dtype=torch.bfloat16, seed: int = 1, size: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Stores random keys and values at every position of every request; returns what the cache holds, float64 [positions, nkv, D] request after request."""
    from nanospec_b200 import ops

    whole = everything(ctx)
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((whole.n_tokens, (nq + 2 * nkv) * dim), generator=g) * size).to(dtype).to(ctx.device)
    ops.kv4_store(qkv, whole, lane, nq, nkv, dim)
    k, v = ops.kv4_read(lane, whole.positions, whole.token_req, nkv, dim)
    return k.double(), v.double()


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ctx, nq: int, scale: float, window: int = 0, sink=None):
    """(output [N, nq, D], tolerances of it for weights held in 8 bits and in float) of the step's tokens.  k, v [positions, nkv, D], request after request.

    The tolerances: a score is off by (D + 8) half steps of float32 of the sum of its terms' magnitudes, which moves a weight by as much, relatively; a
    weight rounded to bfloat16 by 2^-8 of itself; the sums over n keys by n half steps; the exponential by 2^-20.  Each counts on the sum of |weight * value|.
    And a weight below 2^-126, the smallest normal float, may become zero (the largest is 1 or, before it is divided, more): each such key is off by
    2^-126 |value| at most, and an output below 2^-126 by that."""
    N, D = q.shape[0], k.shape[2]
    q = q.double().reshape(N, nq, D)
    G = nq // k.shape[1]
    out = torch.zeros((N, nq, D), dtype=F64, device=q.device)
    tol8, tol32 = torch.zeros_like(out), torch.zeros_like(out)
    row = at = 0
    for n, kv in zip(ctx.q_lens, ctx.kv_lens):
        key, pos = torch.arange(kv, device=q.device), torch.arange(kv - n, kv, device=q.device)[:, None]
        hidden = (key > pos) | ((pos - key >= window) if window else (key < 0))
        for h in range(nq):
            kk, vv = k[at: at + kv, h // G], v[at: at + kv, h // G]
            s = (q[row: row + n, h] @ kk.T * scale).masked_fill(hidden, -math.inf)
            off = ((q[row: row + n, h].abs() @ kk.abs().T) * abs(scale)).masked_fill(hidden, 0.0).amax(1, keepdim=True) * (D + 8) * TINY
            top = s.amax(1, keepdim=True)
            if sink is not None:
                top = torch.maximum(top, sink[h].double())
            e = torch.exp(s - top)
            total = e.sum(1, keepdim=True) + (torch.exp(sink[h].double() - top) if sink is not None else 0.0)
            w = e / total
            out[row: row + n, h] = w @ vv
            mass = w @ vv.abs()
            tol32[row: row + n, h] = mass * (4 * off + (kv + 16) * TINY + 2.0 ** -20) + (vv.abs().sum(0) + 1) * 2.0 ** -126
            tol8[row: row + n, h] = tol32[row: row + n, h] + mass * 2.0 ** -8
        row += n
        at += kv
    return out, tol8, tol32
