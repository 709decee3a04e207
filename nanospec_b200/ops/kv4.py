"""A paged cache of keys and values in 4 bits: the store (with the rotation), reading back, and attention over it.  A lane's `k` and `v`
are then uint8 [pages, kv heads, page_size * head_dim * 5 / 8] (`kv4_pages`); csrc/kv4.cuh says what the bytes are and stand for."""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch

from . import BF16, TILE_Q, TILE_Q_TCGEN05, _i32, _on_current_device, _ptr, _stream, attention_prefill, dtype_code, lib, sm_count
from .lib import KernelError

KV4_GROUP = 32  # features that share a pair of numbers
KV4_MAX_HEAD = 256


@functools.lru_cache(maxsize=256)
def kv4_block_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of a page of one kv head (of keys, and as many of values): half a byte a feature and 4 bytes a group of 32."""
    if head_dim % KV4_GROUP or not KV4_GROUP <= head_dim <= KV4_MAX_HEAD or page_size < 1:
        raise KernelError(f"a 4-bit cache takes heads in multiples of {KV4_GROUP} up to {KV4_MAX_HEAD} and pages of one token at least, not {head_dim} and {page_size}")
    return page_size * head_dim * 5 // 8


def kv4_pages(pages: int, kv_heads: int, page_size: int, head_dim: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """Pages of keys, or of values, of a lane: every feature zero."""
    return torch.zeros((pages, kv_heads, kv4_block_bytes(page_size, head_dim)), dtype=torch.uint8, device=device)


def _check_lane(who: str, lane, nkv: int, head_dim: int) -> None:
    k, v, table = lane.k, lane.v, lane.block_table
    size = kv4_block_bytes(lane.page_size, head_dim)
    if k is None or v is None or k.dtype is not torch.uint8 or v.dtype is not torch.uint8 or k.shape != v.shape or k.shape[1:] != (nkv, size) \
            or not k.is_contiguous() or not v.is_contiguous() or (k.data_ptr() | v.data_ptr()) & 15:
        raise KernelError(f"{who}: the lane's pages must be contiguous uint8 [pages, {nkv}, {size}] on 16-byte boundaries (kv4_pages makes them)")
    if table is None or table.dtype is not torch.int32 or table.dim() != 2 or table.stride()[1] != 1:
        raise KernelError(f"{who}: block_table must be int32 [requests, pages] with unit inner stride")


def _check_step(who: str, positions: torch.Tensor, token_req: torch.Tensor, n: int) -> None:
    _i32(positions, "positions"), _i32(token_req, "token_req")
    if positions.numel() != n or token_req.numel() != n:
        raise KernelError(f"{who}: one position and one request per token ({n})")


def kv4_store(qkv: torch.Tensor, ctx, lane, nq: int, nkv: int, head_dim: int, inv_freq: torch.Tensor | None = None,
              q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotates q and k of the packed [q | k | v] rows (pairs j and j + head_dim / 2 by position * inv_freq[j]; None: as they are), writes k
    and v in 4 bits at each token's position, and q to `q_out` ([N, nq * head_dim]; None: in place).  The rotated k is rounded to the
    activations' type before it is quantised, as a cache in that type would hold it.  Rows of padding (token_req < 0) are left as they
    are; no two rows of a step have the same position of the same request.  Returns where q went."""
    _on_current_device(qkv, ctx.positions, ctx.token_req, lane.block_table, lane.k, lane.v, inv_freq, q_out)
    _check_lane("kv4_store", lane, nkv, head_dim)
    code, size = dtype_code(qkv.dtype), qkv.element_size()
    n = qkv.shape[0]
    _check_step("kv4_store", ctx.positions, ctx.token_req, n)
    if qkv.dim() != 2 or qkv.shape[1] != (nq + 2 * nkv) * head_dim or nq < 1:
        raise KernelError(f"kv4_store: qkv must be [N, {(nq + 2 * nkv) * head_dim}], not {tuple(qkv.shape)}")
    target = qkv if q_out is None else q_out
    if q_out is not None and (q_out.dtype != qkv.dtype or q_out.shape != (n, nq * head_dim)):
        raise KernelError("kv4_store: q_out must be [N, nq * head_dim] in the type of qkv")
    (ld, inner), (ldq, inner_q) = qkv.stride(), target.stride()
    if n and (inner != 1 or inner_q != 1 or (ld | ldq) * size % 16 or (qkv.data_ptr() | target.data_ptr()) % 16):
        raise KernelError("kv4_store: rows must start on 16-byte boundaries with unit inner stride")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous() or inv_freq.numel() > head_dim // 2):
        raise KernelError(f"kv4_store: inv_freq must be contiguous float32, at most {head_dim // 2} numbers")
    lib.call("ns_kv4_store", qkv.data_ptr(), ld, target.data_ptr(), ldq, ctx.positions.data_ptr(), ctx.token_req.data_ptr(),
             lane.block_table.data_ptr(), lane.block_table.stride(0), _ptr(inv_freq), 0 if inv_freq is None else inv_freq.numel(), lane.k.data_ptr(),
             lane.v.data_ptr(), lane.page_size, nq, nkv, head_dim, n, sm_count(), code, _stream())
    return target


def kv4_read(lane, positions: torch.Tensor, token_req: torch.Tensor, nkv: int, head_dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds at positions[n] of request token_req[n]: keys and values [N, nkv, head_dim] in bfloat16, as `attention_kv4` sees them
    (zeros where token_req is negative, and where the block table has no page for the position, as behind a window)."""
    _on_current_device(lane.k, lane.v, lane.block_table, positions, token_req)
    _check_lane("kv4_read", lane, nkv, head_dim)
    n = positions.numel()
    _check_step("kv4_read", positions, token_req, n)
    k, v = torch.empty((2, n, nkv, head_dim), dtype=torch.bfloat16, device=lane.k.device).unbind(0)
    lib.call("ns_kv4_read", lane.k.data_ptr(), lane.v.data_ptr(), positions.data_ptr(), token_req.data_ptr(), lane.block_table.data_ptr(),
             lane.block_table.stride(0), *lane.block_table.shape, lane.k.shape[0], k.data_ptr(), v.data_ptr(), n, lane.page_size, nkv, head_dim, sm_count(),
             _stream())
    return k, v


KV4_TILE = 32  # keys that a warp of csrc/attention_kv4_tc.cu takes at a time


def kv4_tensor_core_ok(dtype: torch.dtype, head_dim: int, page_size: int) -> bool:
    return dtype == torch.bfloat16 and head_dim in (64, 128, 256) and (page_size in (8, 16) or page_size % 32 == 0)


KV4_PARTS_MAX = 256  # blocks of a row and kv head


def kv4_shape(lengths: tuple[int, ...] | None, rows: int, per_row: int, sms: int, head_dim: int, n_blocks: int = 1, window: int = 0) -> tuple[int, int, int]:
    """(warps of a block, blocks of a row's kv head, tiles of 32 keys that such a block takes at least, or 0: one block, which needs no joining).

    `lengths`: keys of each row (or tile of tokens), None when the device alone knows them, at most `window` where there is one; `per_row`: (kv head, column tile) pairs.  Us on a B200, the requests
    ragged down to a fifth of the length, 8 kv heads of 128:
    Several blocks while one each would take no more than half of the places, or while one request would outlast the others.  One request on 1,000 keys: one block of
    eight warps 14.4, several 12.3; on 100,000: a cluster of sixteen blocks 71.7, several 46.6; 16 requests on 1,000: 16.4, 18.4; on 4,000: 34.8, 30.7; one on 100,000
    among 63 on 500: 580, 63.  The two costs below are fits to such figures.
    Blocks of eight warps rather than four while places are left, or while the longest row would outlast the others: 48 requests on 3,000 keys 43.0, 49.2; 96 on
    8,000 143, 154; 64 on 500 22.5, 20.5; 200 on 2,300 107, 96."""
    slots = sms * (2 if head_dim > 128 else 3 if n_blocks > 1 else 6 if head_dim == 64 else 4)  # blocks of four warps that the SMs hold
    total = rows * per_row
    if lengths is None:
        # The window's keys stand for the lengths only while a block then has no more than eight tiles: a window beyond all contexts would leave them few blocks (one request
        # on 5,000 keys, a window of 131,072: 3 of 74, 28.7 us, now 18.4; 8 on 30,000: 305, now 90; 8 on 2,000, a window of 32,768: 36.9, now 24.6).
        full = kv4_shape((window,) * rows, rows, per_row, sms, head_dim, n_blocks) if window else None
        if full and full[2] <= 8:
            return full
        return (4, min(KV4_PARTS_MAX, slots // total), 8) if total * 2 <= slots else (8 if total <= 2 * sms else 4, 1, 0)
    tiles = [-(-n // KV4_TILE) for n in lengths]
    longest, all_tiles = max(tiles), sum(tiles)
    rate = 0.75 * slots / sms * head_dim / 512                            # us a tile of each block while all places are taken
    chain = 0.18 * head_dim / 128 * (1.5 if n_blocks > 1 else 1)          # us a tile of a block of eight warps, one an SM
    if longest > 4 and (total * 2 <= slots or longest * chain > 2 * (10 + all_tiles * per_row / slots * rate)):
        room = max(slots // per_row, 2 * rows)  # blocks of a kv head of all rows
        least = max(4, -(-all_tiles // room), -(-longest // KV4_PARTS_MAX))
        while (blocks := sum(-(-t // least) for t in tiles)) > room:
            least += 1 + least // 16
        splits, wave = -(-longest // least), blocks * per_row / slots
        if splits > 1 and 12 + 2 * wave + least * max(0.33, wave) * rate < 9 + longest * chain * (1 if total <= sms else 1.5):
            return 4, splits, least
    return 8 if total <= 2 * sms or total * 32 <= sms * longest else 4, 1, 0


def kv4_jobs(rows: list[tuple[int, int]], lengths: tuple[int, ...], least: int) -> list[int]:
    """(first row, tokens, part, parts) of every block's share of the tiles of (first row, tokens), then (first of them, parts) of each."""
    jobs, spans = [], []
    for (row, tokens), n in zip(rows, lengths):
        parts = max(1, -(-n // (KV4_TILE * least)))
        spans += (len(jobs) // 4, parts)
        for p in range(parts):
            jobs += (row, tokens, p, parts)
    return jobs + spans


def kv4_token_tiles(requests: list[tuple[int, int, int]], group: int) -> tuple[list[tuple[int, int]], int]:
    """(first row, tokens) of the tiles of requests of (first row, tokens, ...), in their order, and the n-blocks of 8 columns that the tiles need: a column
    is a (query head, token) pair, 16 at most to a tile."""
    blocks = 1 if max(n for _, n, *_ in requests) * group <= 8 else 2
    per = max(1, 8 * blocks // group)
    return [(row + at, min(per, n - at)) for row, n, *_ in requests for at in range(0, n, per)], blocks


KV4_UNFOLD_MAX = 1 << 30      # bytes of keys and values in bfloat16 at a time: more requests, or kv heads, go one after another
KV4_UNFOLD_PAGE = 64          # tokens of a page of theirs


def kv4_unfolded(requests: list[tuple[int, int]], group: int, nkv: int, head_dim: int, window: int, sms: int, tensor_core: bool) -> list[int]:
    """Which of the requests of (tokens brought, positions held after the step) meet their keys and values in bfloat16, unfolded once for all of the portion's
    tokens.  From the bytes the keys are unpacked again for every 16 (query head, token) pairs: about 17,000 keys of a head of 128 a us; unfolded they cost 3.3
    MB a us, and a block of 256 tokens of a head takes 11 ns a key, one block an SM.  Us on a B200, from the bytes / unfolded, heads of 128, 4 to each of
    8 kv heads: one request on 30,000 positions, 64 tokens 202 / 328, 96 378 / 330; 8 on 3,000, 24 tokens 74 / 104, 48 137 / 104; 32 on 1,000, 32
    tokens 141 / 152, 48 203 / 154; 8 on 500, 24 tokens 27 / 34, 48 45 / 35.  Without the tensor cores a token goes by itself, 3,000 keys a us."""
    scale = head_dim / 128
    cost = []  # (request, from the bytes, unfolding and blocks together, one block)
    for i, (n, kv) in enumerate(requests):
        if n < 2:
            continue
        seen = min(kv, window + n) if window else kv
        packed = -(-n * group // 16) * seen * nkv * scale / 17000 if tensor_core else n * -(-group // 8) * seen * nkv * scale / 3000
        cost.append((i, packed, seen * nkv * head_dim * 4 / 3.3e6 + nkv * group * -(-n // 256) * seen * 0.011 / sms, seen * 0.011))
    chosen = [c for c in cost if c[1] > c[2]]
    if not chosen or sum(c[1] for c in chosen) < 10 + max(sum(c[2] for c in chosen), max(c[3] for c in chosen)):
        return []
    return [c[0] for c in chosen]


def kv4_unfold_runs(chunks: list[int], nkv: int, head_dim: int, limit: int) -> list[tuple[int, int, int, int]]:
    """(first request, requests, first kv head, kv heads) of the runs that keep `chunks` of 64 positions a request within `limit` bytes: whole
    requests together while they fit, one request's heads in parts where they do not."""
    one = KV4_UNFOLD_PAGE * head_dim * 4  # of a kv head
    runs, first, held = [], 0, 0
    for i, n in enumerate(chunks):
        if held and (held + n) * nkv * one > limit:
            runs.append((first, i - first, 0, nkv))
            first, held = i, 0
        if n * nkv * one > limit:
            heads = max(1, min(nkv, limit // (n * one)))
            runs += [(i, 1, h, min(heads, nkv - h)) for h in range(0, nkv, heads)]
            first, held = i + 1, 0
        else:
            held += n
    if held:
        runs.append((first, len(chunks) - first, 0, nkv))
    return runs


def _check_table(lane, held: int, requests: int) -> None:
    rows, columns = lane.block_table.shape
    if held > columns * lane.page_size or requests > rows:
        raise KernelError(f"attention_kv4: {requests} requests of up to {held} positions, the block table has {rows} rows of {columns} pages of {lane.page_size}")


def _kv4_plan(ctx, lane, group: int, nkv: int, head_dim: int, window: int, tensor_core: bool, unfold: bool) -> dict:
    """Once per step and kind of layer: which rows run by themselves, the tiles of a few tokens, and the portions that are unfolded.  `tensor_core`: rows and
    tiles are those of csrc/attention_kv4_tc.cu; else rows alone, of csrc/attention_kv4.cu."""
    key = ("kv4_plan", group, nkv, head_dim, window, tensor_core, unfold)
    plan = ctx.extras.get(key)
    if plan is not None:
        return plan
    total = ctx.positions.numel()
    made = []

    def on_device(v):
        if not v:
            return None
        if torch.cuda.is_current_stream_capturing():
            raise KernelError("attention_kv4: a step's lists cannot go to the device while a graph is captured; ctx.extras['graph'] says that every row is a "
                              "request's one token, which needs none, and another step has a call before the capture")
        made.append(torch.tensor(v, dtype=torch.int32).to(ctx.device, non_blocking=True))
        return made[-1]

    if ctx.extras.get("graph"):  # every row is a request's one token, and lengths are the device's
        plan = {"rows": None, "n_rows": total, "longest": None, "held": 0, "requests": 0, "portions": [],
                "runs": [_kv4_run(None, None, total, None, nkv, group, head_dim, 1 if group <= 8 else 2, window=window)] if tensor_core and total else []}
    else:
        if sum(ctx.q_lens) > total:
            raise KernelError(f"attention_kv4: the requests bring {sum(ctx.q_lens)} tokens, the step holds {total}")
        held = max(ctx.kv_lens, default=0)
        _check_table(lane, held, len(ctx.kv_lens))
        starts, row = [], 0
        for n in ctx.q_lens:
            starts.append(row)
            row += n
        requests = list(zip(starts, ctx.q_lens, ctx.kv_lens))
        long = kv4_unfolded(list(zip(ctx.q_lens, ctx.kv_lens)), group, nkv, head_dim, window, sm_count(), tensor_core) if unfold else []
        if long:
            for name, t, least in (("kv_len", ctx.kv_len, len(requests)), ("qo_indptr", ctx.qo_indptr, len(requests) + 1)):
                _i32(t, name)
                if t.numel() < least:
                    raise KernelError(f"attention_kv4: {name} holds {t.numel()} numbers for {len(requests)} requests")
            _on_current_device(ctx.kv_len, ctx.qo_indptr)
        unfolded = set(long)
        rest = [(s, n, kv) for i, (s, n, kv) in enumerate(requests) if i not in unfolded]
        rest.sort(key=lambda r: -r[2])  # the longest first: blocks are scheduled in this order
        rows = [s + i for s, n, _ in rest for i in range(n) if n == 1 or not tensor_core]
        plan = {"rows": None if rows == list(range(total)) else on_device(rows), "n_rows": len(rows),
                "longest": max((kv for _, n, kv in rest if n == 1 or not tensor_core), default=0), "held": held,
                "requests": len(ctx.kv_lens), "portions": [], "runs": []}
        if tensor_core:
            seen = tuple(min(kv, window or kv) for _, n, kv in rest if n == 1)
            if rows:
                plan["runs"].append(_kv4_run(plan["rows"], None, len(rows), seen, nkv, group, head_dim, 1 if group <= 8 else 2, on_device, [(row, 1) for row in rows]))
            few = [r for r in rest if r[1] > 1]
            if few:
                tiles, n_blocks = kv4_token_tiles(few, group)
                keys = {row + i: min(kv, window + n) if window else kv for row, n, kv in few for i in range(n)}
                plan["runs"].append(_kv4_run(None, on_device(tiles), len(tiles), tuple(keys[row] for row, _ in tiles), nkv, group, head_dim, n_blocks, on_device, tiles))
        for first, count, head, heads in kv4_unfold_runs([-(-ctx.kv_lens[i] // KV4_UNFOLD_PAGE) - _first_chunk(ctx, i, window) for i in long], nkv, head_dim,
                                                         KV4_UNFOLD_MAX):
            plan["portions"].append(_kv4_portion(ctx, long[first: first + count], window, head, heads, on_device))
        if made:  # (a captured step has none)
            ready = torch.cuda.Event()
            ready.record()
            plan.update(lists=made, ready=ready, streams={_stream()})
    ctx.extras[key] = plan
    return plan


_captured_lists: list = []  # of steps that were captured without `ctx.extras["graph"]`: a graph reads them for as long as it lives


def _plan_on_this_stream(plan: dict, stream: int) -> None:
    """The plan's lists go to the device on the stream of the step's first call; a call on another one waits for them there.  One that is captured
    waits on the host, once (its graph then finds them in place wherever it is replayed), and the lists stay."""
    streams = plan.get("streams")
    if streams is None:
        return
    if torch.cuda.is_current_stream_capturing():
        if not plan.get("captured"):
            if lib.load().ns_event_synchronize(plan["ready"].cuda_event):
                raise KernelError(f"attention_kv4: waiting for the step's lists failed: {lib.load().ns_last_error().decode(errors='replace')}")
            _captured_lists.append(plan["lists"])
            plan["captured"] = True
        return
    if stream in streams:
        return
    here = torch.cuda.current_stream()
    here.wait_event(plan["ready"])
    lib.load().ns_full_launch_next()  # (it has a prerequisite beside its predecessor in the stream)
    for t in plan["lists"]:
        t.record_stream(here)
    streams.add(stream)


def _kv4_run(rows, items, count: int, lengths, nkv: int, group: int, head_dim: int, n_blocks: int, on_device=None, taken=None, window: int = 0) -> tuple:
    """What the launch for `count` rows, or tiles of tokens (`taken`: (first row, tokens) of them, where the host knows their `lengths`, which are within the window), is: (rows, items, how many,
    n-blocks of columns, shape, jobs, how many, floats of the workspace)."""
    per_row = nkv * -(-group // (8 * n_blocks))
    warps, splits, least = kv4_shape(lengths, count, per_row, sm_count(), head_dim, n_blocks, window)
    units, jobs = (count * splits, None) if least else (0, None)
    if least and on_device:
        listed = kv4_jobs(taken, lengths, least)
        units, jobs = (len(listed) - 2 * count) // 4, on_device(listed)
    return rows, items, count, n_blocks, (warps, splits, least), jobs, units if jobs is not None else 0, units * per_row * 8 * n_blocks * (head_dim + 2)


def _first_chunk(ctx, i: int, window: int) -> int:
    return max(0, ctx.kv_lens[i] - ctx.q_lens[i] - window + 1) // KV4_UNFOLD_PAGE if window else 0


def _kv4_portion(ctx, requests: list[int], window: int, head: int, heads: int, on_device) -> dict:
    """What the unfolding and the attention of `requests` need: chunks of 64 positions, a block table of theirs, tiles of queries."""
    items, table = [], [[0] * max(-(-ctx.kv_lens[i] // KV4_UNFOLD_PAGE) for i in requests) for _ in ctx.q_lens]
    for i in requests:
        for c in range(_first_chunk(ctx, i, window), -(-ctx.kv_lens[i] // KV4_UNFOLD_PAGE)):
            table[i][c] = len(items)
            items.append((i, c))

    def tiles(step):  # those that see the most keys come first: blocks are scheduled in this order
        found = [(i, at) for i in requests for at in range(0, ctx.q_lens[i], step)]
        found.sort(key=lambda t: -(ctx.kv_lens[t[0]] - ctx.q_lens[t[0]] + min(t[1] + step, ctx.q_lens[t[0]])))
        return on_device(found)

    return {"items": on_device(items), "n": len(items), "table": on_device(table), "tiles": tiles(TILE_Q), "tiles_tc": tiles(TILE_Q_TCGEN05), "head": head, "heads": heads}


@dataclass
class _Unfolded:
    """A lane in bfloat16 that holds what a step's portions see of one in 4 bits."""

    k: torch.Tensor
    v: torch.Tensor
    block_table: torch.Tensor
    page_size: int = KV4_UNFOLD_PAGE


def _attend_unfolded(qkv, lane, ctx, out, nkv: int, group: int, head_dim: int, scale: float, window: int, sink, portion: dict, wide_weights: bool) -> None:
    head, heads, n = portion["head"], portion["heads"], portion["n"]
    k, v = torch.empty((2, n, heads, KV4_UNFOLD_PAGE, head_dim), dtype=torch.bfloat16, device=out.device).unbind(0)
    lib.call("ns_kv4_unfold", lane.k.data_ptr(), lane.v.data_ptr(), lane.block_table.data_ptr(), lane.block_table.stride(0), portion["items"].data_ptr(), n,
             ctx.kv_len.data_ptr(), k.data_ptr(), v.data_ptr(), lane.page_size, nkv, head, heads, head_dim, _stream())
    at, width = head * group * head_dim, heads * group * head_dim
    attention_prefill(qkv[:, at: at + width], _Unfolded(k, v, portion["table"]), ctx, out[:, at: at + width], heads * group, heads, head_dim, scale, window,
                      portion["tiles"], portion["tiles_tc"], wide_weights=wide_weights, sink=None if sink is None else sink[head * group: (head + heads) * group])


def attention_kv4(qkv: torch.Tensor, lane, ctx, out: torch.Tensor, nq: int, nkv: int, head_dim: int, scale: float | None = None, window: int = 0,
                  sink: torch.Tensor | None = None, wide_weights: bool = False) -> torch.Tensor:
    """Attention of the step's queries (the first nq * head_dim columns of `qkv`, rotated) over a lane in 4 bits: every token sees the positions
    up to its own (with `window` the last so many of them), which `kv4_store` has filled.  `sink` (float32 [nq]): the softmax's denominator also
    holds exp(sink[h]).  `scale` is head_dim ** -0.5 when None.  float32 and bfloat16; rows of padding (token_req < 0) are left as they are.

    Captured steps: ctx.extras["graph"] says that every row is a request's one token and that the device alone knows the lengths (`positions`), so that a graph
    serves the lengths that it is replayed with.  Another step has a call before its capture, and its graph serves the tokens and lengths of that call; what the
    call copied to the device for them is kept until the process ends.

    bfloat16, softmax weights in bfloat16: single tokens and a few of a request on the tensor cores from the cache's bytes (csrc/attention_kv4_tc.cu: heads
    of 64, 128 or 256, pages of 8, 16 or a multiple of 32 tokens); longer portions of prompts unfold the keys and values that they see into bfloat16 once
    and take the attention over such a cache (heads up to 128, rows of q on 16-byte boundaries).  Everything else, float32 above all: float
    throughout (csrc/attention_kv4.cu).  `wide_weights`: bfloat16 in float too, portions with weights of about 16 bits, as `attention` has it."""
    _on_current_device(qkv, out, lane.k, lane.v, lane.block_table, ctx.positions, ctx.token_req, sink)
    _check_lane("attention_kv4", lane, nkv, head_dim)
    if qkv.dim() != 2 or out.dim() != 2:
        raise KernelError("attention_kv4: q and out are matrices, a row to a token")
    n = out.shape[0]
    code = dtype_code(qkv.dtype)
    _check_step("attention_kv4", ctx.positions, ctx.token_req, n)
    if nq < 1 or nq % nkv or window < 0:
        raise KernelError(f"attention_kv4: {nq} query heads over {nkv}, a window of {window}")
    (ldq, inner), (ldo, inner_o) = qkv.stride(), out.stride()
    if qkv.shape[0] != n or qkv.shape[1] < nq * head_dim or out.shape != (n, nq * head_dim) or out.dtype != qkv.dtype or (n and (inner != 1 or inner_o != 1)):
        raise KernelError(f"attention_kv4: q [N, >= {nq * head_dim}] and out [N, {nq * head_dim}] in one type with unit inner strides are needed")
    if sink is not None and (sink.dtype != torch.float32 or sink.numel() != nq or not sink.is_contiguous()):
        raise KernelError("attention_kv4: the sink is one contiguous float32 number per query head")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    group, sms, window = nq // nkv, sm_count(), min(int(window), 1 << 30)
    tensor_core = not wide_weights and kv4_tensor_core_ok(qkv.dtype, head_dim, lane.page_size)
    unfold = code == BF16 and head_dim <= 128 and ldq % 8 == 0 and ldo % 2 == 0 and qkv.data_ptr() % 16 == 0 and out.data_ptr() % 4 == 0
    plan, stream = _kv4_plan(ctx, lane, group, nkv, head_dim, window, tensor_core, unfold), _stream()
    _check_table(lane, plan["held"], plan["requests"])
    _plan_on_this_stream(plan, stream)
    if plan["n_rows"] and not tensor_core:
        longest, splits = plan["longest"], 1
        if window and longest is not None:
            longest = min(longest, window)
        blocks = plan["n_rows"] * nkv * -(-group // 8)
        while splits < 8 and blocks * splits * 2 <= 2 * sms and (longest is None or longest > 256 * splits):  # a tile of 32 keys to each of eight warps
            splits *= 2
        lib.call("ns_attention_kv4", qkv.data_ptr(), qkv.stride(0), lane.k.data_ptr(), lane.v.data_ptr(), lane.block_table.data_ptr(),
                 lane.block_table.stride(0), ctx.token_req.data_ptr(), ctx.positions.data_ptr(), _ptr(plan["rows"]), plan["n_rows"], out.data_ptr(),
                 out.stride(0), nq, nkv, head_dim, lane.page_size, scale, window, _ptr(sink), splits, code, stream)
    for rows, items, count, n_blocks, (warps, splits, least), jobs, n_jobs, floats in plan["runs"]:
        part = torch.empty(floats, dtype=torch.float32, device=out.device) if floats else None
        lib.call("ns_attention_kv4_tc", qkv.data_ptr(), ldq, lane.k.data_ptr(), lane.v.data_ptr(), lane.block_table.data_ptr(), lane.block_table.stride(0),
                 ctx.token_req.data_ptr(), ctx.positions.data_ptr(), _ptr(rows), _ptr(items), count, out.data_ptr(), ldo, nq, nkv, head_dim, lane.page_size,
                 scale, window, _ptr(sink), n_blocks, warps, splits, _ptr(part), _ptr(jobs), n_jobs, least, stream)
    for portion in plan["portions"]:
        _attend_unfolded(qkv, lane, ctx, out, nkv, group, head_dim, scale, window, sink, portion, wide_weights)
    return out
