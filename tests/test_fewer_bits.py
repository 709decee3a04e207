"""Serving in fewer bits without a GPU: what is refused before a launch, and sizes."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor
from types import SimpleNamespace

import pytest
import torch

from plain_fewer_bits import held4, rows_i8, step, to_bf16


def test_operands_on_the_cpu_are_refused():
    from nanospec_b200 import ops
    from nanospec_b200.ops import KernelError
    ctx, lane, qkv = step([(3, 2)], 16, 2, 64, nq=4, device="cpu")
    x, w = torch.randn(2, 16), ops.RowsI8(torch.zeros((8, 16), dtype=torch.int8), torch.ones(8))
    for call in (lambda: ops.quantize_rows(x), lambda: ops.linear_i8(x, w, torch.empty(2, 8)), lambda: ops.kv4_store(qkv, ctx, lane, 4, 2, 64),
                 lambda: ops.kv4_read(lane, ctx.positions, ctx.token_req, 2, 64),
                 lambda: ops.attention_kv4(qkv, lane, ctx, torch.empty((2, 256), dtype=torch.bfloat16), 4, 2, 64)):
        with pytest.raises(KernelError, match="CUDA"):
            call()


def test_sizes_of_pages():
    from nanospec_b200 import ops
    from nanospec_b200.ops import KernelError
    assert ops.kv4_block_bytes(16, 128) == 16 * 80 and ops.kv4_block_bytes(1, 32) == 20
    assert ops.kv4_pages(3, 2, 16, 64, "cpu").shape == (3, 2, 640)
    for page, dim in ((0, 64), (16, 48), (16, 288), (16, 0)):
        with pytest.raises(KernelError):
            ops.kv4_block_bytes(page, dim)


def test_the_plain_statement_of_four_bits():
    """What the statement that the kernels are held against does itself: borders of its range, and how far a value is off."""
    x = torch.randn((50, 64), dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    y = held4(x)
    g, h = x.reshape(50, 2, 32), y.reshape(50, 2, 32)
    spread = (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) * 16 / 15
    assert ((g - h).abs() <= spread * (1 / 32 + 2.0 ** -7) + (g.abs().amax(-1, keepdim=True) + spread) * 2.0 ** -7).all()
    assert torch.equal(held4(torch.full((1, 32), 3.0, dtype=torch.float64)), torch.full((1, 32), 3.0, dtype=torch.float64))
    for v, want in ((1.0 + 2.0 ** -8, 1.0), (1.0 + 3 * 2.0 ** -8, 1.0 + 2.0 ** -6), (1.0 + 2.0 ** -8 + 2.0 ** -40, 1.0 + 2.0 ** -7)):
        assert to_bf16(torch.tensor([v], dtype=torch.float64)).item() == want
    q, s = rows_i8(torch.tensor([[127.0, 0.5, 1.5, -2.5], [0.0, 0.0, 0.0, 0.0]]))
    assert q.tolist() == [[127, 0, 2, -2], [0, 0, 0, 0]] and s.tolist() == [1.0, 0.0]


@pytest.mark.parametrize("M,N,K,tile", [
    (1, 2048, 2048, (16, 128, 8)), (8, 28672, 4096, (16, 128, 1)), (8, 4096, 14336, (16, 128, 8)), (32, 4096, 4096, (32, 128, 4)), (64, 28672, 4096, (64, 128, 1)),
    (77, 1003, 2051, (128, 128, 8)), (128, 28672, 4096, (256, 256, 1)), (200, 4096, 4096, (256, 64, 1)), (256, 4096, 14336, (256, 128, 2)),
    (512, 4096, 14336, (256, 256, 2)), (512, 6144, 4096, (256, 192, 1)), (4096, 28672, 4096, (256, 256, 1)), (5, 10, 1, (16, 128, 1)), (500, 10, 1, (256, 64, 1)),
])
def test_tiles_of_products(M, N, K, tile):
    """The fastest of those measured, at sizes on both sides of every border."""
    from nanospec_b200 import ops
    assert ops.i8_tiles(M, N, K, 148) == tile


@pytest.mark.parametrize("requests,group,nkv,dim,unfolded", [
    # from the bytes, unfolded (us)
    ([(64, 30064)], 4, 8, 128, False),             # 202, 328
    ([(24, 3024)] * 8, 4, 8, 128, False),          # 74, 104
    ([(64, 3064)] * 8, 4, 8, 128, True),           # 166, 106
    ([(24, 1024)] * 32, 4, 8, 128, False),         # 113, 143
    ([(48, 1048)] * 32, 4, 8, 128, True),          # 203, 154
    ([(64, 564)] * 8, 4, 8, 128, True),            # 61, 35
    ([(16, 516)] * 8, 4, 8, 128, False),           # 23, 33
    ([(24, 3024)] * 8, 8, 8, 128, False),          # 135, 172
    ([(48, 3048)] * 8, 8, 8, 128, True),           # 240, 175
    ([(1, 5000)] * 4, 4, 8, 128, False),           # nothing but decoding
    ([(2, 100), (512, 3512)], 4, 8, 128, True),
])
def test_which_portions_are_unfolded(requests, group, nkv, dim, unfolded):
    from nanospec_b200 import ops
    got = ops.kv4_unfolded(requests, group, nkv, dim, 0, 148, True)
    assert bool(got) == unfolded
    if unfolded:
        assert got == [i for i, (n, _) in enumerate(requests) if n > 2]


def test_runs_of_what_is_unfolded():
    from nanospec_b200 import ops
    one = ops.KV4_UNFOLD_PAGE * 128 * 4
    runs = lambda chunks, limit: ops.kv4_unfold_runs(chunks, 4, 128, limit * one)  # noqa: E731
    assert runs([3, 4, 5], 48) == [(0, 3, 0, 4)]
    assert runs([3, 4, 5], 28) == [(0, 2, 0, 4), (2, 1, 0, 4)]
    assert runs([3, 40, 5], 80) == [(0, 1, 0, 4), (1, 1, 0, 2), (1, 1, 2, 2), (2, 1, 0, 4)]
    assert runs([40], 1) == [(0, 1, h, 1) for h in range(4)]
    assert runs([], 10) == []


def test_tiles_of_a_few_tokens():
    from nanospec_b200 import ops
    assert ops.kv4_token_tiles([(0, 2, 9), (5, 6, 9)], 4) == ([(0, 2), (5, 4), (9, 2)], 2)
    assert ops.kv4_token_tiles([(3, 2, 9)], 4) == ([(3, 2)], 1)
    assert ops.kv4_token_tiles([(0, 3, 9)], 20) == ([(0, 1), (1, 1), (2, 1)], 2)


@pytest.mark.parametrize("head_dim,n_blocks,resident", [(128, 1, 4), (128, 2, 3), (64, 1, 6), (64, 2, 3), (256, 1, 2), (256, 2, 2)])
def test_shape_of_a_launch(head_dim, n_blocks, resident):
    from nanospec_b200 import ops
    for per_row in (1, 2, 8, 1000):
        for lengths in ((1,), (0,), (33,), (1000,), (100000,), (3000000,), (100000, 61000), (5, 100000), (700,) * 16, (4000,) * 16, (2300, 500) * 32, (9,) * 5000,
                        (100000,) + (500,) * 63):
            slots, rows = 148 * resident, len(lengths)
            for known in (True, False):
                warps, splits, least = ops.kv4_shape(lengths if known else None, rows, per_row, 148, head_dim, n_blocks)
                assert warps in (4, 8) and 1 <= splits <= 256 and (least > 0) == (splits > 1)
                if splits > 1 and known:
                    jobs = ops.kv4_jobs([(7 * z, z % 3 + 1) for z in range(rows)], lengths, least)
                    n = (len(jobs) - 2 * rows) // 4
                    assert warps == 4 and least >= 4 and n <= max(slots // per_row, 2 * rows)  # every block has its place at once, or two waves at most
                    spans = [jobs[4 * n + 2 * z: 4 * n + 2 * z + 2] for z in range(rows)]
                    for (first, parts), keys in zip(spans, lengths):
                        assert parts == max(1, -(-keys // (32 * least))) <= splits
                    assert [jobs[4 * i: 4 * i + 4] for i in range(n)] == [[7 * z, z % 3 + 1, p, parts] for z, (_, parts) in enumerate(spans) for p in range(parts)]
                    assert [first for first, _ in spans] == [sum(parts for _, parts in spans[:z]) for z in range(rows)]
                elif splits > 1:
                    assert rows * per_row * splits <= slots
    assert ops.kv4_shape((100000,) + (500,) * 63, 64, 8, 148, 128)[1] > 50  # (one request would outlast all others)
    assert ops.kv4_shape((100000,), 1, 1, 148, 128)[1] > 200  # (one kv head: more blocks than are joined would find a place)
    assert ops.kv4_shape((100000,), 1, 8, 148, 128)[1] > 60 and ops.kv4_shape((16,), 1, 8, 148, 128) == (8, 1, 0)


def _in_a_thread(fn):
    """(What a launch asks of its thread ends with the thread.)"""
    with ThreadPoolExecutor(1) as pool:
        return pool.submit(fn).result()


class _Stream:
    """A stream that notes what is asked of it, and whether the thread's next launch is a full one by then."""

    def __init__(self, seen):
        self.seen = seen

    def wait_event(self, event):
        self.seen.append((event, self.pending()))

    @staticmethod
    def pending():
        from nanospec_b200.ops import lib
        return lib.load().ns_full_launch_pending()


def test_a_call_that_waits_for_a_steps_lists_starts_when_they_are_there(monkeypatch):
    """The launch behind the wait is not made to overlap its predecessor in the stream: it has a prerequisite beside it."""
    from nanospec_b200.ops import kv4
    seen, kept = [], []
    here = _Stream(seen)
    monkeypatch.setattr(kv4.torch.cuda, "current_stream", lambda *a: here)
    monkeypatch.setattr(kv4.torch.cuda, "is_current_stream_capturing", lambda: False)
    held = SimpleNamespace(record_stream=kept.append)
    plan = {"lists": [held, held], "ready": "copied", "streams": {7}}

    def calls():
        kv4._plan_on_this_stream({"lists": []}, 7), kv4._plan_on_this_stream(plan, 7)  # no lists; the stream that copied them
        before = here.pending()
        kv4._plan_on_this_stream(plan, 8)
        return before, here.pending()
    assert _in_a_thread(calls) == (0, 1)
    assert seen == [("copied", 0)] and kept == [here, here] and plan["streams"] == {7, 8}

    def again():
        kv4._plan_on_this_stream(plan, 8)
        return here.pending()
    assert _in_a_thread(again) == 0 and len(seen) == 1


def test_a_captured_call_keeps_a_steps_lists(monkeypatch):
    """Without the mark of captured steps: waited for on the host, once, and kept beyond the step."""
    from nanospec_b200.ops import KernelError, kv4
    status, waited = [0], []

    def wait(event):
        waited.append(event)
        return status[0]
    monkeypatch.setattr(kv4.lib, "load", lambda: SimpleNamespace(ns_event_synchronize=wait, ns_last_error=lambda: b"why"))
    monkeypatch.setattr(kv4.torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(kv4, "_captured_lists", [])
    lists = ["rows", "jobs"]
    plan = {"lists": lists, "ready": SimpleNamespace(cuda_event=5), "streams": {7}}
    kv4._plan_on_this_stream({"lists": []}, 7)
    assert kv4._captured_lists == []
    for stream in (7, 8, 8):
        kv4._plan_on_this_stream(plan, stream)
    assert waited == [5] and len(kv4._captured_lists) == 1 and kv4._captured_lists[0] is lists and plan["streams"] == {7}
    status[0] = 1
    with pytest.raises(KernelError, match="why"):
        kv4._plan_on_this_stream({"lists": lists, "ready": SimpleNamespace(cuda_event=6), "streams": {7}}, 7)


def test_a_steps_lists_are_not_made_in_a_capture(monkeypatch):
    from nanospec_b200.ops import KernelError, kv4
    ctx, lane, _ = step([(40, 1), (100, 1)], 16, 2, 64, nq=4, device="cpu")
    monkeypatch.setattr(kv4, "sm_count", lambda: 148)
    monkeypatch.setattr(kv4.torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(KernelError, match="captured"):
        kv4._kv4_plan(ctx, lane, 2, 2, 64, 0, True, True)
    assert not ctx.extras
    ctx.extras["graph"] = True
    assert kv4._kv4_plan(ctx, lane, 2, 2, 64, 0, True, True)["runs"]


def test_shape_of_a_captured_step_with_a_window():
    """A window far beyond the contexts hides nothing: as without one.  One that decides how many keys there are at most: as if all requests held it."""
    from nanospec_b200 import ops
    for head_dim, n_blocks in ((64, 1), (128, 1), (128, 2), (256, 1)):
        for rows in (1, 2, 8, 30, 64, 200):
            for per_row in (1, 2, 8):
                free = ops.kv4_shape(None, rows, per_row, 148, head_dim, n_blocks)
                for window in (1, 40, 200, 1000, 4096, 32768, 131072, 1 << 30):
                    shape = ops.kv4_shape(None, rows, per_row, 148, head_dim, n_blocks, window)
                    known = ops.kv4_shape((window,) * rows, rows, per_row, 148, head_dim, n_blocks)
                    assert shape == (known if known[2] <= 8 else free)  # never fewer blocks for a short context than one for each eight tiles
    for rows, window, splits in ((1, 131072, 74), (8, 131072, 9), (8, 32768, 9)):
        assert ops.kv4_shape(None, rows, 8, 148, 128, 1, window) == ops.kv4_shape(None, rows, 8, 148, 128) == (4, splits, 8)


def test_a_captured_steps_plan_with_a_window(monkeypatch):
    from nanospec_b200.ops import kv4
    monkeypatch.setattr(kv4, "sm_count", lambda: 148)
    ctx, lane, _ = step([(40, 1)], 16, 8, 128, nq=32, device="cpu")
    ctx.extras["graph"] = True
    wide, none = (kv4._kv4_plan(ctx, lane, 4, 8, 128, window, True, True)["runs"] for window in (131072, 0))
    assert wide == none and none[0][4] == (4, 74, 8)


def test_the_lengths_of_portions_are_checked(monkeypatch):
    """The device's lengths and first rows of requests, which the kernels of unfolded portions read: a number to each request, 32 bits, on the device."""
    from nanospec_b200.ops import KernelError, kv4
    monkeypatch.setattr(kv4, "sm_count", lambda: 148)
    monkeypatch.setattr(kv4, "kv4_unfolded", lambda *a: [0])
    ctx, lane, _ = step([(2000, 300), (5, 1)], 16, 2, 64, nq=4, device="cpu")
    for name, bad in (("kv_len", ctx.kv_len.long()), ("kv_len", ctx.kv_len[:1]), ("qo_indptr", ctx.qo_indptr.long()), ("qo_indptr", ctx.qo_indptr[:2])):
        with pytest.raises(KernelError, match=name):
            kv4._kv4_plan(SimpleNamespace(**{**vars(ctx), name: bad}), lane, 2, 2, 64, 0, True, True)
    with pytest.raises(KernelError, match="CUDA"):
        kv4._kv4_plan(ctx, lane, 2, 2, 64, 0, True, True)
    assert not ctx.extras
