"""What a fork or a join asks of its own thread's next launch, other threads leave alone."""

from __future__ import annotations

import threading

import pytest
import torch


def _in_thread(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    return out[0]


def test_a_full_launch_is_asked_of_one_thread():
    from nanospec_b200.ops import lib
    native = lib.load()

    def ask():
        native.ns_full_launch_next()
        return native.ns_full_launch_pending(), _in_thread(native.ns_full_launch_pending)
    assert _in_thread(ask) == (1, 0)
    assert native.ns_full_launch_pending() == 0


@pytest.mark.gpu
def test_another_threads_launch_does_not_take_it():
    from nanospec_b200 import ops
    from nanospec_b200.ops import lib
    native = lib.load()
    table, ids, out = torch.randn(8, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.empty(2, 64, device="cuda")

    def launch():
        ops.embed(table, ids, out)
        return native.ns_full_launch_pending()

    def ask():
        native.ns_full_launch_next()
        return _in_thread(launch), native.ns_full_launch_pending(), launch()
    assert _in_thread(ask) == (0, 1, 0)


@pytest.mark.gpu
def test_attention_beside_attention_asks_for_full_launches(monkeypatch):
    """Single tokens beside portions of prompts: the side stream's launch behind the fork, and the next one behind the join, overlap nothing."""
    from nanospec_b200 import ops
    from nanospec_b200.ops import lib
    from plain_fewer_bits import step
    native = lib.load()
    ctx, lane, qkv = step([(30, 1), (0, 40), (7, 1)], 16, 2, 64, torch.bfloat16, 4)
    lane.k, lane.v = (torch.randn((lane.k.shape[0], 2, 16, 64), device="cuda").bfloat16() for _ in range(2))
    want = torch.zeros((ctx.n_tokens, 256), dtype=torch.bfloat16, device="cuda")
    monkeypatch.setattr(ops, "OVERLAP_MIXED_ATTENTION", False)
    ops.attention(qkv, lane, ctx, want, 4, 2, 64, 0.125)
    monkeypatch.setattr(ops, "OVERLAP_MIXED_ATTENTION", True)
    seen, decode, prefill = [], ops.attention_decode, ops.attention_prefill

    def noted(name, fn):
        def call(*args):
            seen.append((name, native.ns_full_launch_pending()))
            return fn(*args)
        return call
    monkeypatch.setattr(ops, "attention_decode", noted("decode", decode))
    monkeypatch.setattr(ops, "attention_prefill", noted("prefill", prefill))
    out = torch.zeros_like(want)
    ops.attention(qkv, lane, ctx, out, 4, 2, 64, 0.125)
    assert seen == [("prefill", 0), ("decode", 1)] and native.ns_full_launch_pending() == 1
    ops.embed(torch.randn(8, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.empty(2, 64, device="cuda"))
    assert native.ns_full_launch_pending() == 0
    assert torch.equal(out, want)
