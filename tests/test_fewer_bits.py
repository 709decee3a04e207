"""Serving in fewer bits without a GPU: what is refused before a launch, and sizes."""

from __future__ import annotations

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
