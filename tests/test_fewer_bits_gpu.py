"""Serving in fewer bits on the GPU, against plain statements in 64 bits: rows and products in 8-bit integers, the 4-bit cache, attention over it."""

from __future__ import annotations

import math

import pytest
import torch

from plain_fewer_bits import F64, TINY, attend, everything, fill, half_step, held4, in_type, rotated, rows_i8, step, to_bf16

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _near(got, want, tol):
    """Nowhere off by more than its tolerance; says where if it is."""
    off = (got.double().reshape(want.shape) - want).abs()
    at = ~(off <= tol)  # (a NaN is off)
    assert not at.any(), f"{int(at.sum())} of {at.numel()} off, the first at {at.nonzero()[0].tolist()}: {got.reshape(want.shape)[at][0]} for {want[at][0]}, tolerance {tol[at][0]}"


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ---- rows in 8-bit integers -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,K,dtype", [(1, 1, F32), (3, 7, BF16), (5, 16, F32), (70, 2048, BF16), (2, 8193, F32), (4, 20000, BF16), (1, 131072, F32)])
def test_rows_are_the_definition_to_the_last_bit(rows, K, dtype):
    from nanospec_b200 import ops
    x = (_rand(rows, K, seed=K) * torch.exp(2 * _rand(rows, 1, seed=1))).to(dtype)
    got, (q, scale) = ops.quantize_rows(x), rows_i8(x)
    assert torch.equal(got.scale, scale) and torch.equal(got.q.double(), q)
    assert got.q.stride(0) % 16 == 0 and got.q.data_ptr() % 16 == 0
    assert torch.equal(got.values(), q.float() * scale[:, None])


def test_rows_at_ties():
    from nanospec_b200 import ops
    # the largest is 127 steps: halves of a step are ties, their neighbours in float32 are not
    for unit in (1.0, 0.25, 2.0 ** -60):
        k = torch.arange(-253, 254, 2, device="cuda").double() / 2
        x = torch.cat([k, torch.tensor([127.0], device="cuda", dtype=F64)]).float() * unit
        near = torch.cat([torch.nextafter(x, x + 1), torch.nextafter(x, x - 1)])
        m = torch.stack([x, near[: x.numel()].clamp(-127 * unit, 127 * unit), near[x.numel():].clamp(-127 * unit, 127 * unit)])
        m[:, -1] = 127 * unit
        got, (q, scale) = ops.quantize_rows(m), rows_i8(m)
        assert torch.equal(got.scale, scale) and torch.equal(got.q.double(), q)


def test_rows_that_are_zero_tiny_or_not_finite():
    from nanospec_b200 import ops
    x = _rand(8, 40)
    x[0] = 0
    x[1, 3], x[2, 39], x[3, 0] = math.inf, math.nan, -math.inf
    x[4] *= 2.0 ** -122
    x[5] *= 2.0 ** -100
    x[6, 0] = 3.3e38
    got, (q, scale) = ops.quantize_rows(x), rows_i8(x)
    assert torch.equal(got.scale.isnan(), scale.isnan()) and got.scale.isnan().tolist() == [False, True, True, True, False, False, False, False]
    assert torch.equal(got.scale.nan_to_num(-1.0), scale.nan_to_num(-1.0)) and torch.equal(got.q.double(), q)


def test_rows_of_a_wider_buffer():
    from nanospec_b200 import ops
    wide = _rand(6, 100, dtype=BF16)
    for x in (wide[:, 3:50], wide[::2], wide[:, 8:96]):
        got, (q, scale) = ops.quantize_rows(x), rows_i8(x)
        assert torch.equal(got.scale, scale) and torch.equal(got.q.double(), q)
    assert ops.quantize_rows(wide[:0]).q.shape == (0, 100)


# ---- products -------------------------------------------------------------------------------------------------------------------------
def _product(x, w, dtype, bias=None):
    """(what comes, its tolerance): the sum's, the scales' and their product's rounding, the bias's and the output's."""
    y = (x.q.double() @ w.q.double().T) * x.scale.double()[:, None] * w.scale.double()[None, :]
    tol = y.abs() * 3.01 * TINY
    if bias is not None:
        y = y + bias.double()
        tol = tol + y.abs() * TINY
    return y, tol + y.abs() * 1.01 * half_step(dtype)


SIZES = [(1, 1, 1), (1, 128, 16), (2, 129, 17), (7, 333, 100), (16, 256, 128), (17, 1000, 2051), (33, 128, 4096), (64, 640, 1024), (65, 200, 300),
         (100, 515, 129), (128, 384, 2048), (129, 257, 640), (200, 1000, 4100), (256, 512, 256), (300, 1003, 515), (513, 770, 1000), (1000, 129, 130)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product(M, N, K, dtype):
    from nanospec_b200 import ops
    x, w = _rand(M, K, seed=1, dtype=dtype), ops.quantize_rows(_rand(N, K, seed=2))
    bias = _rand(N, seed=3)
    held = ops.quantize_rows(x)
    for b in (None, bias):
        out = torch.full((M, N), math.nan, dtype=dtype, device="cuda")
        assert ops.linear_i8(x, w, out, b) is out
        want, tol = _product(held, w, dtype, b)
        _near(out, want, tol)
        again = torch.empty_like(out)
        ops.linear_i8(held, w, again, b)
        assert torch.equal(out, again)


@pytest.mark.parametrize("M", [1, 20, 100, 300])
def test_product_sums_are_exact(M):
    """Every term the largest: sums beyond 2^24, where float would round; and the sign of every corner."""
    from nanospec_b200 import ops
    K, N = 131072, 130
    x = torch.full((M, K), 127, dtype=torch.int8, device="cuda")
    x[M // 2, K // 2:] = -127
    w = torch.full((N, K), -127, dtype=torch.int8, device="cuda")
    w[5, 1] = 126
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    out = torch.empty((M, N), device="cuda")
    ops.linear_i8(ops.RowsI8(x, one(M)), ops.RowsI8(w, one(N)), out)
    assert torch.equal(out, (x.double() @ w.double().T).float())


@pytest.mark.parametrize("M", [3, 40, 140, 520])
def test_product_with_strides_and_what_lies_beside(M):
    from nanospec_b200 import ops
    K, N = 200, 300
    x, held = _rand(M, K, seed=1), torch.full((N, 320), 99, dtype=torch.int8, device="cuda")
    w = ops.quantize_rows(_rand(N, K, seed=2))
    held[:, 16: 16 + K] = w.q
    for off, gap in ((0, 0), (3, 5), (8, 12)):
        buf = torch.full((M + 2, N + off + gap), 7.0, dtype=BF16, device="cuda")
        out = buf[1: M + 1, off: off + N]
        ops.linear_i8(x, ops.RowsI8(held[:, 16: 16 + K], w.scale), out)
        want, tol = _product(ops.quantize_rows(x), w, BF16)
        _near(out, want, tol)
        assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :off] == 7).all() and (buf[:, off + N:] == 7).all()


@pytest.mark.parametrize("M,N,K", [(200, 300, 520), (300, 129, 2051), (40, 770, 1000)])
def test_product_has_the_same_bits_in_every_tile(M, N, K):
    from nanospec_b200 import ops
    x, w, bias = ops.quantize_rows(_rand(M, K, seed=1)), ops.quantize_rows(_rand(N, K, seed=2)), _rand(N, seed=3)
    tiles = [(t, 128, s) for t in (16, 32, 64, 128) for s in (1, 2, 4)] + [(256, f, s) for f in (64, 128, 192, 256) for s in (1, 2)]
    outs = [ops.linear_i8(x, w, torch.empty((M, N), device="cuda"), bias, t) for t in tiles]
    assert all(torch.equal(outs[0], o) for o in outs)
    ops.check_kernel_errors()


def test_weights_quantised_directly_before_the_product():
    """The product asks for its weights ahead of its turn: not before the kernel that writes them is through."""
    from nanospec_b200 import ops
    x = _rand(8, 4096, seed=1, dtype=BF16)
    raw = [_rand(8192, 4096, seed=s) for s in (2, 3)]
    want = []
    for r in raw:
        w = ops.quantize_rows(r)
        torch.cuda.synchronize()
        want.append(ops.linear_i8(x, w, torch.empty((8, 8192), device="cuda")))
    torch.cuda.synchronize()
    held = ops.quantize_rows(raw[0])
    for i in range(20):
        new = ops.quantize_rows(raw[i % 2])
        held.q.copy_(new.q), held.scale.copy_(new.scale)
        assert torch.equal(ops.linear_i8(x, ops.quantize_rows(raw[i % 2]), torch.empty((8, 8192), device="cuda")), want[i % 2])
        assert torch.equal(ops.linear_i8(x, held, torch.empty((8, 8192), device="cuda")), want[i % 2])
        assert torch.equal(ops.linear_i8(ops.quantize_rows(x), ops.quantize_rows(raw[i % 2]), torch.empty((8, 8192), device="cuda")), want[i % 2])


def test_product_keeps_what_is_not_finite_in_its_row():
    from nanospec_b200 import ops
    for M in (4, 90, 300):
        x, w = _rand(M, 64, seed=1), ops.quantize_rows(_rand(140, 64, seed=2))
        want = ops.linear_i8(x, w, torch.empty((M, 140), device="cuda")).clone()
        x[2, 7] = math.nan
        x[3, 1] = math.inf
        got = ops.linear_i8(x, w, torch.empty((M, 140), device="cuda"))
        assert got[2:4].isnan().all()
        keep = [i for i in range(M) if i not in (2, 3)]
        assert torch.equal(got[keep], want[keep])


def test_product_refusals():
    from nanospec_b200 import ops
    from nanospec_b200.ops import KernelError
    x, w = _rand(4, 64), ops.quantize_rows(_rand(32, 64))
    out = torch.empty((4, 32), device="cuda")
    bad = [
        (x, w, torch.empty((4, 31), device="cuda"), None),
        (x, w, torch.empty((32, 4), device="cuda").T, None),
        (x, w, out.half(), None),
        (x.half(), w, out, None),
        (x[:, :63], w, out, None),
        (x.T.contiguous().T, w, out, None),
        (x, ops.RowsI8(w.q.float(), w.scale), out, None),
        (x, ops.RowsI8(w.q, w.scale[:31]), out, None),
        (x, ops.RowsI8(w.q, w.scale.double()), out, None),
        (x, ops.RowsI8(w.q[:, :50].contiguous(), w.scale), out, None),
        (x, w, out, torch.zeros(31, device="cuda")),
        (x, w, out, torch.zeros(32, device="cuda", dtype=BF16)),
        (x.cpu(), w, out, None),
        (x, w, out.cpu(), None),
        (x[:, :0], ops.RowsI8(w.q[:, :0], w.scale), out, None),
        (torch.zeros((4, 131073), device="cuda"), ops.RowsI8(torch.zeros((32, 131088), dtype=torch.int8, device="cuda")[:, :131073], w.scale), out, None),
    ]
    for args in bad:
        with pytest.raises(KernelError):
            ops.linear_i8(*args)
    for t in (x.half(), x[0], x.T, x[:, :0], torch.zeros((2, 131073), device="cuda")):
        with pytest.raises(KernelError):
            ops.quantize_rows(t)
    assert ops.linear_i8(x[:0], w, out[:0]).shape == (0, 32)


# ---- the store ----------------------------------------------------------------------------------------------------------------------------
def _inv_freq(dim, base=500000.0, pairs=None):
    return (base ** (-torch.arange(dim // 2, dtype=F64) * 2 / dim)).float()[: pairs if pairs is not None else dim // 2].contiguous().cuda()


@pytest.mark.parametrize("lens,page,nq,nkv,dim,pairs", [
    ([(0, 1)], 16, 1, 1, 32, None), ([(5, 1), (131000, 1), (15, 1)], 16, 4, 2, 64, None), ([(0, 33), (7, 5)], 8, 3, 3, 96, None),
    ([(100, 40)], 16, 32, 8, 128, None), ([(3, 20), (0, 2)], 3, 7, 1, 256, None), ([(0, 17)], 1, 2, 2, 160, 40), ([(9, 12)], 64, 8, 4, 128, 32),
    ([(0, 6)], 16, 4, 2, 64, 0), ([(1000, 300)], 32, 8, 8, 64, None),
])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_store_is_the_definition_to_the_last_bit(lens, page, nq, nkv, dim, pairs, dtype):
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, page, nkv, dim, dtype, nq, seed=dim + len(lens))
    qkv *= torch.exp(_rand(1, qkv.shape[1], seed=5)).to(dtype)
    f = None if pairs == 0 else _inv_freq(dim, pairs=pairs)
    x = qkv.clone().reshape(ctx.n_tokens, -1, dim)
    q_out = torch.empty((ctx.n_tokens, nq * dim), dtype=dtype, device="cuda")
    assert ops.kv4_store(qkv, ctx, lane, nq, nkv, dim, f, q_out=q_out) is q_out
    assert torch.equal(qkv, x.reshape(qkv.shape))
    k, v = ops.kv4_read(lane, ctx.positions, ctx.token_req, nkv, dim)
    turned = rotated(x[:, : nq + nkv], ctx.positions, f)
    assert torch.equal(k.double(), held4(in_type(turned[:, nq:], dtype)))
    assert torch.equal(v.double(), held4(x[:, nq + nkv:].double()))
    # q: the sine and cosine rounded, two products and a sum in float, then the type
    pairs_of = x[:, :nq].double().abs()
    size = pairs_of + torch.cat([pairs_of[..., dim // 2:], pairs_of[..., : dim // 2]], -1)
    _near(q_out, turned[:, :nq], size * 4 * TINY + turned[:, :nq].abs() * 1.01 * half_step(dtype))
    ops.kv4_store(qkv, ctx, lane, nq, nkv, dim, f)
    assert torch.equal(qkv[:, : nq * dim], q_out) and torch.equal(qkv[:, nq * dim:], x[:, nq:].reshape(ctx.n_tokens, -1))


def test_store_at_borders():
    """Codes that lie half way between two, groups of one value, spreads next to nothing, huge offsets."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(0, 12)], 16, 1, 64, F32, 1)
    v = qkv[:, 128:]
    v[0, :32] = torch.arange(32, device="cuda").float() / 2            # S = 16.5 -> bf16, ties and near ties
    v[1, :32] = torch.arange(32, device="cuda").float().remainder(16) - 0.5
    v[1, :2] = torch.tensor([0.0, 15.0], device="cuda") - 8            # S = 16, B a whole number: .5 are ties
    v[2] = 3.7
    v[3] = 0.0
    v[4] = 1e-30 * v[4]
    v[5] = 1e-33 * v[5]
    v[6] = 100 + 1e-3 * v[6]
    v[7] = -1e4 + v[7]
    v[8] = 1e30 * v[8]
    v[9, 0] = 1e-20
    v[10, :32] = torch.nextafter(v[1, :32], v[1, :32] + 1)
    v[11, :32] = torch.nextafter(v[1, :32], v[1, :32] - 1)
    v[10:12, 0], v[10:12, 1] = -8.0, 7.0
    want = held4(v.double().unsqueeze(1))
    ops.kv4_store(qkv, ctx, lane, 1, 1, 64)
    _, got = ops.kv4_read(lane, ctx.positions, ctx.token_req, 1, 64)
    assert torch.equal(got.double(), want)
    # a value is off by half a code, the rounding of S over 16 codes, the rounding of B, and its own
    g = v.double().reshape(12, 2, 32)
    spread = (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) * 16 / 15
    tol = spread * (1 / 32 + 2.0 ** -7) + (g.abs().amax(-1, keepdim=True) + spread) * 2.0 ** -7 + 2.0 ** -100
    assert ((got.double().reshape(12, 2, 32) - g).abs() <= tol).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_store_of_what_is_not_finite(dim, dtype):
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(0, 6)], 16, 2, dim, dtype, 1)
    x = qkv.reshape(6, 5, dim)
    x[1, 1, 3] = math.nan                 # a key of head 0
    x[2, 4, dim - 1] = math.inf           # a value of head 1
    x[3, 3, 0], x[3, 3, 1] = math.inf, -math.inf
    big = torch.finfo(dtype).max
    x[4, 2, 0], x[4, 2, 1] = big, -big    # a spread beyond bfloat16's range
    ops.kv4_store(qkv, ctx, lane, 1, 2, dim)
    k, v = ops.kv4_read(lane, ctx.positions, ctx.token_req, 2, dim)
    assert v.isfinite().all()
    nan = k.isnan()
    assert nan.all(-1).tolist() == [[False, False], [True, False], [False, True], [True, False], [False, True], [False, False]]
    assert torch.equal(nan.any(-1), nan.all(-1))
    assert (v[2, 1, -32:] == 0).all() and (v[3, 0, :32] == 0).all() and torch.equal(v[2, 1, :-32].double(), held4(x[2, 4, :-32].double()))


def test_store_leaves_what_is_not_its_own():
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(5, 3), (20, 1)], 8, 2, 64, BF16, 2, padding=3)
    lane.k.fill_(77), lane.v.fill_(78)
    before = qkv.clone()
    ops.kv4_store(qkv, ctx, lane, 2, 2, 64, _inv_freq(64))
    assert torch.equal(qkv[4:], before[4:])  # rows of padding
    at = lane.block_table.cpu()
    wrote = {(int(at[r, p // 8]), p % 8) for r, p in zip(ctx.token_req.tolist(), ctx.positions.tolist()) if r >= 0}
    codes = lane.k[..., : 8 * 32].reshape(-1, 2, 8, 32), lane.v[..., : 8 * 32].reshape(-1, 2, 8, 32)
    pairs = lane.k[..., 8 * 32:].reshape(-1, 2, 8, 8), lane.v[..., 8 * 32:].reshape(-1, 2, 8, 8)
    for page in range(lane.k.shape[0]):
        for slot in range(8):
            same = [bool((t[page, :, slot] == mark).all()) for group in (codes, pairs) for t, mark in zip(group, (77, 78))]
            assert all(same) != ((page, slot) in wrote)
    k, v = ops.kv4_read(lane, ctx.positions, ctx.token_req, 2, 64)
    assert (k[4:] == 0).all() and (v[4:] == 0).all()


# ---- attention ----------------------------------------------------------------------------------------------------------------------------
def _check(lens, page, nq, nkv, dim, dtype=BF16, window=0, sink=None, scale=None, padding=0, seed=0):
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, page, nkv, dim, dtype, nq, seed=seed, padding=padding)
    lane.k.fill_(255), lane.v.fill_(255)  # what nobody stored stands for NaN
    k, v = fill(ctx, lane, nq, nkv, dim, dtype, seed=seed + 1)
    n = ctx.n_tokens - padding
    out = torch.full((ctx.n_tokens, nq * dim), 5.0, dtype=dtype, device="cuda")
    assert ops.attention_kv4(qkv, lane, ctx, out, nq, nkv, dim, scale, window=window, sink=sink) is out
    want, tol8, tol32 = attend(qkv[:n, : nq * dim], k, v, ctx, nq, dim ** -0.5 if scale is None else scale, window, sink)
    got = out[:n].double().reshape(want.shape)
    tol = (tol32 if dtype == F32 else tol8) + want.abs() * 1.01 * half_step(dtype)
    _near(got, want, tol)
    assert (out[n:] == 5).all()
    again = torch.empty_like(out)
    ops.attention_kv4(qkv, lane, ctx, again, nq, nkv, dim, scale, window=window, sink=sink)
    assert torch.equal(again[:n], out[:n])


DECODE = [[(0, 1)], [(1, 1)], [(15, 1), (16, 1), (17, 1)], [(31, 1), (32, 1), (33, 1), (0, 1)], [(1000, 1)], [(63, 1), (640, 1), (127, 1), (2, 1), (300, 1)], [(5000, 1), (7, 1)]]


@pytest.mark.parametrize("lens", DECODE)
@pytest.mark.parametrize("nq,nkv,dim,page", [(32, 8, 128, 16), (8, 2, 64, 16), (3, 1, 128, 8), (7, 7, 64, 32), (12, 1, 128, 64), (20, 1, 64, 16), (16, 2, 256, 16)])
def test_decode(lens, nq, nkv, dim, page):
    _check(lens, page, nq, nkv, dim)


@pytest.mark.parametrize("dim,page,dtype", [(32, 16, BF16), (96, 16, BF16), (160, 8, BF16), (192, 16, BF16), (224, 16, F32), (256, 4, F32), (64, 16, F32), (128, 5, BF16),
                                            (128, 1, BF16), (64, 24, BF16), (128, 48, BF16), (128, 16, F32), (64, 3, F32), (64, 12, BF16)])
def test_heads_and_pages_of_every_size(dim, page, dtype):
    _check([(70, 1), (3, 4), (0, 20), (33, 1)], page, 6, 2, dim, dtype)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 100, 700])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, BF16), (64, F32)])
def test_windows(window, dim, dtype):
    _check([(600, 1), (5, 1), (90, 3), (64, 70), (0, 40)], 16, 8, 2, dim, dtype, window=window)


@pytest.mark.parametrize("lens", [[(0, 2)], [(0, 40)], [(3, 2), (31, 3), (100, 4)], [(200, 8), (50, 16), (0, 5), (10, 1)], [(1000, 6), (500, 17)], [(0, 300), (77, 130)],
                                  [(1500, 129), (4, 1), (0, 257)], [(20, 64), (16, 65)]])
@pytest.mark.parametrize("nq,nkv,dim,page", [(32, 8, 128, 16), (8, 2, 64, 16), (5, 5, 128, 32), (9, 1, 64, 8)])
def test_portions(lens, nq, nkv, dim, page):
    _check(lens, page, nq, nkv, dim)


@pytest.mark.parametrize("nq,nkv,dim,page,dtype", [(32, 8, 128, 16, BF16), (16, 2, 64, 8, BF16), (6, 2, 96, 16, BF16), (8, 4, 256, 32, BF16), (4, 2, 64, 16, F32)])
def test_steps_of_every_kind_of_request(nq, nkv, dim, page, dtype):
    """Single tokens, a few tokens, portions and requests that bring none in one step."""
    _check([(500, 1), (0, 200), (90, 3), (1200, 300), (3, 1), (40, 17), (0, 1), (300, 2)], page, nq, nkv, dim, dtype, padding=3)
    _check([(500, 1), (20, 200), (90, 3), (1200, 300), (3, 1)], page, nq, nkv, dim, dtype, window=150)


@pytest.mark.parametrize("lens", [[(900, 1), (300, 1)], [(900, 3), (20, 2)], [(900, 80), (10, 200)]])
@pytest.mark.parametrize("dim,page,dtype", [(128, 16, BF16), (64, 8, BF16), (128, 32, BF16), (128, 5, BF16), (64, 16, F32)])
def test_pages_behind_a_window_may_be_given_back(lens, dim, page, dtype):
    """Their table entries are then -1, and the pages hold somebody else's bytes, NaN among what those stand for."""
    from nanospec_b200 import ops
    window = 100
    ctx, lane, qkv = step(lens, page, 2, dim, dtype, 4)
    k, v = fill(ctx, lane, 4, 2, dim, dtype)
    for i, (held, _) in enumerate(lens):
        gone = max(0, held - window + 1) // page
        lane.k[lane.block_table[i, :gone].long()] = 255
        lane.v[lane.block_table[i, :gone].long()] = 255
        lane.block_table[i, :gone] = -1
    out = torch.empty((ctx.n_tokens, 4 * dim), dtype=dtype, device="cuda")
    ops.attention_kv4(qkv, lane, ctx, out, 4, 2, dim, window=window)
    want, tol8, tol32 = attend(qkv[:, : 4 * dim], k, v, ctx, 4, dim ** -0.5, window)
    _near(out, want, (tol32 if dtype == F32 else tol8) + want.abs() * 1.01 * half_step(dtype))


def test_portions_beyond_what_is_unfolded_at_a_time(monkeypatch):
    """Requests one after another, and a request whose kv heads go in parts: the same bits as together."""
    from nanospec_b200 import ops
    from nanospec_b200.ops import kv4
    ctx, lane, qkv = step([(0, 200), (700, 100), (64, 300), (10, 1)], 16, 4, 128, BF16, 8)
    fill(ctx, lane, 8, 4, 128)
    sink = _rand(8, seed=4)
    monkeypatch.setattr(kv4, "kv4_unfolded", lambda requests, *a: [i for i, (n, _) in enumerate(requests) if n > 1])
    want = ops.attention_kv4(qkv, lane, ctx, torch.zeros((ctx.n_tokens, 1024), dtype=BF16, device="cuda"), 8, 4, 128, sink=sink)
    one = kv4.KV4_UNFOLD_PAGE * 128 * 4
    for limit in (13 * 4 * one, 10 * 2 * one, one):
        monkeypatch.setattr(kv4, "KV4_UNFOLD_MAX", limit)
        ctx.extras = {}
        got = ops.attention_kv4(qkv, lane, ctx, torch.zeros_like(want), 8, 4, 128, sink=sink)
        assert torch.equal(got, want)


def test_more_rows_than_a_grid_dimension_holds():
    from nanospec_b200 import ops
    rows = 66000
    ctx, lane, qkv = step([(i, 1) for i in range(40)], 8, 1, 64, BF16, 1)
    k, v = fill(ctx, lane, 1, 1, 64)
    want, tol, _ = attend(qkv[:, :64], k, v, ctx, 1, 0.125)
    tol = tol + want.abs() * 1.01 * half_step(BF16)
    many = torch.arange(rows, device="cuda") % 40  # the same requests over and over
    ctx.positions, ctx.token_req, lane.block_table = ctx.positions[many], torch.arange(rows, dtype=torch.int32, device="cuda"), lane.block_table[many]
    ctx.q_lens, ctx.kv_lens = [1] * rows, [i % 40 + 1 for i in range(rows)]
    for graph in (False, True):
        ctx.extras = {"graph": True} if graph else {}
        got = ops.attention_kv4(qkv[many], lane, ctx, torch.empty((rows, 64), dtype=BF16, device="cuda"), 1, 1, 64)
        _near(got.double().reshape(rows, *want.shape[1:]), want[many], tol[many])


def test_two_calls_at_once():
    """The same cache read by two streams, and products of two streams: no scratch is shared."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(700, 1), (90, 5), (30, 120)], 16, 2, 128, BF16, 8)
    fill(ctx, lane, 8, 2, 128)
    x, w = _rand(90, 1024, dtype=BF16), ops.quantize_rows(_rand(1024, 1024, seed=2))
    want = ops.attention_kv4(qkv, lane, ctx, torch.zeros((ctx.n_tokens, 1024), dtype=BF16, device="cuda"), 8, 2, 128)
    product = ops.linear_i8(x, w, torch.empty((90, 1024), dtype=BF16, device="cuda"))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append((ops.attention_kv4(qkv, lane, ctx, torch.zeros_like(want), 8, 2, 128), ops.linear_i8(x, w, torch.empty_like(product))))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, product) for a, b in results)
    ops.check_kernel_errors()


@pytest.mark.parametrize("lens", [[(9, 1), (900, 1), (100, 1)], [(20, 1), (200, 3), (40, 90)]])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F32)])
def test_a_step_whose_calls_run_on_several_streams(lens, dim, dtype):
    """The first call's stream is late with the step's lists; the calls on others wait for them."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, 16, 2, dim, dtype, 8)
    fill(ctx, lane, 8, 2, dim, dtype)
    want = ops.attention_kv4(qkv, lane, ctx, torch.zeros((ctx.n_tokens, 8 * dim), dtype=dtype, device="cuda"), 8, 2, dim)
    outs = [torch.zeros_like(want) for _ in range(3)]
    ctx.extras = {}
    torch.cuda.synchronize()
    for i, (out, s) in enumerate(zip(outs, [torch.cuda.Stream() for _ in outs])):
        with torch.cuda.stream(s):
            if i == 0:
                torch.cuda._sleep(20_000_000)
            ops.attention_kv4(qkv, lane, ctx, out, 8, 2, dim)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("lens", [[(300, 1), (9, 1)], [(200, 3)], [(40, 90)]])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F32)])
def test_sink_scale_and_padding(lens, dim, dtype):
    sink = _rand(8, seed=9) * 3
    _check(lens, 16, 8, 2, dim, dtype, sink=sink, padding=5)
    _check(lens, 16, 8, 2, dim, dtype, scale=0.3, padding=1)
    _check(lens, 16, 8, 2, dim, dtype, scale=-0.2)
    _check(lens, 16, 8, 2, dim, dtype, scale=0.0, window=50)


@pytest.mark.parametrize("lens", [[(40, 1)], [(40, 5)], [(40, 100)]])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, BF16), (64, F32)])
def test_a_token_that_is_not_finite_reaches_those_that_see_it(lens, dim, dtype):
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, 16, 2, dim, dtype, 4)
    fill(ctx, lane, 4, 2, dim, dtype)
    total = ctx.kv_lens[0]
    clean = torch.empty((ctx.n_tokens, 4 * dim), dtype=dtype, device="cuda")
    for key, window in ((20, 0), (total - 1, 0), (10, 12), (total - 3, 0)):
        ops.attention_kv4(qkv, lane, ctx, clean, 4, 2, dim, window=window)
        kept = lane.k.clone(), lane.v.clone()
        one = type(ctx)(**vars(ctx))
        one.positions, one.token_req = (torch.tensor([v], dtype=torch.int32, device="cuda") for v in (key, 0))
        bad = torch.randn((1, 8 * dim), device="cuda").to(dtype)
        bad[0, 7 * dim + 1] = math.nan  # the value of kv head 1
        ops.kv4_store(bad, one, lane, 4, 2, dim)
        out = torch.empty_like(clean)
        ops.attention_kv4(qkv, lane, ctx, out, 4, 2, dim, window=window)
        pos = ctx.positions[:, None]
        sees = ((pos >= key) & ((window == 0) | (key > pos - window))).expand(-1, 2 * dim)
        assert torch.equal(out[:, 2 * dim:].isnan(), sees)
        assert torch.equal(out[:, 2 * dim:][~sees], clean[:, 2 * dim:][~sees])
        lane.k.copy_(kept[0]), lane.v.copy_(kept[1])


@pytest.mark.parametrize("nq,nkv,dim,page", [(8, 2, 128, 16), (4, 4, 64, 8), (20, 1, 128, 32), (6, 1, 256, 16)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_requests_over_several_blocks(nq, nkv, dim, page, tokens, monkeypatch):
    """The same step with its keys dealt to one block or to many: blocks without a tile, the most there may be, fewer than a request has tiles."""
    from nanospec_b200 import ops
    from nanospec_b200.ops import kv4
    lens = [(5200, tokens), (70, tokens), (0, tokens), (2111, tokens)]
    sink = _rand(nq, seed=3)
    ctx, lane, qkv = step(lens, page, nkv, dim, BF16, nq, padding=2)
    lane.k.fill_(255), lane.v.fill_(255)
    k, v = fill(ctx, lane, nq, nkv, dim)
    n = ctx.n_tokens - 2
    for window in (0, 100):
        want, tol, _ = attend(qkv[:n, : nq * dim], k, v, ctx, nq, dim ** -0.5, window, sink)
        tol = tol + want.abs() * 1.01 * half_step(BF16)
        for graph in (False, True) if tokens == 1 else (False,):
            for shape in (None, (4, 1, 0), (8, 1, 0), (4, 256, 1), (4, 7, 9), (4, 2, 100), (8, 3, 1)):
                if shape:
                    monkeypatch.setattr(kv4, "kv4_shape", lambda *a: shape)
                ctx.extras = {"graph": True} if graph else {}  # (with the blocks of each row listed, or as many for every row)
                out = torch.full((ctx.n_tokens, nq * dim), 5.0, dtype=BF16, device="cuda")
                ops.attention_kv4(qkv, lane, ctx, out, nq, nkv, dim, window=window, sink=sink)
                _near(out[:n].double().reshape(want.shape), want, tol)
                assert (out[n:] == 5).all()
                monkeypatch.undo()


def test_scores_far_apart():
    """Keys whose scores differ by hundreds: the maximum moves late, early keys vanish."""
    from nanospec_b200 import ops
    for dtype, lens in ((BF16, [(400, 1)]), (F32, [(400, 1)]), (BF16, [(300, 40)]), (BF16, [(300, 3)])):
        ctx, lane, qkv = step(lens, 16, 1, 128, dtype, 2)
        k, v = fill(ctx, lane, 2, 1, 128, dtype, size=8.0)
        qkv *= 8
        out = torch.empty((ctx.n_tokens, 256), dtype=dtype, device="cuda")
        ops.attention_kv4(qkv, lane, ctx, out, 2, 1, 128, 1.0)
        want, tol8, tol32 = attend(qkv[:, :256], k, v, ctx, 2, 1.0)
        tol = (tol32 if dtype == F32 else tol8) + want.abs() * 1.01 * half_step(dtype)
        _near(out, want, tol)


def test_rows_and_outputs_with_strides():
    from nanospec_b200 import ops
    for lens in ([(50, 1), (8, 1)], [(30, 4)], [(10, 60)]):
        ctx, lane, qkv = step(lens, 16, 2, 64, BF16, 4)
        fill(ctx, lane, 4, 2, 64)
        want = torch.empty((ctx.n_tokens, 256), dtype=BF16, device="cuda")
        ops.attention_kv4(qkv, lane, ctx, want, 4, 2, 64)
        for off, gap in ((0, 3), (1, 0), (2, 6), (8, 8)):
            wide = torch.zeros((ctx.n_tokens, off + 256 + gap), dtype=BF16, device="cuda")
            wide[:, off: off + 256] = qkv[:, :256]
            buf = torch.full((ctx.n_tokens, off + 256 + gap), 3.0, dtype=BF16, device="cuda")
            ops.attention_kv4(wide[:, off: off + 256], lane, ctx, buf[:, off: off + 256], 4, 2, 64)
            got = buf[:, off: off + 256]
            # another kernel may take rows off 16-byte boundaries: the weights' rounding, not more
            k, v = ops.kv4_read(lane, everything(ctx).positions, everything(ctx).token_req, 2, 64)
            y, tol8, _ = attend(qkv[:, :256], k.double(), v.double(), ctx, 4, 0.125)
            _near(got, y, tol8 + y.abs() * 1.01 * half_step(BF16))
            assert (buf[:, :off] == 3).all() and (buf[:, off + 256:] == 3).all()


def test_cache_refusals():
    from nanospec_b200 import ops
    from nanospec_b200.ops import KernelError
    ctx, lane, qkv = step([(5, 2)], 16, 2, 64, BF16, 4)
    out = torch.empty((2, 256), dtype=BF16, device="cuda")
    other = lambda o, **k: type(o)(**{**vars(o), **k})  # noqa: E731
    store = lambda qkv=qkv, ctx=ctx, lane=lane, nq=4, nkv=2, dim=64, f=None, q_out=None: ops.kv4_store(qkv, ctx, lane, nq, nkv, dim, f, q_out)  # noqa: E731
    attn = lambda qkv=qkv, ctx=ctx, lane=lane, out=out, nq=4, nkv=2, dim=64, **k: ops.attention_kv4(qkv, lane, ctx, out, nq, nkv, dim, **k)  # noqa: E731
    bad = [
        lambda: store(qkv.half()), lambda: store(qkv[:, :-64]), lambda: store(dim=48), lambda: store(nkv=1), lambda: store(qkv.cpu()),
        lambda: store(lane=other(lane, k=lane.k.float())), lambda: store(lane=other(lane, k=lane.k[:, :, :-4])), lambda: store(lane=other(lane, page_size=8)),
        lambda: store(lane=other(lane, block_table=lane.block_table.long())), lambda: store(ctx=other(ctx, positions=ctx.positions.long())),
        lambda: store(ctx=other(ctx, token_req=ctx.token_req[:1])), lambda: store(f=torch.ones(33, device="cuda")),
        lambda: store(f=torch.ones(32, device="cuda", dtype=F64)), lambda: store(q_out=torch.empty((2, 255), dtype=BF16, device="cuda")),
        lambda: store(q_out=torch.empty((2, 256), device="cuda")), lambda: store(q_out=torch.empty((2, 257), dtype=BF16, device="cuda")[:, 1:]),
        lambda: store(torch.empty((2, 513), dtype=BF16, device="cuda")[:, 1:]),
        lambda: attn(qkv.half()), lambda: attn(out=out.float()), lambda: attn(out=out[:, :-1]), lambda: attn(nq=3), lambda: attn(window=-1),
        lambda: attn(qkv[:, :200]), lambda: attn(sink=torch.zeros(3, device="cuda")), lambda: attn(sink=torch.zeros(4, device="cuda", dtype=BF16)),
        lambda: attn(lane=other(lane, v=lane.v.int())), lambda: attn(dim=288), lambda: attn(out=out.cpu()), lambda: attn(ctx=other(ctx, positions=ctx.positions[:1])),
        lambda: attn(ctx=other(ctx, kv_lens=[33], extras={})), lambda: attn(lane=other(lane, block_table=lane.block_table[:0])),
        lambda: ops.kv4_read(lane, ctx.positions.long(), ctx.token_req, 2, 64), lambda: ops.kv4_read(lane, ctx.positions, ctx.token_req[:1], 2, 64),
        lambda: ops.kv4_pages(3, 2, 0, 64), lambda: ops.kv4_pages(3, 2, 16, 288), lambda: ops.kv4_pages(3, 2, 16, 40),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            print("not refused:", i)
    none = other(ctx, positions=ctx.positions[:0], token_req=ctx.token_req[:0], q_lens=[], kv_lens=[], extras={}, n_tokens=0)
    assert store(qkv[:0], ctx=none).shape == (0, 512) and attn(qkv[:0], ctx=none, out=out[:0]).shape == (0, 256)


# ---- streams, graphs, a run of them together ----------------------------------------------------------------------------------------------
def _block(x, w_qkv, w_out, ctx, lane, nq, nkv, dim, f):
    """An attention block in fewer bits: x -> qkv -> rotation and store -> attention -> output projection."""
    from nanospec_b200 import ops
    n = x.shape[0]
    qkv = torch.empty((n, w_qkv.shape[0]), dtype=x.dtype, device="cuda")
    o = torch.zeros((n, nq * dim), dtype=x.dtype, device="cuda")
    y = torch.empty((n, w_out.shape[0]), dtype=x.dtype, device="cuda")
    ops.linear_i8(x, w_qkv, qkv)
    ops.kv4_store(qkv, ctx, lane, nq, nkv, dim, f)
    ops.attention_kv4(qkv, lane, ctx, o, nq, nkv, dim)
    return ops.linear_i8(o, w_out, y), qkv, o


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_run_of_them_together(dtype):
    """A prompt in two portions, then tokens one by one: each output against the plain statement on the operators' own intermediate results."""
    from nanospec_b200 import ops
    nq, nkv, dim, width = 8, 2, 64, 512
    w_qkv, w_out = ops.quantize_rows(_rand((nq + 2 * nkv) * dim, width, seed=1) * width ** -0.5), ops.quantize_rows(_rand(width, nq * dim, seed=2) * 0.04)
    f = _inv_freq(dim)
    whole, lane, _ = step([(0, 140)], 16, nkv, dim, dtype, nq)
    xs = _rand(140, width, seed=3, dtype=dtype)
    kept_k, kept_v = [], []
    for held, n in ((0, 60), (60, 70), (130, 3), *((p, 1) for p in range(133, 140))):
        ctx, _, _ = step([(held, n)], 16, nkv, dim, dtype, nq)
        x = xs[held: held + n]
        xq = ops.quantize_rows(x)
        proj, tol = _product(xq, w_qkv, dtype)
        before = torch.empty((n, w_qkv.shape[0]), dtype=dtype, device="cuda")
        ops.linear_i8(x, w_qkv, before)
        _near(before, proj, tol)
        y, qkv, o = _block(x, w_qkv, w_out, ctx, lane, nq, nkv, dim, f)
        heads = before.reshape(n, -1, dim)
        kept_k.append(held4(in_type(rotated(heads[:, nq: nq + nkv], ctx.positions, f), dtype)))
        kept_v.append(held4(heads[:, nq + nkv:].double()))
        want, tol8, tol32 = attend(qkv[:, : nq * dim], torch.cat(kept_k), torch.cat(kept_v), ctx, nq, dim ** -0.5)
        _near(o, want, (tol32 if dtype == F32 else tol8) + want.abs() * 1.01 * half_step(dtype))
        last, tol = _product(ops.quantize_rows(o), w_out, dtype)
        _near(y, last, tol)


def test_captured_and_replayed_on_another_stream():
    from nanospec_b200 import ops
    nq, nkv, dim, width = 8, 2, 128, 1024
    w_qkv, w_out = ops.quantize_rows(_rand((nq + 2 * nkv) * dim, width, seed=1) * width ** -0.5), ops.quantize_rows(_rand(width, nq * dim, seed=2) * 0.04)
    f = _inv_freq(dim)
    lens = [(300, 1), (17, 1), (1200, 1)]
    ctx, lane, _ = step(lens, 16, nkv, dim, BF16, nq)
    fill(ctx, lane, nq, nkv, dim)
    x = _rand(3, width, seed=3, dtype=BF16)
    eager = [t.clone() for t in _block(x, w_qkv, w_out, ctx, lane, nq, nkv, dim, f)]
    ctx.extras = {"graph": True}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(x, w_qkv, w_out, ctx, lane, nq, nkv, dim, f)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same step: nothing that they share is scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_block(x, w_qkv, w_out, ctx, lane, nq, nkv, dim, f))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out in outs:
        # (the lengths are not known when a graph is captured, so keys may be divided otherwise: the weights' rounding, not more)
        k, v = ops.kv4_read(lane, everything(ctx).positions, everything(ctx).token_req, nkv, dim)
        want, tol8, _ = attend(out[1][:, : nq * dim], k.double(), v.double(), ctx, nq, dim ** -0.5)
        assert torch.equal(out[1], eager[1])
        _near(out[2], want, tol8 + want.abs() * 1.01 * half_step(BF16))
        assert torch.equal(out[2], outs[0][2]) and torch.equal(out[0], outs[0][0])
    # the same graph with the positions moved on: what is read at replay is what counts
    ctx.positions.sub_(4)
    graphs[0].replay()
    torch.cuda.synchronize()
    moved = type(ctx)(**{**vars(ctx), "kv_lens": [n - 4 for n in ctx.kv_lens], "extras": {}})
    k, v = ops.kv4_read(lane, everything(moved).positions, everything(moved).token_req, nkv, dim)
    want, tol8, _ = attend(outs[0][1][:, : nq * dim], k.double(), v.double(), moved, nq, dim ** -0.5)
    _near(outs[0][2], want, tol8 + want.abs() * 1.01 * half_step(BF16))


def test_pages_far_into_a_large_pool():
    """Addresses beyond 32 bits: a pool of more than 4 GB, its last pages in use."""
    from nanospec_b200 import ops
    nkv, dim, page = 8, 128, 64
    size = ops.kv4_block_bytes(page, dim) * nkv
    pages = (1 << 32) // size + 200
    ctx, lane, qkv = step([(150, 1), (20, 40)], page, nkv, dim, BF16, 8)
    lane.k, lane.v = (torch.zeros((pages, nkv, size // nkv), dtype=torch.uint8, device="cuda") for _ in range(2))
    lane.block_table = torch.where(lane.block_table >= 0, pages - lane.block_table, lane.block_table).contiguous()
    k, v = fill(ctx, lane, 8, nkv, dim)
    out = torch.empty((ctx.n_tokens, 8 * dim), dtype=BF16, device="cuda")
    ops.attention_kv4(qkv, lane, ctx, out, 8, nkv, dim)
    want, tol8, _ = attend(qkv[:, : 8 * dim], k, v, ctx, 8, dim ** -0.5)
    _near(out, want, tol8 + want.abs() * 1.01 * half_step(BF16))
    assert k.abs().sum() > 0


# ---- values at the end of bfloat16's range ------------------------------------------------------------------------------------------------
BIG = torch.finfo(BF16).max
BEYOND = 0.148  # features from here to 1 times the largest: S and B are finite, what the largest feature's code stands for rounds beyond it


def test_the_borders_of_a_group_at_the_end_of_the_range():
    """What the tests below are about, in 64 bits."""
    for at, beyond in ((BEYOND, True), (0.5, False)):
        lo = torch.tensor([at * BIG]).bfloat16().double()
        S = to_bf16((BIG - lo) * 16 / 15)
        B = to_bf16(lo - S)
        assert S < BIG and B.abs() < BIG and bool(to_bf16(B + S * 31 / 16) > BIG) == beyond


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_store_of_a_group_whose_largest_code_is_beyond_the_range(dim, dtype):
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(0, 4)], 16, 2, dim, dtype, 1)
    x = qkv.reshape(4, 5, dim)
    ramp = torch.linspace(BEYOND, 1.0, 32, device="cuda").double() * BIG
    ramp[0], ramp[-1] = torch.tensor(BEYOND * BIG).bfloat16().double(), BIG
    x[1, 2, :32] = ramp.to(dtype).clamp(max=BIG)            # a key of head 1
    x[2, 3, dim - 32:] = ramp.to(dtype).clamp(max=BIG)      # a value of head 0
    half = torch.linspace(0.5, 1.0, 32, device="cuda").double() * BIG
    x[3, 1, :32] = half.to(dtype).clamp(max=BIG)            # (within the range: held as it is)
    ops.kv4_store(qkv, ctx, lane, 1, 2, dim)
    k, v = ops.kv4_read(lane, ctx.positions, ctx.token_req, 2, dim)
    assert v.isfinite().all()
    nan = k.isnan()
    assert nan.all(-1).tolist() == [[False, False], [False, True], [True, False], [False, False]] and torch.equal(nan.any(-1), nan.all(-1))
    assert (k.isfinite() | nan).all() and (v[2, 0, -32:] == 0).all()
    assert torch.equal(k[3, 0].double(), held4(x[3, 1].double()))


@pytest.mark.parametrize("tokens", [3, 100])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_value_beyond_the_range_reaches_only_those_that_see_it(tokens, dim):
    """A few tokens in one tile, and a portion: the rows before the token's position meet a weight of zero for it."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(40, tokens)], 16, 2, dim, BF16, 4)
    fill(ctx, lane, 4, 2, dim)
    key = 40 + tokens - 1
    one = type(ctx)(**{**vars(ctx), "positions": ctx.positions[-1:].clone(), "token_req": ctx.token_req[-1:].clone()})
    bad = _rand(1, 8 * dim, dtype=BF16)
    bad[0, 7 * dim: 7 * dim + 32] = torch.linspace(BEYOND, 1.0, 32).double().mul(BIG).bfloat16().cuda().clamp(max=BIG)  # the value of kv head 1
    ops.kv4_store(bad, one, lane, 4, 2, dim)
    out = torch.empty((ctx.n_tokens, 4 * dim), dtype=BF16, device="cuda")
    ops.attention_kv4(qkv, lane, ctx, out, 4, 2, dim)
    sees = (ctx.positions[:, None] >= key).expand(-1, 2 * dim)
    assert torch.equal(out[:, 2 * dim:].isnan(), sees) and out[:, : 2 * dim].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_codes_of_features_further_apart_from_the_base_than_float_reaches(dtype):
    """x - B is up to 1.95 S: beyond float's range for the largest S."""
    from nanospec_b200 import ops
    lens = [(0, 6)]
    ctx, lane, qkv = step(lens, 16, 1, 64, dtype, 1)
    v = qkv[:, 128:]
    for i, (lo, hi) in enumerate(((-1.3e38, 0.575e38), (-1.0e38, 2.0e38), (0.0, 3.0e38), (-0.2e38, 2.9e38), (1.0e38, 1.9e38))):
        v[i, :32] = torch.linspace(lo, hi, 32).to(dtype).cuda()
        v[i, 32:] = torch.linspace(lo, hi, 32).flip(0).to(dtype).cuda()
    v[2, 5], v[2, 40] = 1e-30, -1e-38 if dtype == BF16 else -1e-44
    g = v.double().reshape(6, 2, 32)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    S = to_bf16((hi - lo) * 16 / 15)
    B = to_bf16(lo - S)
    beyond = (S > BIG) | (B.abs() > BIG) | (to_bf16(B + S * 31 / 16).abs() > BIG)  # groups that count as not finite: zeros
    assert beyond[..., 0].tolist() == [[False, False], [True, True], [False, False], [True, True], [False, False], [False, False]]
    want = held4(v.double().unsqueeze(1)).masked_fill(beyond.expand(-1, -1, 32).reshape(6, 1, 64), 0.0)
    ops.kv4_store(qkv, ctx, lane, 1, 1, 64)
    _, got = ops.kv4_read(lane, ctx.positions, ctx.token_req, 1, 64)
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs", [None, 0, 8])
def test_features_of_q_that_are_not_rotated_stay_as_they_are(pairs, dtype):
    """Also beside a partner that is not finite, and to a buffer of its own."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(7, 3)], 16, 1, 64, dtype, 2)
    f = None if pairs is None else _inv_freq(64, pairs=pairs)
    n = pairs or 0
    x = qkv[:, :128].reshape(3, 2, 64)
    x[0, 0, 20], x[1, 1, 31], x[2, 0, 32 + 9], x[2, 1, 63] = math.inf, math.nan, -math.inf, math.nan
    q = x.clone()
    still = torch.tensor([j % 32 >= n for j in range(64)], device="cuda")
    out = ops.kv4_store(qkv, ctx, lane, 2, 1, 64, f, q_out=torch.empty((3, 128), dtype=dtype, device="cuda"))
    for got in (out, ops.kv4_store(qkv, ctx, lane, 2, 1, 64, f)[:, :128]):
        got = got.reshape(3, 2, 64)
        assert torch.equal(got[..., still].isnan(), q[..., still].isnan())
        assert torch.equal(got[..., still].nan_to_num(0.25), q[..., still].nan_to_num(0.25)) and got[..., ~still].isfinite().all()


@pytest.mark.parametrize("page", [8, 5])
def test_reading_where_the_cache_holds_nothing(page):
    """Pages given back, positions and requests that the table does not have, entries beyond the pool: zeros, and nothing of the pool's surroundings is read."""
    from nanospec_b200 import ops
    ctx, lane, _ = step([(40, 1), (23, 1)], page, 2, 64)
    held, _ = fill(ctx, lane, 1, 2, 64)
    lane.block_table[0, :2] = -1
    lane.block_table[1, 1] = lane.k.shape[0]
    rows, columns = lane.block_table.shape
    asked = [(0, 0, False), (0, 2 * page - 1, False), (0, 2 * page, True), (0, 40, True), (1, page, False), (1, 2, True), (1, 23, True), (rows, 0, False), (1 << 30, 3, False),
             (0, columns * page, False), (0, 2 ** 31 - 1, False), (1, -1, False), (1, -2 ** 31, False), (-1, 5, False)]
    i32 = lambda i: torch.tensor([a[i] for a in asked], dtype=torch.int32, device="cuda")  # noqa: E731
    for k, v in (ops.kv4_read(lane, i32(1), i32(0), 2, 64), ops.kv4_read(lane, i32(1).repeat(400), i32(0).repeat(400), 2, 64)):
        for n, (req, pos, there) in enumerate(asked):
            assert torch.equal(k[n].double(), held[41 * req + pos]) if there else not k[n].any() and not v[n].any()


@pytest.mark.parametrize("lens", [[(9, 1), (900, 1), (100, 1)], [(20, 1), (200, 3), (40, 90)]])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F32)])
def test_a_step_whose_calls_follow_other_kernels_on_their_streams(lens, dim, dtype):
    """The lists are late, and a kernel stands ready on each later stream that the attention's launch could overlap."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, 16, 2, dim, dtype, 8)
    fill(ctx, lane, 8, 2, dim, dtype)
    want = ops.attention_kv4(qkv, lane, ctx, torch.zeros((ctx.n_tokens, 8 * dim), dtype=dtype, device="cuda"), 8, 2, dim)
    x, w = _rand(64, 1024, dtype=BF16), ops.quantize_rows(_rand(1024, 1024, seed=2))
    outs, products = [torch.zeros_like(want) for _ in range(3)], [torch.empty((64, 1024), dtype=BF16, device="cuda") for _ in range(3)]
    ctx.extras = {}
    torch.cuda.synchronize()
    for i, (out, product, s) in enumerate(zip(outs, products, [torch.cuda.Stream() for _ in outs])):
        with torch.cuda.stream(s):
            if i == 0:
                torch.cuda._sleep(20_000_000)
            ops.linear_i8(x, w, product)
            ops.attention_kv4(qkv, lane, ctx, out, 8, 2, dim)
            ops.linear_i8(x, w, product)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs) and all(torch.equal(p, products[0]) for p in products)
    ops.check_kernel_errors()


@pytest.mark.parametrize("lens", [[(9, 1), (900, 1), (100, 1)], [(5000, 1)], [(30, 5), (2000, 3)], [(20, 1), (200, 3), (40, 90)]])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F32)])
def test_a_step_captured_without_its_mark(lens, dim, dtype):
    """Its graph finds the step's lists whatever becomes of the step."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, 16, 2, dim, dtype, 8)
    fill(ctx, lane, 8, 2, dim, dtype)
    out = torch.zeros((ctx.n_tokens, 8 * dim), dtype=dtype, device="cuda")
    call = lambda: ops.attention_kv4(qkv, lane, ctx, out, 8, 2, dim)  # noqa: E731
    want = call().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    ctx.extras = {}
    other = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 2, 3, 5, 8, 40, 130, 500, 2000) for _ in range(8)]  # what the lists would have made room for
    call(), out.zero_()  # (the step anew, with lists of its own)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not any(o.any() for o in other)


def test_a_capture_waits_for_lists_that_are_on_their_way():
    from nanospec_b200 import ops
    ctx, lane, qkv = step([(9, 1), (900, 1), (40, 3)], 16, 2, 128, BF16, 8)
    fill(ctx, lane, 8, 2, 128)
    out = torch.zeros((ctx.n_tokens, 1024), dtype=BF16, device="cuda")
    call = lambda: ops.attention_kv4(qkv, lane, ctx, out, 8, 2, 128)  # noqa: E731
    want = call().clone()
    torch.cuda.synchronize()
    ctx.extras = {}
    first, second, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(first):
        torch.cuda._sleep(20_000_000)
        call()
    plan = next(iter(ctx.extras.values()))
    with torch.cuda.stream(second):
        graph.capture_begin()
        call()
        graph.capture_end()
    assert plan["ready"].query()
    first.synchronize()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_a_first_call_in_a_capture_is_refused():
    from nanospec_b200 import ops
    from nanospec_b200.ops import KernelError
    ctx, lane, qkv = step([(9, 1), (900, 1)], 16, 2, 128, BF16, 8)
    fill(ctx, lane, 8, 2, 128)
    out, x = torch.zeros((2, 1024), dtype=BF16, device="cuda"), torch.zeros(3, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # (and the capture goes on)
        with pytest.raises(KernelError, match="captured"):
            ops.attention_kv4(qkv, lane, ctx, out, 8, 2, 128)
        x += 1
    graph.replay()
    assert (x == 1).all() and not any(k[0] == "kv4_plan" for k in ctx.extras)


@pytest.mark.parametrize("nq,nkv,dim,page,dtype", [(32, 8, 128, 16, BF16), (16, 2, 64, 8, BF16), (6, 2, 96, 16, BF16), (4, 2, 64, 16, F32)])
@pytest.mark.parametrize("lens,window,padding", [([(60, 0), (500, 1), (0, 0), (90, 3), (33, 0), (100, 200), (3, 1), (7, 0)], 0, 2),
                                                 ([(60, 0), (0, 1), (31, 0)], 20, 0), ([(60, 0), (40, 0)], 0, 1)])
def test_requests_that_bring_nothing(lens, window, padding, nq, nkv, dim, page, dtype):
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, page, nkv, dim, dtype, nq, padding=padding)
    lane.k.fill_(255), lane.v.fill_(255)
    k, v = fill(ctx, lane, nq, nkv, dim, dtype)
    n = ctx.n_tokens - padding
    out = torch.full((ctx.n_tokens, nq * dim), 5.0, dtype=dtype, device="cuda")
    ops.attention_kv4(qkv, lane, ctx, out, nq, nkv, dim, window=window)
    held = [(a, kv) for a, kv in zip(ctx.q_lens, ctx.kv_lens) if kv]  # (the plain statement takes requests that hold something)
    at = type(ctx)(**{**vars(ctx), "q_lens": [a for a, _ in held], "kv_lens": [kv for _, kv in held]})
    want, tol8, tol32 = attend(qkv[:n, : nq * dim], k, v, at, nq, dim ** -0.5, window)
    if n:
        _near(out[:n], want, (tol32 if dtype == F32 else tol8) + want.abs() * 1.01 * half_step(dtype))
    assert (out[n:] == 5).all()


@pytest.mark.parametrize("window", [0, 40, 100000])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, BF16), (96, BF16), (64, F32)])
def test_captured_steps_with_windows_and_sinks(window, dim, dtype):
    from nanospec_b200 import ops
    nq, nkv = 8, 2
    ctx, lane, qkv = step([(2900, 1), (17, 1), (0, 1), (300, 1)], 16, nkv, dim, dtype, nq, padding=1)
    k, v = fill(ctx, lane, nq, nkv, dim, dtype)
    sink = _rand(nq, seed=6)
    ctx.extras = {"graph": True}
    out = torch.full((5, nq * dim), 5.0, dtype=dtype, device="cuda")
    call = lambda: ops.attention_kv4(qkv, lane, ctx, out, nq, nkv, dim, window=window, sink=sink)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for shift in (0, 3):
        ctx.positions[:2] -= shift  # read at replay
        out[:4] = 0
        graph.replay()
        at = type(ctx)(**{**vars(ctx), "kv_lens": [n - (shift if i < 2 else 0) for i, n in enumerate(ctx.kv_lens)], "extras": {}})
        rows = torch.cat([torch.arange(n, device="cuda") + sum(ctx.kv_lens[:i]) for i, n in enumerate(at.kv_lens)])
        want, tol8, tol32 = attend(qkv[:4, : nq * dim], k[rows], v[rows], at, nq, dim ** -0.5, window, sink)
        tol = (tol32 if dtype == F32 else tol8) + want.abs() * 1.01 * half_step(dtype)
        _near(out[:4], want, tol)
        assert (out[4] == 5).all()


@pytest.mark.parametrize("lens", [[(300, 1), (2000, 1), (0, 1)], [(200, 3), (31, 6)], [(500, 1), (0, 200), (90, 3), (1200, 300)]])
@pytest.mark.parametrize("nq,nkv,dim,page,dtype", [(32, 8, 128, 16, BF16), (8, 2, 64, 8, BF16), (4, 1, 256, 16, BF16), (6, 2, 96, 16, BF16), (4, 2, 64, 16, F32)])
@pytest.mark.parametrize("window", [0, 150])
def test_weights_in_more_than_eight_bits(lens, nq, nkv, dim, page, dtype, window):
    """In float, or, in portions, as two bfloat16: the first is off by 2^-8 of the weight, which the second holds but for 2^-8 of itself."""
    from nanospec_b200 import ops
    ctx, lane, qkv = step(lens, page, nkv, dim, dtype, nq, padding=1)
    lane.k.fill_(255), lane.v.fill_(255)
    k, v = fill(ctx, lane, nq, nkv, dim, dtype)
    n, sink = ctx.n_tokens - 1, _rand(nq, seed=8)
    want, tol8, tol32 = attend(qkv[:n, : nq * dim], k, v, ctx, nq, dim ** -0.5, window, sink)
    rounding = want.abs() * 1.01 * half_step(dtype)
    for wide in (True, False, True):  # (the two forms of a step do not meet in its plan)
        out = torch.full((ctx.n_tokens, nq * dim), 5.0, dtype=dtype, device="cuda")
        ops.attention_kv4(qkv, lane, ctx, out, nq, nkv, dim, window=window, sink=sink, wide_weights=wide)
        _near(out[:n], want, (tol32 + (tol8 - tol32) * (2.0 ** -8 if wide else 1.0)) + rounding)
        assert (out[n:] == 5).all()
