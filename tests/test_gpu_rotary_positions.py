"""cos | sin rows, rotation of q and k in tensors of their own, and the MLA prologue, against 64-bit references."""
import math

import pytest
import torch

from xllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------
# frequencies and rows

def test_frequencies():
    inv, factor = ops.rope_frequencies(128, device="cpu")
    i = torch.arange(64, dtype=torch.float64)
    assert torch.allclose(inv, 10000.0 ** (-i / 64), rtol=1e-15, atol=0) and factor == 1.0
    lin, _ = ops.rope_frequencies(128, scaling=ops.RopeScaling("linear", factor=8.0), device="cpu")
    assert torch.allclose(lin, inv / 8, rtol=1e-15, atol=0)
    dyn = ops.RopeScaling("dynamic", factor=2.0, original_max_position=4096)
    assert torch.equal(ops.rope_frequencies(128, scaling=dyn, seq_len=4096, device="cpu")[0], inv)
    far, _ = ops.rope_frequencies(128, scaling=dyn, seq_len=8192, device="cpu")
    assert torch.allclose(far, (10000.0 * 3 ** (128 / 126)) ** (-i / 64), rtol=1e-14, atol=0)
    l3, _ = ops.rope_frequencies(128, base=500000.0, device="cpu",
                                 scaling=ops.RopeScaling("llama3", factor=8.0, original_max_position=8192))
    plain, _ = ops.rope_frequencies(128, base=500000.0, device="cpu")
    turns = 8192 * plain / (2 * math.pi)
    assert torch.allclose(l3[turns > 4], plain[turns > 4], rtol=1e-15, atol=0)
    assert torch.allclose(l3[turns < 1], plain[turns < 1] / 8, rtol=1e-15, atol=0)
    yarn = ops.RopeScaling("yarn", factor=40.0, original_max_position=4096)
    y, m = ops.rope_frequencies(64, scaling=yarn, device="cpu")
    p, _ = ops.rope_frequencies(64, device="cpu")
    assert y[0] == p[0] and torch.allclose(y[-1], p[-1] / 40, rtol=1e-14, atol=0) and abs(m - 1 - 0.1 * math.log(40)) < 1e-15
    both = ops.RopeScaling("yarn", factor=40.0, original_max_position=4096, mscale=1.0, mscale_all_dim=1.0)
    assert ops.rope_frequencies(64, scaling=both, device="cpu")[1] == 1.0
    for bad in (dict(kind="nope"), dict(kind="linear", factor=0.5), dict(kind="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(64, scaling=ops.RopeScaling(**bad), device="cpu")
    for dim in (0, 7):
        with pytest.raises(ValueError):
            ops.rope_frequencies(dim, device="cpu")


def check_rows(rows, inv, pos, factor):
    """One rounding of the exact value; the angle's own error in 64 bits (2^-53 of it) and the polynomials' are below 1e-9
    for angles up to 2^22."""
    angle = pos.double().cpu()[:, None] * inv.cpu()
    want = torch.cat([angle.cos(), angle.sin()], 1) * factor
    err = (rows.double().cpu() - want).abs()
    tiny = torch.finfo(rows.dtype).smallest_normal * torch.finfo(rows.dtype).eps / 2
    assert (err <= half_step(rows.dtype) * want.abs() + 1e-9 + tiny).all(), err.max()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("dim", [2, 6, 32, 40, 64, 96, 128, 256])
def test_rows_of_positions_and_of_a_range(dtype, dim):
    inv, factor = ops.rope_frequencies(dim, scaling=ops.RopeScaling("yarn", factor=4.0, original_max_position=2048), device=DEV)
    for n in (1, 77, 1000):
        pos = torch.randint(0, 1 << 22, (n,), generator=torch.Generator().manual_seed(n)).to(DEV)
        check_rows(ops.build_cos_sin_cache(inv, position_ids=pos, attention_factor=factor, dtype=dtype), inv, pos, factor)
        first = 12345
        got = ops.build_cos_sin_cache(inv, n, first_position=first, attention_factor=factor, dtype=dtype)
        check_rows(got, inv, torch.arange(first, first + n), factor)


@pytest.mark.parametrize("dtype,dim,n", [(FP32, 96, 21901), (FP32, 256, 9001), (FP32, 64, 33000), (BF16, 96, 50001),
                                         (FP16, 128, 33001), (BF16, 32, 131101), (FP32, 2048, 1101), (FP32, 4096, 600)])
def test_long_ranges(dtype, dim, n):
    """Ranges whose rows are made from one another: the same bound; the row count leaves lines of the last pass over."""
    inv, factor = ops.rope_frequencies(dim, scaling=ops.RopeScaling("yarn", factor=4.0, original_max_position=2048), device=DEV)
    for first in (0, 4_000_000):
        buf = torch.full((n + 2, dim), 7.0, dtype=dtype, device=DEV)
        got = ops.build_cos_sin_cache(inv, n, first_position=first, attention_factor=factor, dtype=dtype, out=buf[1:n + 1])
        check_rows(got, inv, torch.arange(first, first + n), factor)
        assert (buf[0] == 7).all() and (buf[n + 1] == 7).all()


def test_rows_into_a_given_tensor_and_far_positions():
    inv, _ = ops.rope_frequencies(64, device=DEV)
    buf = torch.full((12, 64), 7.0, device=DEV)
    out = ops.build_cos_sin_cache(inv, 10, out=buf[1:11])
    check_rows(out, inv, torch.arange(10), 1.0)
    assert (buf[0] == 7).all() and (buf[11] == 7).all()
    # every position gives a point of the unit circle, negative and very large ones too
    pos = torch.tensor([-1, -12345, 2 ** 40, 2 ** 48 + 1], device=DEV)
    rows = ops.build_cos_sin_cache(inv, position_ids=pos).double()
    assert ((rows[:, :32] ** 2 + rows[:, 32:] ** 2 - 1).abs() < 1e-6).all()
    assert ops.build_cos_sin_cache(inv, position_ids=pos[:0]).shape == (0, 64)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("dim,n", [(2, 300), (6, 3001), (32, 9001), (40, 7003), (96, 3001), (128, 33001), (256, 9001), (1024, 1500),
                                   (2048, 1101)])
@pytest.mark.parametrize("first", [0, 12345, 2 ** 22 - 5, 2 ** 40 + 3])
def test_a_position_has_one_row(dtype, dim, n, first):
    """The same bits for a position whichever way its row is asked for: in a long range, in ranges of a few rows that begin
    anywhere, in a list, and into memory off the 16-byte boundary."""
    inv, factor = ops.rope_frequencies(dim, scaling=ops.RopeScaling("yarn", factor=4.0, original_max_position=2048), device=DEV)
    kw = dict(attention_factor=factor, dtype=dtype)
    whole = ops.build_cos_sin_cache(inv, n, first_position=first, **kw)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(n)).to(DEV)
    assert torch.equal(ops.build_cos_sin_cache(inv, position_ids=first + order, **kw), whole[order])
    few = order[:50].contiguous()
    assert torch.equal(ops.build_cos_sin_cache(inv, position_ids=first + few, **kw), whole[few])
    for at, m in ((0, 1), (0, 9), (1, 8), (7, 2), (n // 2 + 3, 13), (n - 1, 1), (3, n - 5)):
        assert torch.equal(ops.build_cos_sin_cache(inv, m, first_position=first + at, **kw), whole[at:at + m]), (at, m)
    odd = torch.empty(n * dim + 1, dtype=dtype, device=DEV)[1:].view(n, dim)
    assert torch.equal(ops.build_cos_sin_cache(inv, n, first_position=first, attention_factor=factor, out=odd), whole)


# ------------------------------------------------------------------------------------------
# rotation

def rotate64(x, table, pos, offset, interleave, inverse):
    """(result, bound on the fp32 arithmetic) of x [T, H, D] in 64 bits."""
    R = table.shape[1]
    ok = (pos >= 0) & (pos < table.shape[0])
    rows = table.double()[pos.clamp(0, table.shape[0] - 1)]
    c = torch.where(ok[:, None], rows[:, :R // 2], 1.0)[:, None]
    s = torch.where(ok[:, None], rows[:, R // 2:], 0.0)[:, None] * (-1 if inverse else 1)
    y, bound = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    part = slice(offset, offset + R)
    p = y[..., part]
    ia = slice(0, R, 2) if interleave else slice(0, R // 2)
    ib = slice(1, R, 2) if interleave else slice(R // 2, R)
    a, b = p[..., ia].clone(), p[..., ib].clone()
    y[..., part][..., ia] = a * c - b * s
    y[..., part][..., ib] = b * c + a * s
    # a product rounded, then a fused multiply-add rounded: two roundings of 2^-24 of terms up to |a c| + |b s|
    bound[..., part][..., ia] = 2.0 ** -23 * (a * c).abs() + 2.0 ** -23 * (b * s).abs()
    bound[..., part][..., ib] = 2.0 ** -23 * (b * c).abs() + 2.0 ** -23 * (a * s).abs()
    return y, bound


def assert_rotated(got, x, table, pos, offset, interleave, inverse):
    want, bound = rotate64(x, table, pos, offset, interleave, inverse)
    err = (got.double() - want).abs()
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    assert (err <= half_step(x.dtype) * (want.abs() + bound) + bound + tiny).all(), err.max()
    R = table.shape[1]
    assert torch.equal(got[..., :offset], x[..., :offset]) and torch.equal(got[..., offset + R:], x[..., offset + R:])


def table_of(rows, R, dtype):
    inv, _ = ops.rope_frequencies(R, device=DEV)
    return ops.build_cos_sin_cache(inv, rows, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,Hq,Hk,D,R,off", [
    (1, 1, 1, 64, 64, 0), (1, 32, 8, 128, 128, 0), (5, 7, 3, 96, 32, 64), (64, 32, 8, 128, 128, 0), (33, 5, 0, 80, 32, 48),
    (17, 6, 2, 256, 64, 192), (3, 2, 1, 10, 6, 4), (9, 3, 3, 40, 20, 0), (2, 1, 1, 4, 2, 1), (130, 64, 8, 128, 64, 32),
    (700, 24, 8, 192, 64, 128)])
@pytest.mark.parametrize("interleave", [False, True])
def test_rotation(dtype, T, Hq, Hk, D, R, off, interleave):
    gen = torch.Generator(device=DEV).manual_seed(T + D)
    q = torch.randn(T, Hq, D, generator=gen, device=DEV).to(dtype)
    k = torch.randn(T, Hk, D, generator=gen, device=DEV).to(dtype) if Hk else None
    table = table_of(500, R, FP32 if D != 96 else BF16)
    pos = torch.randint(-1, 502, (T,), generator=torch.Generator().manual_seed(T)).to(DEV)   # (a few outside the table)
    for inverse in (False, True):
        oq, ok = torch.full_like(q, 9), None if k is None else torch.full_like(k, 9)
        ops.rotary_embedding(pos, q, k, table, interleave=interleave, rotary_offset=off, inverse=inverse, out_query=oq, out_key=ok)
        assert_rotated(oq, q, table, pos, off, interleave, inverse)
        if k is not None:
            assert_rotated(ok, k, table, pos, off, interleave, inverse)
        iq, ik = q.clone(), None if k is None else k.clone()
        ops.rotary_embedding(pos, iq, ik, table, interleave=interleave, rotary_offset=off, inverse=inverse)
        assert torch.equal(iq, oq) and (k is None or torch.equal(ik, ok))   # in place: the same bits


@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_strides_slices_and_alignment(interleave, shift):
    """q and k as slices of one buffer, head-major tensors, tensors that start off a 16-byte boundary, one head of a size."""
    T, Hq, Hk, D, R = 21, 6, 2, 64, 32
    table = table_of(64, R, FP32)
    pos = torch.randint(0, 64, (T,), generator=torch.Generator().manual_seed(1)).to(DEV)
    buf = torch.randn(T * (Hq + Hk) * D + 16, device=DEV).to(BF16)
    qkv = buf[shift:shift + T * (Hq + Hk) * D].view(T, (Hq + Hk) * D)
    q, k = qkv[:, :Hq * D].view(T, Hq, D), qkv[:, Hq * D:].view(T, Hk, D)
    want_q, want_k = q.clone(), k.clone()
    ops.rotary_embedding(pos, want_q, want_k, table, interleave=interleave, rotary_offset=16)
    head_major = torch.empty(Hq, T, D, dtype=BF16, device=DEV).transpose(0, 1)
    ok = torch.empty(T, Hk, D + 8, dtype=BF16, device=DEV)[..., :D]
    ops.rotary_embedding(pos, q, k, table, interleave=interleave, rotary_offset=16, out_query=head_major, out_key=ok)
    assert torch.equal(head_major, want_q) and torch.equal(ok, want_k)
    before = buf.clone()
    ops.rotary_embedding(pos, q, k, table, interleave=interleave, rotary_offset=16)   # both slices in place
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(buf[:shift], before[:shift])
    assert torch.equal(buf[shift + T * (Hq + Hk) * D:], before[shift + T * (Hq + Hk) * D:])


@pytest.mark.parametrize("T", [1, 2, 77])
@pytest.mark.parametrize("layout", ["heads", "grouped", "head major"])
def test_results_in_slices_of_one_buffer(T, layout):
    """Results, and operands in place, that interleave in memory without meeting."""
    Hq, D = 4, 64
    Hk = 2 if layout == "heads" else 4
    gen = torch.Generator(device=DEV).manual_seed(T)

    def halves(x):
        if layout == "heads":      # [T, Hq + Hk, D]
            return x[:, :Hq], x[:, Hq:]
        if layout == "grouped":    # [T, H, q | k]
            return x[..., :D], x[..., D:]
        return x[:Hq].transpose(0, 1), x[Hq:].transpose(0, 1)   # [Hq + Hk, T, D]

    shape = {"heads": (T, Hq + Hk, D), "grouped": (T, Hq, 2 * D), "head major": (Hq + Hk, T, D)}[layout]
    x = torch.randn(shape, generator=gen, device=DEV).to(BF16)
    q, k = halves(x)
    pos = torch.arange(T, device=DEV) * 3
    table = ops.build_cos_sin_cache(ops.rope_frequencies(D, device=DEV)[0], 3 * T)
    want_q, want_k = torch.empty_like(q.contiguous()), torch.empty_like(k.contiguous())
    ops.rotary_embedding(pos, q, k, table, out_query=want_q, out_key=want_k)
    oq, ok = halves(torch.full_like(x, 7.0))
    ops.rotary_embedding(pos, q, k, table, out_query=oq, out_key=ok)
    assert torch.equal(oq, want_q) and torch.equal(ok, want_k)
    ops.rotary_embedding(pos, q, k, table)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)


def test_sides_of_their_own_sizes():
    """Queries whose rotated part is the tail of a wide head, keys that are nothing else: the MLA shapes, and out of place
    for one side only."""
    T = 13
    q, k = torch.randn(T, 16, 192, device=DEV).to(BF16)[:, :5], torch.randn(T, 1, 64, device=DEV).to(BF16)
    table, pos = table_of(99, 64, FP32), torch.arange(T, device=DEV) * 7
    out_q = torch.empty(T, 5, 192, dtype=BF16, device=DEV)
    k0 = k.clone()
    ops.rotary_embedding(pos, q, k, table, interleave=True, rotary_offset=128, key_rotary_offset=0, out_query=out_q)
    assert_rotated(out_q, q, table, pos, 128, True, False)
    assert_rotated(k, k0, table, pos, 0, True, False)


def test_gradient_and_inverse():
    """The inverse form is the transpose: <R x, y> = <x, R^T y>, it agrees with differences of the forward map, and it undoes
    the forward map."""
    T, H, D = 6, 3, 64
    table, pos = table_of(50, 32, FP32), torch.randint(0, 50, (T,), device=DEV)
    for interleave in (False, True):
        kw = dict(interleave=interleave, rotary_offset=8)

        def turn(v, **more):
            return ops.rotary_embedding(pos, v, None, table, out_query=torch.empty_like(v), **kw, **more)[0]
        x, y = torch.randn(T, H, D, device=DEV), torch.randn(T, H, D, device=DEV)
        grad = turn(y, inverse=True)
        lhs, rhs = (turn(x).double() * y.double()).sum(), (x.double() * grad.double()).sum()
        assert abs(lhs - rhs) <= 2.0 ** -22 * (x.double().norm() * y.double().norm())
        # differences: the map is linear, so a step of one in an input changes <R x, y> by the gradient there
        for t, h, d in ((0, 0, 8), (1, 2, 25), (5, 1, 39), (2, 0, 3)):
            e = torch.zeros_like(x)
            e[t, h, d] = 1.0
            diff = (turn(e).double() * y.double()).sum()
            assert abs(diff - grad[t, h, d].double()) <= 2.0 ** -22 * y.abs().max().double() * 2
        back = turn(turn(x), inverse=True)
        assert (back - x).abs().max() <= 2.0 ** -21 * x.abs().max()


def test_gradient_through_an_autograd_function():
    """What a training step does: the rotation in the forward, its transpose in the backward.  Outside of one, an operand that
    requires grad is refused instead of losing its gradient."""
    T, H, D = 5, 3, 64
    table, pos = table_of(50, 32, FP32), torch.randint(0, 50, (T,), device=DEV)

    class Rotate(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return ops.rotary_embedding(pos, x, None, table, rotary_offset=8, out_query=torch.empty_like(x))[0]

        @staticmethod
        def backward(ctx, g):
            return ops.rotary_embedding(pos, g.contiguous(), None, table, rotary_offset=8, inverse=True, out_query=torch.empty_like(g))[0]

    x, y = torch.randn(T, H, D, device=DEV, requires_grad=True), torch.randn(T, H, D, device=DEV)
    (Rotate.apply(x) * y).sum().backward()
    want, bound = rotate64(y, table, pos, 8, False, True)   # the formula's gradient: the transposed map of y
    assert ((x.grad.double() - want).abs() <= bound + half_step(FP32) * (want.abs() + bound)).all()
    for call in (ops.rotary_embedding, lambda *a: torch.ops.xllm_ops.rotary_embedding(*a)):
        with pytest.raises((ValueError, RuntimeError)):
            call(pos, x, None, table)
    before = x.detach().clone()
    with torch.no_grad():
        ops.rotary_embedding(pos, x, None, table)
    assert_rotated(x.detach(), before, table, pos, 0, False, False)


def test_infinities_and_nan_stay_in_their_pair():
    T, H, D = 4, 4, 64
    x = torch.randn(T, H, D, device=DEV).to(BF16)
    clean = x.clone()
    x[1, 2, 5], x[2, 0, 40] = float("inf"), float("nan")
    table, pos = table_of(9, 64, FP32), torch.arange(T, device=DEV)
    got, ref = ops.rotary_embedding(pos, x.clone(), None, table)[0], ops.rotary_embedding(pos, clean.clone(), None, table)[0]
    touched = torch.zeros(T, H, D, dtype=torch.bool, device=DEV)
    touched[1, 2, [5, 37]] = True
    touched[2, 0, [40, 8]] = True
    assert torch.equal(got[~touched], ref[~touched]) and not torch.isfinite(got[touched]).all()


def test_rotation_graph_and_stream():
    T, H, D = 31, 8, 128
    table = table_of(100, D, FP32)
    pos, q, k = torch.zeros(T, dtype=torch.int64, device=DEV), torch.zeros(T, H, D, dtype=BF16, device=DEV), \
        torch.zeros(T, 2, D, dtype=BF16, device=DEV)
    oq, ok = torch.empty_like(q), torch.empty_like(k)
    ops.rotary_embedding(pos, q, k, table, out_query=oq, out_key=ok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary_embedding(pos, q, k, table, out_query=oq, out_key=ok)
    for i in range(3):
        pos.copy_(torch.randint(0, 100, (T,)))
        q.copy_(torch.randn(T, H, D))
        k.copy_(torch.randn(T, 2, D))
        graph.replay()
        eager = ops.rotary_embedding(pos, q.clone(), k.clone(), table)
        torch.cuda.synchronize()
        assert torch.equal(oq, eager[0]) and torch.equal(ok, eager[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.rotary_embedding(pos, q, k, table, out_query=torch.empty_like(q), out_key=torch.empty_like(k))
    side.synchronize()
    assert torch.equal(again[0], oq) and torch.equal(again[1], ok)


def test_rotation_refusals():
    T, H, D = 4, 2, 64
    q, k = torch.zeros(T, H, D, dtype=BF16, device=DEV), torch.zeros(T, H, D, dtype=BF16, device=DEV)
    table, pos = table_of(9, 32, FP32), torch.zeros(T, dtype=torch.int64, device=DEV)
    good = (pos, q, k, table)
    ops.rotary_embedding(*good)
    empty = torch.empty(0, H, D, dtype=BF16, device=DEV)
    assert ops.rotary_embedding(pos[:0], empty, None, table)[0] is empty
    for args, kw in [((pos.int(), q, k, table), {}), ((pos[:3], q, k, table), {}), ((pos, q.double(), k, table), {}),
                     ((pos, q, k.float(), table), {}), ((pos, q, k[:3], table), {}), ((pos, q, k, table[:, ::2]), {}),
                     ((pos, q, k, table.double()), {}), (good, dict(rotary_offset=33)), (good, dict(rotary_offset=-1)),
                     (good, dict(out_query=q[:, :1])), (good, dict(out_query=k)), (good, dict(out_query=q.view(H, T, D).transpose(0, 1))),
                     ((pos, q, None, table), dict(out_key=k)), ((pos, q[:1].expand(T, H, D), None, table), {}),
                     ((pos, q.transpose(1, 2), None, table), {}), ((pos, q, q, table), {}), ((pos, q, k, table[:0]), {}),
                     ((pos.cpu(), q, k, table), {})]:
        with pytest.raises((ValueError, TypeError)):
            ops.rotary_embedding(*args, **kw)


def test_lanes_beyond_31_bits():
    """Tables and operands off the 16-byte boundary take a lane per pair: more than 2^31 of them."""
    inv, _ = ops.rope_frequencies(66, device=DEV)
    n = 2 ** 31 // 33 + 1000
    rows = ops.build_cos_sin_cache(inv, n, dtype=BF16)
    assert rows.numel() // 2 > 2 ** 31
    few = torch.cat([torch.arange(50), torch.arange(n // 2, n // 2 + 50), torch.arange(n - 1100, n)]).to(DEV)
    assert torch.equal(rows[few], ops.build_cos_sin_cache(inv, position_ids=few, dtype=BF16))
    del rows
    T, H, D = 2 ** 19 + 3, 64, 128
    buf = torch.zeros(T * H * D + 1, dtype=BF16, device=DEV)
    q = buf[1:].view(T, H, D)
    table, pos = table_of(64, D, FP32), torch.arange(T, device=DEV) % 64
    at = torch.tensor([0, 1, T // 2, T - 4, T - 1], device=DEV)
    part = torch.randn(5, H, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(BF16)
    q[at] = part
    ops.rotary_embedding(pos, q, None, table)
    assert torch.equal(q[at], ops.rotary_embedding(pos[at], part, None, table)[0])
    q[at] = 0
    assert buf[:2 ** 30].count_nonzero() == 0 and buf[-2 ** 30:].count_nonzero() == 0


# ------------------------------------------------------------------------------------------
# MLA prologue

def mla_inputs(T, H, dtype, seed=0, rows=300):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(T, H, 192, generator=gen, device=DEV).to(dtype)
    kv = (torch.randn(T, 640, generator=gen, device=DEV) * 2).to(dtype)[:, 32:608]
    w = (1 + 0.2 * torch.randn(512, generator=gen, device=DEV)).to(dtype)
    pos = torch.randint(0, rows, (T,), generator=torch.Generator().manual_seed(seed)).to(DEV)
    return q[..., 128:], kv, w, pos


def assert_prologue(oq, rows, q_pe, kv, w, eps, table, pos, interleave):
    assert_rotated(oq, q_pe, table, pos, 0, interleave, False)
    assert_rotated(rows[:, None, 512:], kv[:, None, 512:], table, pos, 0, interleave, False)
    x = kv[:, :512].double()
    want = x * torch.rsqrt(x.square().mean(1, keepdim=True) + eps) * w.double()
    # the sum of 512 squares in a tree of 8 + 6 additions, the root and two products: below 20 roundings of 2^-24
    err = (rows[:, :512].double() - want).abs()
    tiny = torch.finfo(kv.dtype).smallest_normal * torch.finfo(kv.dtype).eps / 2
    assert (err <= (half_step(kv.dtype) + 20 * 2.0 ** -24 * 1.01) * want.abs() + tiny).all(), err.max()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 128), (3, 5), (64, 20), (65, 128), (301, 128), (6, 130)])
@pytest.mark.parametrize("interleave", [True, False])
def test_mla_prologue(dtype, T, H, interleave):
    q_pe, kv, w, pos = mla_inputs(T, H, dtype, seed=T + H)
    table = table_of(300, 64, FP32)
    bs = 16
    blocks = -(-T // bs) + 2
    cache = torch.full((blocks, bs, 1, 576), 5.0, dtype=dtype, device=DEV)
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(T))[:T].to(torch.int32)
    if T > 2:
        slots[1], slots[2] = -1, blocks * bs   # skipped
    oq = torch.full((T, H, 64), 9.0, dtype=dtype, device=DEV)
    out_kv = torch.full((T, 576), 9.0, dtype=dtype, device=DEV)
    ops.mla_norm_rope_and_cache(q_pe, kv, w, 1e-6, table, interleave, pos, k_cache=cache, slot_mapping=slots.to(DEV),
                                out_q_pe=oq, out_kv=out_kv)
    assert_prologue(oq, out_kv, q_pe, kv, w, 1e-6, table, pos, interleave)
    want = torch.full((blocks * bs, 576), 5.0, dtype=dtype)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * bs:
            want[s] = out_kv[t].cpu()
    assert torch.equal(cache.view(-1, 576).cpu(), want)   # the rows, and nothing else
    # in place, and without a cache: the same bits
    q2, kv2 = q_pe.clone(), kv.clone()
    ops.mla_norm_rope_and_cache(q2, kv2, w, 1e-6, table, interleave, pos, out_kv=kv2)
    assert torch.equal(q2, oq) and torch.equal(kv2, out_kv)
    only_cache = torch.zeros_like(cache)
    ops.mla_norm_rope_and_cache(q_pe, kv, w, 1e-6, table, interleave, pos, k_cache=only_cache, slot_mapping=slots.to(DEV),
                                out_q_pe=torch.empty_like(oq))
    assert torch.equal(only_cache.view(-1, 576)[slots[0].item()], out_kv[0])


def test_mla_prologue_of_no_tokens():
    table = ops.build_cos_sin_cache(ops.rope_frequencies(64, device=DEV)[0], 8)
    cache = torch.full((2, 16, 1, 576), 3.0, dtype=BF16, device=DEV)
    q, kv = torch.empty(0, 4, 64, dtype=BF16, device=DEV), torch.empty(0, 576, dtype=BF16, device=DEV)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    got = ops.mla_norm_rope_and_cache(q, kv, torch.ones(512, dtype=BF16, device=DEV), 1e-6, table, True, none, cache, none.int())
    assert got[0] is q and got[1] is None and (cache == 3).all()


@pytest.mark.parametrize("T", [1, 5])
def test_mla_prologue_on_slices_of_one_buffer(T):
    """The latent rows and the queries of one projection's output, both in place."""
    H, width = 4, 576 + 4 * 192
    x = torch.randn(T, width, generator=torch.Generator(device=DEV).manual_seed(T), device=DEV).to(BF16)
    w = torch.ones(512, dtype=BF16, device=DEV)
    table = ops.build_cos_sin_cache(ops.rope_frequencies(64, device=DEV)[0], 8)
    pos = torch.arange(T, device=DEV)

    def parts(y):
        return y[:, 576:].view(T, H, 192)[..., 128:], y[:, :576]

    q, kv = parts(x)
    oq, okv = torch.empty(T, H, 64, dtype=BF16, device=DEV), torch.empty(T, 576, dtype=BF16, device=DEV)
    ops.mla_norm_rope_and_cache(q, kv, w, 1e-6, table, False, pos, out_q_pe=oq, out_kv=okv)
    y = x.clone()
    q, kv = parts(y)
    ops.mla_norm_rope_and_cache(q, kv, w, 1e-6, table, False, pos, out_kv=kv)
    assert torch.equal(q, oq) and torch.equal(kv, okv)
    assert torch.equal(y[:, 576:].view(T, H, 192)[..., :128], x[:, 576:].view(T, H, 192)[..., :128])


def test_mla_prologue_zero_rows_and_positions_outside():
    q_pe, kv, w, pos = mla_inputs(9, 4, BF16)
    kv[3] = 0
    pos[2], pos[5] = -1, 300
    table = table_of(300, 64, BF16)
    oq, rows = torch.empty(9, 4, 64, dtype=BF16, device=DEV), torch.empty(9, 576, dtype=BF16, device=DEV)
    ops.mla_norm_rope_and_cache(q_pe, kv, w, 1e-6, table, True, pos, out_q_pe=oq, out_kv=rows)
    assert_prologue(oq, rows, q_pe, kv, w, 1e-6, table, pos, True)
    assert (rows[3, :512] == 0).all() and torch.equal(rows[2, 512:], kv[2, 512:]) and torch.equal(oq[5], q_pe[5])


def test_mla_prologue_graph():
    T, H = 7, 16
    q_pe, kv, w, pos = mla_inputs(T, H, BF16)
    table, cache = table_of(300, 64, FP32), torch.zeros(4, 16, 1, 576, dtype=BF16, device=DEV)
    slots, oq = torch.arange(T, dtype=torch.int32, device=DEV), torch.empty(T, H, 64, dtype=BF16, device=DEV)
    run = lambda c, o: ops.mla_norm_rope_and_cache(q_pe, kv, w, 1e-6, table, True, pos, k_cache=c, slot_mapping=slots, out_q_pe=o)
    run(cache, oq)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(cache, oq)
    for i in range(3):
        pos.copy_(torch.randint(0, 300, (T,)))
        slots.copy_(torch.randperm(64)[:T])
        kv.copy_(torch.randn(T, 576))
        eager, o2 = cache.clone(), torch.empty_like(oq)
        graph.replay()
        run(eager, o2)
        torch.cuda.synchronize()
        assert torch.equal(cache, eager) and torch.equal(oq, o2)


def test_mla_prologue_refusals():
    T, H = 4, 2
    q_pe, kv, w, pos = mla_inputs(T, H, BF16)
    table, cache = table_of(9, 64, FP32), torch.zeros(2, 16, 1, 576, dtype=BF16, device=DEV)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    base = dict(q_pe=q_pe, kv=kv, kv_norm_weight=w, eps=1e-6, cos_sin_cache=table, interleave=True, position_ids=pos,
                k_cache=cache, slot_mapping=slots, out_q_pe=torch.empty(T, H, 64, dtype=BF16, device=DEV))
    ops.mla_norm_rope_and_cache(**base)
    for change in (dict(k_cache=None), dict(slot_mapping=None), dict(k_cache=None, slot_mapping=None), dict(kv=kv.float()),
                   dict(kv=kv[:3]), dict(kv=kv[:, :575]), dict(cos_sin_cache=table_of(9, 32, FP32)), dict(position_ids=pos.int()),
                   dict(slot_mapping=slots.long()), dict(slot_mapping=slots[:3]), dict(k_cache=cache[..., :512]),
                   dict(k_cache=cache.half()), dict(out_q_pe=torch.empty(T, H, 32, dtype=BF16, device=DEV)),
                   dict(out_kv=kv[:, 1:]), dict(q_pe=q_pe.float()), dict(kv_norm_weight=w[:256])):
        args = dict(base)
        args.update(change)
        with pytest.raises((ValueError, TypeError)):
            ops.mla_norm_rope_and_cache(**args)
    # what the library itself refuses: rows off the 16-byte boundary, another latent width
    odd = torch.zeros(T, 584, dtype=BF16, device=DEV)[:, 4:580]
    with pytest.raises(Exception, match="aligned"):
        ops.mla_norm_rope_and_cache(**dict(base, kv=odd))
    with pytest.raises(Exception, match="not implemented"):
        ops.mla_norm_rope_and_cache(**dict(base, kv=torch.zeros(T, 256 + 64, dtype=BF16, device=DEV), kv_norm_weight=w[:256].clone(),
                                           k_cache=torch.zeros(2, 16, 1, 320, dtype=BF16, device=DEV)))
