"""Rotary positions and their backward pass against 64 bits.  Bounds: a rounding of the result (half a step), and 2^-19 of the
pair's size for sine, cosine and two products in 32 bits."""
import math

import pytest

from tests import long_context_ref as R

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from tests import gpu_util as U

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return U


def types():
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16}


def turned(x, positions, freq, rot, interleaved, magnitude, sign):
    """(values, bounds) in 64 bits; x [tokens][heads][dim]."""
    import torch

    u = R.unit(x.dtype)
    x = x.double()
    angle = (positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device))[:, None]
    c, s = angle.cos() * magnitude, angle.sin() * magnitude * sign
    y, e = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    p, q = x[..., a], x[..., b]
    y[..., a], y[..., b] = p * c - q * s, q * c + p * s
    size = (p.abs() + q.abs()) * abs(magnitude)
    for at in (a, b):
        e[..., at] = u * y[..., at].abs() + 2.0 ** -19 * size + 2.0 ** -25
    return y, e


CASES = [
    # tokens, heads, kv_heads, dim, rot, interleaved
    (1, 1, 1, 64, 64, False),
    (5, 3, 1, 64, 64, True),
    (37, 8, 8, 128, 128, False),
    (200, 12, 4, 128, 96, True),
    (33, 4, 2, 64, 22, False),
    (33, 4, 2, 64, 22, True),
    (7, 2, 2, 80, 2, False),
    (9, 5, 3, 6, 4, True),
    (3000, 32, 8, 128, 64, False),
    (2, 3, 1, 256, 256, False),
]


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,heads,kv,dim,rot,interleaved", CASES)
def test_forward_and_backward(env, kind, n, heads, kv, dim, rot, interleaved):
    import torch

    U, pk = env, env.pkg()
    g = torch.Generator("cuda").manual_seed(n + dim)
    row = torch.randn((n, heads + kv + 1, dim), device="cuda", generator=g).to(types()[kind])  # a wider row: strides of a view
    q, k = row[:, :heads], row[:, heads:heads + kv]
    positions = torch.randint(-5, 1000, (n,), device="cuda", generator=g).int()
    plan = pk.RopePlan(U.ctx(), dim, rot_dim=rot, interleaved=interleaved, magnitude=1.25)
    for sign, apply in ((1, plan.forward), (-1, plan.backward)):
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        apply(positions, q, q_out, k, k_out)
        U.ctx().sync()
        for x, got in ((q, q_out), (k, k_out)):
            want, bound = turned(x, positions, plan.frequencies(), rot, interleaved, 1.25, sign)
            assert torch.equal(got[..., rot:], x[..., rot:])
            assert R.worst(got[..., :rot], want[..., :rot], bound[..., :rot]) <= 1.0
        alone = torch.empty_like(q)
        apply(positions, q, alone)
        U.ctx().sync()
        assert torch.equal(alone, q_out)
    # in place, on the views themselves
    want = q_out.clone()
    rest = row[:, heads:].clone()
    plan.backward(positions, q, q)
    U.ctx().sync()
    assert torch.equal(q, want) and torch.equal(row[:, heads:], rest)
    plan.close()


@gpu
@pytest.mark.parametrize("scaling,factor,length,low,high", [(0, 1.0, 0, 1.0, 32.0), (1, 4.0, 0, 1.0, 32.0), (2, 16.0, 8192, 1.0, 32.0), (3, 8.0, 8192, 1.0, 4.0)])
def test_far_positions_and_scalings(env, scaling, factor, length, low, high):
    """Every 32-bit position has its angle, where a product in 32 bits would have none of its digits."""
    import torch

    U, pk = env, env.pkg()
    plan = pk.RopePlan(U.ctx(), 64, base=500000.0, scaling=scaling, factor=factor, original_len=length, low=low, high=high)
    positions = torch.tensor([0, 1, 65535, 1 << 20, 999999937, (1 << 31) - 1, -1, -(1 << 31)], device="cuda").int()
    g = torch.Generator("cuda").manual_seed(3)
    q = torch.randn((8, 2, 64), device="cuda", generator=g).half()
    out = torch.empty_like(q)
    plan.forward(positions, q, out)
    U.ctx().sync()
    # the angles with enough digits: positions times frequencies modulo a turn in Python's integers
    want, bound = q.double().clone(), None
    freq = plan.frequencies()
    for i, p in enumerate(positions.tolist()):
        for j, f in enumerate(freq):
            from fractions import Fraction

            angle = float(Fraction(p) * Fraction(f) % (2 * Fraction(314159265358979323846264338327950288, 10 ** 35)))
            a, b = q[i, :, j].double(), q[i, :, j + 32].double()
            want[i, :, j], want[i, :, j + 32] = a * math.cos(angle) - b * math.sin(angle), b * math.cos(angle) + a * math.sin(angle)
    bound = R.unit(q.dtype) * want.abs() + 2.0 ** -19 * (q.double().abs() + q.double().abs().roll(32, -1)) + 2.0 ** -25
    assert R.worst(out, want, bound) <= 1.0
    plan.close()


@gpu
@pytest.mark.parametrize("offset,extra", [(1, 0), (2, 0), (4, 0), (0, 1), (0, 2), (0, 6), (3, 5)])
def test_any_alignment(env, offset, extra):
    """Data and strides off the widest vectors' boundaries."""
    import torch

    U, pk = env, env.pkg()
    plan = pk.RopePlan(U.ctx(), 64)
    n, heads = 11, 3
    flat = torch.randn(n * heads * (64 + extra) + offset, device="cuda").half()
    q = flat[offset:].view(n, heads, 64 + extra)[..., :64]
    out = torch.empty((n, heads, 64), dtype=torch.float16, device="cuda")
    positions = torch.arange(n, device="cuda").int()
    plan.forward(positions, q, out)
    U.ctx().sync()
    want, bound = turned(q, positions, plan.frequencies(), 64, False, 1.0, 1)
    assert R.worst(out, want, bound) <= 1.0
    plan.close()


@gpu
def test_gradients_against_differences(env):
    """The sum of g * forward(x) moves with x as backward(g) says: the map is linear, so differences are exact up to rounding."""
    import torch

    U, pk = env, env.pkg()
    plan = pk.RopePlan(U.ctx(), 64, rot_dim=48, interleaved=True, magnitude=0.75)
    g = torch.Generator("cuda").manual_seed(1)
    x, dx, w = (torch.randn((50, 4, 64), device="cuda", generator=g).half() for _ in range(3))
    positions = torch.randint(0, 5000, (50,), device="cuda", generator=g).int()
    moved = (x + dx)
    outs = []
    for t in (x, moved):
        y = torch.empty_like(t)
        plan.forward(positions, t, y)
        outs.append(y)
    back = torch.empty_like(w)
    plan.backward(positions, w, back)
    U.ctx().sync()
    step = moved.double() - x.double()
    left, right = (w.double() * (outs[1].double() - outs[0].double())).sum(), (back.double() * step).sum()
    size = (w.double().abs() * (outs[0].double().abs() + outs[1].double().abs())).sum() + (back.double().abs() * step.abs()).sum()
    assert abs(left - right) <= (R.unit(x.dtype) + 2.0 ** -18) * size
    plan.close()


@gpu
def test_refusals(env):
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    for bad in (dict(rot_dim=130), dict(rot_dim=3), dict(base=0.5), dict(scaling=9), dict(scaling=pk.ROPE_RAMP), dict(scaling=pk.ROPE_LINEAR, factor=0.0)):
        with pytest.raises(pk.AigError):
            pk.RopePlan(ctx, 128, **bad)
    plan = pk.RopePlan(ctx, 64)
    q = torch.zeros((4, 2, 64), dtype=torch.float16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for args in ((pos[:3], q, q), (pos.long(), q, q), (pos, q.float(), q.float()), (pos, q[..., :32], q[..., :32]), (pos, q, q.bfloat16()),
                 (pos, q, torch.zeros((4, 3, 64), dtype=torch.float16, device="cuda")), (pos, q.cpu(), q), (pos, q.transpose(1, 2), q), (pos, q, q, q, None)):
        with pytest.raises(ValueError):
            plan.forward(*args)
    lib = pk.lib()
    heads = pk._pack_heads(q.data_ptr(), 2, 128, 64)
    bad_stride = pk._pack_heads(q.data_ptr(), 2, -128, 64)
    null = pk._pack_heads(0, 2, 128, 64)
    assert lib.aig_rope_forward(plan.handle, 2, pos.data_ptr(), 4, heads, heads, None, None) == -1
    assert lib.aig_rope_forward(plan.handle, 0, None, 4, heads, heads, None, None) == -1
    assert lib.aig_rope_forward(plan.handle, 0, pos.data_ptr(), -1, heads, heads, None, None) == -1
    for wrong in (bad_stride, null, None):
        assert lib.aig_rope_forward(plan.handle, 0, pos.data_ptr(), 4, wrong, heads, None, None) == -1
        assert lib.aig_rope_forward(plan.handle, 0, pos.data_ptr(), 4, heads, wrong, None, None) == -1
    empty = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    plan.forward(pos[:0], empty, empty)
    ctx.sync()
    plan.close()


@gpu
def test_offsets_beyond_32_bits(env):
    """Tokens so far apart that they pass 2^32 elements."""
    import torch

    n, tokens, dim = 5 << 30, 70, 64
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("not enough memory")
    wide = torch.empty(n, dtype=torch.float16, device="cuda")
    row = n // tokens // 8 * 8
    q, q_out = (wide.as_strided((tokens, 3, dim), (row, dim, 1), at) for at in (0, 3 * dim))
    q.normal_(generator=torch.Generator("cuda").manual_seed(31))
    positions = torch.arange(tokens, device="cuda").int()
    plan = env.pkg().RopePlan(env.ctx(), dim)
    plan.forward(positions, q, q_out)
    env.ctx().sync()
    want, bound = turned(q, positions, plan.frequencies(), dim, False, 1.0, 1)
    assert R.worst(q_out, want, bound) <= 1.0
    plan.close()
