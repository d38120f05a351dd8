"""Attention over whole sequences with a sliding window and sinks, and its gradients, against 64 bits.  Tolerances are
bounds by arithmetic (tests/long_context_ref.py), element by element."""
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


def tensors(seed, dtype, B, Tq, Tk, H, KV, d, spread=1.0):
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: (torch.randn(s, device="cuda", generator=g) * spread).to(dtype)  # noqa: E731
    return r(B, Tq, H, d), r(B, Tk, KV, d), r(B, Tk, KV, d), r(B, Tq, H, d)


MARK = 7.0  # what rows hold that no call may write


def run_forward(U, q, k, v, window=0, sinks=0, lengths=None, scale=None):
    import torch

    B, Tq, H, d = q.shape
    out = torch.full(q.shape, MARK, dtype=q.dtype, device="cuda")
    lse = torch.full((B, H, Tq), MARK, device="cuda")
    n = None if lengths is None else torch.tensor(lengths, device="cuda").int()
    U.pkg().WindowAttention(U.ctx(), window, sinks, scale).forward(q, k, v, out, lse, n)
    U.ctx().sync()
    return out, lse


def run_backward(U, q, k, v, out, lse, dout, window=0, sinks=0, lengths=None, scale=None):
    import torch

    dq, dk, dv = (torch.full(x.shape, MARK, dtype=q.dtype, device="cuda") for x in (q, k, v))
    delta = torch.empty_like(lse)
    n = None if lengths is None else torch.tensor(lengths, device="cuda").int()
    U.pkg().WindowAttention(U.ctx(), window, sinks, scale).backward(q, k, v, out, lse, dout, dq, dk, dv, delta, n)
    U.ctx().sync()
    return dq, dk, dv


def check(got, want, bound, names):
    for name, x in zip(names, got):
        assert R.worst(x, want[name], bound[name]) <= 1.0, name
        absent = want[name].isnan()
        assert (x[absent] == MARK).all(), "%s: rows behind a sequence's end were written" % name


CASES = [
    # B, Tq, Tk, H, KV, window, sinks, lengths
    (1, 1, 1, 1, 1, 0, 0, None),
    (2, 3, 3, 2, 1, 0, 0, None),
    (2, 64, 64, 8, 8, 0, 0, None),
    (1, 128, 128, 2, 2, 16, 1, None),
    (3, 127, 127, 2, 1, 128, 4, [127, 1, 0]),
    (1, 129, 129, 3, 1, 0, 0, None),
    (2, 200, 200, 4, 2, 1, 0, [200, 131]),
    (1, 257, 257, 2, 2, 33, 3, None),
    (2, 300, 300, 2, 1, 40, 130, [300, 7]),
    (1, 640, 640, 1, 1, 130, 0, None),
    (1, 700, 700, 2, 1, 200, 257, [555]),
    (2, 5, 300, 2, 2, 0, 0, [300, 296]),
    (1, 1, 513, 4, 1, 100, 2, None),
    (2, 200, 333, 2, 1, 64, 64, [333, 200]),
    (1, 260, 1000, 2, 1, 129, 200, None),
]


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("B,Tq,Tk,H,KV,window,sinks,lengths", CASES)
def test_forward_and_gradients(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths):
    import torch

    dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    q, k, v, g = tensors(Tq * 7 + Tk, dtype, B, Tq, Tk, H, KV, d)
    want, bound = R.window_attention(q, k, v, window, sinks, lengths, d ** -0.5, g)
    out, lse = run_forward(env, q, k, v, window, sinks, lengths)
    check((out, lse), want, bound, ("out", "lse"))
    grads = run_backward(env, q, k, v, out, lse, g, window, sinks, lengths)
    check(grads, want, bound, ("dq", "dk", "dv"))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_rows_behind_the_end_may_hold_anything(env, kind, d):
    """Padding of q, k, v, out's gradient and the statistics: NaN and infinities there reach no row that is there."""
    import math

    import torch

    dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    for Tq, Tk, lengths, window, sinks in ((64, 64, [64, 1, 33], 0, 0), (300, 300, [300, 65, 200], 70, 2), (150, 400, [400, 251, 390], 0, 0)):
        q, k, v, g = tensors(3, dtype, 3, Tq, Tk, 4, 2, d)
        want, bound = R.window_attention(q, k, v, window, sinks, lengths, d ** -0.5, g)
        for b, n in enumerate(lengths):
            rows = max(0, n - (Tk - Tq))
            q[b, rows:], g[b, rows:], k[b, n:], v[b, n:] = math.nan, math.inf, math.nan, -math.inf
        out, lse = run_forward(env, q, k, v, window, sinks, lengths)
        check((out, lse), want, bound, ("out", "lse"))
        lse[lse == MARK] = math.nan
        out[out == MARK] = math.nan
        grads = run_backward(env, q, k, v, out, lse, g, window, sinks, lengths)
        check(grads, want, bound, ("dq", "dk", "dv"))


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_layouts(env, d):
    """Columns of a fused projection, heads outside of tokens, a batch with gaps; results into strided tensors too."""
    import torch

    B, T, H, KV = 2, 150, 4, 2
    q, k, v, g = tensors(5, torch.bfloat16, B, T, T, H, KV, d)
    want, bound = R.window_attention(q, k, v, 40, 1, None, d ** -0.5, g)

    def fused(*parts):
        row = torch.cat(parts, 2).contiguous()
        out, at = [], 0
        for x in parts:
            out.append(row[:, :, at:at + x.shape[2]])
            at += x.shape[2]
        return out

    heads_first = lambda *parts: [x.transpose(1, 2).contiguous().transpose(1, 2) for x in parts]  # noqa: E731
    gaps = lambda *parts: [torch.stack((x, x), 1)[:, 0] for x in parts]  # noqa: E731
    wa = env.pkg().WindowAttention(env.ctx(), 40, 1)
    for arrange in (fused, heads_first, gaps):
        a, b, c = arrange(q, k, v)
        o, da, e = arrange(torch.full_like(q, MARK), torch.full_like(q, MARK), g)
        dk, dv = arrange(torch.full_like(k, MARK), torch.full_like(k, MARK))
        lse, delta = torch.empty((B, H, T), device="cuda"), torch.empty((B, H, T), device="cuda")
        wa.forward(a, b, c, o, lse)
        wa.backward(a, b, c, o, lse, e, da, dk, dv, delta)
        env.ctx().sync()
        check((o, lse, da, dk, dv), want, bound, ("out", "lse", "dq", "dk", "dv"))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [1, 60, 300, 700])
def test_one_visible_key_has_no_gradient(env, T, d):
    """A window of one key: the weight is 1 whatever the score, dq and dk are zero exactly, dv is the gradient of the output."""
    import torch

    q, k, v, g = tensors(6, torch.float16, 1, T, T, 2, 2, d)
    out, lse = run_forward(env, q, k, v, window=1)
    assert torch.equal(out, v)
    dq, dk, dv = run_backward(env, q, k, v, out, lse, g, window=1)
    assert not dq.any() and not dk.any() and torch.equal(dv, g)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("scale", [2.0 ** -18, 2.0 ** -9, 1.0, 2.0 ** 7])
def test_fp16_gradients_of_any_size(env, scale, grow, d):
    """Gradients from 4e-6 to 500, even or growing (and shrinking) a thousandfold along the sequence, values likewise: what a plain
    16-bit dS would lose to its smallest steps or its largest value.  The bound leaves out both."""
    import torch

    T = 900
    q, k, v, g = tensors(7, torch.float16, 1, T, T, 2, 1, d)
    slope = torch.logspace(-1.5, 1.5, T, device="cuda")[None, :, None, None] if grow else 1.0
    g = (g.float() * slope * scale).half()
    v = (v.float() * (slope.flip(1) if grow else 1.0)).half()
    want, bound = R.window_attention(q, k, v, 0, 0, None, d ** -0.5, g)
    out, lse = run_forward(env, q, k, v)
    dq, dk, dv = run_backward(env, q, k, v, out, lse, g)
    u = 2.0 ** -11
    for name, x, other in (("dq", dq, k), ("dk", dk, q), ("dv", dv, g)):
        # in the 2-norm: each weight or dS off by a rounding of its own, D by that of the output; the result by its own and by fp16's smallest step
        off, size = (x.double() - want[name]).norm(), want[name].norm()
        assert off <= 4 * u * size + 2.0 ** -25 * x.numel() ** 0.5, (name, float(off / size))


@gpu
def test_gradients_against_differences(env):
    """The derivative of sum(w * out) along a direction, by central differences of the 64-bit form, is what the gradients say."""
    import torch

    B, T, H, KV, d = 1, 90, 4, 2, 64
    q, k, v, w = tensors(8, torch.float16, B, T, T, H, KV, d)
    out, lse = run_forward(env, q, k, v, 30, 2)
    grads = run_backward(env, q, k, v, out, lse, w, 30, 2)
    g = torch.Generator("cuda").manual_seed(9)
    for x, dx in zip((q, k, v), grads):
        way = torch.randn(x.shape, device="cuda", generator=g, dtype=torch.float64)

        def value(step):
            moved = [t.double() + (step * way if t is x else 0) for t in (q, k, v)]
            s = torch.einsum("bqkgd,btkd->bkgqt", moved[0].view(B, T, KV, H // KV, d), moved[1]) * d ** -0.5
            seen = R.visible(T, T, 30, 2, T, "cuda")
            p = torch.softmax(s.masked_fill(~seen, -float("inf")), -1)
            return (torch.einsum("bkgqt,btkd->bqkgd", p, moved[2]).reshape(B, T, H, d) * w.double()).sum()

        h = 1e-4
        slope = (value(h) - value(-h)) / (2 * h)  # off by h^2 times a third derivative of order 1 a term
        said = (dx.double() * way).sum()
        size = (dx.double().abs() * way.abs()).sum()
        assert abs(slope - said) <= 4 * 2.0 ** -11 * size


@gpu
@pytest.mark.parametrize("T,d", [(64, 64), (700, 64), (700, 128)])
def test_same_bits_every_time(env, T, d):
    import torch

    q, k, v, g = tensors(10, torch.float16, 3, T, T, 4, 2, d)
    first = None
    for _ in range(3):
        out, lse = run_forward(env, q, k, v, 100, 1)
        got = (out, lse) + run_backward(env, q, k, v, out, lse, g, 100, 1)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@gpu
def test_every_kernel_of_heads_of_64(env):
    """Sizes on both sides of the choices between kernels: many short sequences and few long ones, with and without sinks."""
    import torch

    for B, T, H, KV, window, sinks in ((40, 130, 8, 8, 0, 0), (24, 500, 8, 8, 64, 0), (24, 500, 8, 4, 64, 3), (1, 1500, 2, 1, 0, 0), (80, 128, 8, 8, 0, 0), (80, 129, 8, 8, 0, 0)):
        q, k, v, g = tensors(T, torch.float16, B, T, T, H, KV, 64)
        some = [0, B // 2, B - 1] if B > 1 else [0]
        want, bound = R.window_attention(q[some], k[some], v[some], window, sinks, None, 0.125, g[some])
        out, lse = run_forward(env, q, k, v, window, sinks)
        grads = run_backward(env, q, k, v, out, lse, g, window, sinks)
        check([x[some] for x in (out, lse) + grads], want, bound, ("out", "lse", "dq", "dk", "dv"))


@gpu
def test_captured_training_step_and_other_streams(env):
    """Forward and backward captured twice and replayed in turn on changing inputs; a context with a stream of its own."""
    import torch

    U, pk = env, env.pkg()
    main = U.ctx()
    for ctx in (main, pk.Context(0, use_torch_stream=False)):
        q, k, v, g = tensors(11, torch.bfloat16, 2, 200, 200, 4, 2, 64)
        out, dq, dk, dv = (torch.empty_like(x) for x in (q, q, k, v))
        lse, delta = torch.empty((2, 4, 200), device="cuda"), torch.empty((2, 4, 200), device="cuda")
        wa = pk.WindowAttention(ctx, 50, 2)
        torch.cuda.synchronize()

        def step():
            wa.forward(q, k, v, out, lse)
            wa.backward(q, k, v, out, lse, g, dq, dk, dv, delta)

        step()
        ctx.sync()
        graphs = []
        for _ in range(2):
            ctx.graph_begin()
            step()
            graphs.append(ctx.graph_end())
        for i in range(4):
            for x in (q, k, v, g):
                x.normal_()
            torch.cuda.synchronize()
            ctx.graph_launch(graphs[i % 2])
            ctx.sync()
            want, bound = R.window_attention(q, k, v, 50, 2, None, 0.125, g)
            check((out, lse, dq, dk, dv), want, bound, ("out", "lse", "dq", "dk", "dv"))
        for x in graphs:
            pk.lib().aig_graph_destroy(x)
        if ctx is not main:
            ctx.close()


@gpu
def test_refusals(env):
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    q, k, v, g = tensors(12, torch.float16, 2, 8, 8, 4, 2, 64)
    out, lse = torch.empty_like(q), torch.empty((2, 4, 8), device="cuda")
    n = torch.tensor([8, 8], device="cuda").int()
    wa = pk.WindowAttention(ctx)
    for args in ((q.float(), k.float(), v.float(), out.float(), lse), (q, k.bfloat16(), v, out, lse), (q, k, v[:, :7], out, lse), (q, k, v, out[:, :7], lse),
                 (q, k, v, out, lse.double()), (q, k, v, out, lse[:, :3]), (q, k, v, out, lse, n[:1]), (q, k, v, out, lse, n.long()), (q[0], k[0], v[0], out[0], lse),
                 (q, k.cpu(), v, out, lse), (q.transpose(2, 3), k, v, out, lse)):
        with pytest.raises(ValueError):
            wa.forward(*args)
    for change in (dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")), dict(sinks=-1)):
        with pytest.raises(pk.AigError) as e:
            pk.WindowAttention(ctx, **change).forward(q, k, v, out, lse)
        assert e.value.code == -1
    with pytest.raises(pk.AigError):  # more queries than keys
        wa.forward(q, k[:, :7], v[:, :7], out, lse)
    with pytest.raises(pk.AigError):  # three heads over two
        wa.forward(q[:, :, :3], k, v, out[:, :, :3], torch.empty((2, 3, 8), device="cuda"))
    with pytest.raises(pk.AigError) as e:  # heads of 32
        wa.forward(q[..., :32], k[..., :32], v[..., :32], out[..., :32], lse)
    assert e.value.code == -4
    flat = torch.empty(q.numel() + 8, dtype=torch.float16, device="cuda")
    with pytest.raises(pk.AigError):  # off a 16-byte boundary
        wa.forward(flat[1:q.numel() + 1].view(q.shape), k, v, out, lse)
    wide = torch.empty((2, 8, 4, 68), dtype=torch.float16, device="cuda")[..., :64]
    with pytest.raises(pk.AigError):  # strides that are no multiples of 8
        wa.forward(wide, k, v, out, lse)
    with pytest.raises(pk.AigError):  # one head's keys for all: a stride of 0
        wa.forward(q, k[:, :, :1].expand(2, 8, 2, 64), v, out, lse)
    empty = q[:0]
    wa.forward(empty, k[:0], v[:0], out[:0], lse[:0])
    wa.forward(q[:, :0], k, v, out[:, :0], lse[:, :, :0].contiguous())
    ctx.sync()


@gpu
def test_no_queries_leave_keys_without_gradient(env):
    """A chunk whose window no longer reaches the first keys: their gradients are zeros."""
    import torch

    q, k, v, g = tensors(13, torch.bfloat16, 1, 100, 600, 2, 1, 64)
    want, bound = R.window_attention(q, k, v, 50, 0, None, 0.125, g)
    out, lse = run_forward(env, q, k, v, 50)
    grads = run_backward(env, q, k, v, out, lse, g, 50)
    check((out, lse) + grads, want, bound, ("out", "lse", "dq", "dk", "dv"))
    assert not grads[1][:, :400].any() and not grads[2][:, :400].any()


SHARED = [
    # few blocks of keys, each of which many queries see: several thread blocks share one; short sequences leave some of them nothing
    (1, 700, 700, 8, 1, 0, 0, None),
    (1, 700, 700, 3, 1, 0, 0, [70]),
    (2, 1000, 1000, 4, 2, 0, 0, [1000, 130]),
    (1, 90, 2000, 8, 1, 0, 0, None),
    # the sinks' blocks in a launch of their own, next to the others'
    (1, 1500, 1500, 8, 1, 100, 3, None),
    (2, 1500, 1500, 8, 2, 100, 130, [1500, 200]),
    (1, 900, 1200, 8, 1, 64, 1, [1100]),
    (2, 600, 600, 8, 1, 1, 2, [600, 0]),
    (1, 400, 1500, 6, 2, 30, 1600, None),
    (24, 1000, 1000, 8, 2, 30, 1, None),
]


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("B,Tq,Tk,H,KV,window,sinks,lengths", SHARED)
def test_blocks_of_keys_that_many_queries_see(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths):
    test_forward_and_gradients(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 2)])
def test_fp16_gradients_that_grow_over_shared_blocks(env, d, window, sinks):
    """Thread blocks that share a block of keys meet gradients of sizes that differ a thousandfold: each has its own power of two."""
    import torch

    T = 1200
    q, k, v, g = tensors(41, torch.float32, 1, T, T, 8, 1, d)
    size = torch.logspace(-3, 3, T, base=2 ** 3.3, device="cuda")[None, :, None, None]
    q, k, v, g = q.half(), k.half(), v.half(), (g * size).half()
    want, bound = R.window_attention(q, k, v, window, sinks, None, d ** -0.5, g)
    out, lse = run_forward(env, q, k, v, window, sinks)
    check(run_backward(env, q, k, v, out, lse, g, window, sinks), want, bound, ("dq", "dk", "dv"))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths", [None, [2000, 150]])
def test_what_follows_finds_all_gradients(env, lengths, d):
    """The backward's last two launches overlap: a call right behind it, eager or in a graph, reads complete gradients, with the
    same bits every time."""
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    B, T, H = 2, 2000, 8
    q, k, v, g = tensors(42, torch.bfloat16, B, T, T, H, 1, d)
    n = None if lengths is None else torch.tensor(lengths, device="cuda").int()
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    lse, delta = torch.empty((B, H, T), device="cuda"), torch.empty((B, H, T), device="cuda")
    dk, dv, seen = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(q)
    statistics = torch.zeros_like(lse)
    wa, next_op = pk.WindowAttention(ctx, 64, 1), pk.WindowAttention(ctx)
    torch.cuda.synchronize()

    def step():
        wa.forward(q, k, v, out, lse, n)
        wa.backward(q, k, v, out, lse, g, dq, dk, dv, delta, n)
        next_op.forward(q, dk, dv, seen, statistics, n)

    step()
    ctx.sync()
    first = [x.clone() for x in (dk, dv, seen, statistics)]
    again = torch.zeros_like(q)
    next_op.forward(q, dk, dv, again, torch.empty_like(lse), n)
    ctx.sync()
    assert torch.equal(again, seen)
    ctx.graph_begin()
    step()
    graph = ctx.graph_end()
    for i in range(20):
        for x in (dk, dv):
            x.fill_(float("nan"))
            if lengths is not None:
                x[1, lengths[1]:] = 0
        torch.cuda.synchronize()
        ctx.graph_launch(graph) if i % 2 else step()
        ctx.sync()
        valid = slice(None) if lengths is None else slice(0, lengths[1])
        for x, y in zip((dk, dv, seen), first):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1, valid], y[1, valid])
    pk.lib().aig_graph_destroy(graph)


FEW = [
    # few tiles of queries that see many keys: the keys are shared by several thread blocks, some of which may see none
    (1, 70, 4000, 2, 1, 0, 0, None),
    (1, 4000, 4000, 1, 1, 0, 0, [3900]),
    (2, 300, 3000, 2, 1, 0, 0, [3000, 2701]),
    (1, 128, 3000, 3, 3, 1500, 130, None),
    (2, 200, 2500, 2, 2, 1000, 3, [2500, 2301]),
    (1, 1, 5000, 1, 1, 0, 0, None),
    (1, 257, 2000, 1, 1, 700, 1100, [1999]),
    (2, 1030, 1030, 4, 2, 0, 0, None),
]


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("B,Tq,Tk,H,KV,window,sinks,lengths", FEW)
def test_few_queries_that_see_many_keys(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths):
    test_forward_and_gradients(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_shared_keys_of_very_different_scores(env, d):
    """Scores that grow along the keys by hundreds: the parts' maxima differ by more than fp32's exponents reach."""
    import torch

    q, k, v, g = tensors(43, torch.float32, 1, 130, 3000, 2, 1, d)
    k = k + q[:, :1, :1] * torch.linspace(-3, 3, 3000, device="cuda")[None, :, None, None] * (q * q)[:, :1, :1].sum(-1, keepdim=True) ** -0.5 * 8
    q = q + q[:, :1, :1] * 4
    q, k, v, g = (x.bfloat16() for x in (q, k, v, g))
    want, bound = R.window_attention(q, k, v, 0, 0, None, d ** -0.5, g)
    out, lse = run_forward(env, q, k, v)
    check((out, lse), want, bound, ("out", "lse"))
    check(run_backward(env, q, k, v, out, lse, g), want, bound, ("dq", "dk", "dv"))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks,Tq", [(0, 0, 2500), (0, 0, 100), (900, 2, 400)])
def test_fp16_gradients_over_shared_keys_of_growing_values(env, d, window, sinks, Tq):
    """Thread blocks that share a tile of queries meet values that differ a thousandfold: each has its own power of two."""
    import torch

    T = 2500
    q, k, v, g = tensors(44, torch.float32, 1, Tq, T, 1, 1, d)
    v = v * torch.logspace(-3, 3, T, base=2 ** 3.3, device="cuda")[None, :, None, None]
    q, k, v, g = q.half(), k.half(), v.half(), (g * 2.0 ** -6).half()
    want, bound = R.window_attention(q, k, v, window, sinks, None, d ** -0.5, g)
    out, lse = run_forward(env, q, k, v, window, sinks)
    check((out, lse), want, bound, ("out", "lse"))
    check(run_backward(env, q, k, v, out, lse, g, window, sinks), want, bound, ("dq", "dk", "dv"))


SHORT = [
    # sequences of one tile: many of them with heads on their own or in groups, and a few with large groups
    (80, 33, 33, 6, 2, 0, 0, [33, 1, 0, 17] * 20),
    (160, 64, 64, 3, 1, 5, 2, None),
    (150, 7, 60, 8, 1, 30, 1, [60, 59, 53, 40, 0] * 30),
    (3, 64, 64, 16, 1, 0, 0, [64, 20, 3]),
    (2, 50, 61, 8, 1, 16, 20, None),
    (5, 1, 64, 2, 2, 0, 0, [64, 63, 0, 1, 64]),
    (1, 16, 16, 2, 1, 1, 0, None),
    (1, 49, 49, 1, 1, 48, 0, None),
]


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("B,Tq,Tk,H,KV,window,sinks,lengths", SHORT)
def test_sequences_of_one_tile(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths):
    test_forward_and_gradients(env, kind, d, B, Tq, Tk, H, KV, window, sinks, lengths)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,H,KV", [(1, 2, 1), (160, 5, 1)])
@pytest.mark.parametrize("scale", [2.0 ** -18, 1.0, 2.0 ** 7])
def test_fp16_gradients_of_short_sequences(env, scale, B, H, KV, d):
    """Heads of a group whose gradients differ two hundredfold, rising and falling, and sequences likewise."""
    import torch

    q, k, v, g = tensors(45, torch.float32, B, 61, 61, H, KV, d)
    size = torch.tensor([1.0, 2.0 ** -7.5, 2.0 ** -3, 0.0, 2.0 ** -5], device="cuda")
    heads = size[(torch.arange(H, device="cuda")[None] + torch.arange(B, device="cuda")[:, None]) % 5]
    q, k, v, g = q.half(), k.half(), v.half(), (g * heads[:, None, :, None] * scale).half()
    want, bound = R.window_attention(q, k, v, 20, 1, None, d ** -0.5, g)
    out, lse = run_forward(env, q, k, v, 20, 1)
    check(run_backward(env, q, k, v, out, lse, g, 20, 1), want, bound, ("dq", "dk", "dv"))


def put(v, pattern):
    """Values with blocks of keys whose sizes have nothing to do with the others'."""
    import torch

    T = v.shape[1]
    if pattern == "first 64 zero":
        v[:, :64] = 0
    elif pattern == "first 128 zero":
        v[:, :128] = 0
    elif pattern == "middle zero":
        v[:, T // 2 // 128 * 128:T // 2 // 128 * 128 + 128] = 0
    elif pattern == "zero but the last":
        v[:, :T - 1] = 0
    elif pattern == "small":
        v[:, T // 2 // 128 * 128 - 128:T // 2 // 128 * 128] *= 2.0 ** -16
    elif pattern == "step":
        v[:, :T // 2] *= 2.0 ** -10
        v[:, T // 2:] *= 2.0 ** 9
    elif pattern == "zero but a part":  # of the keys that thread blocks share
        v[:, :T * 3 // 8] = 0
        v[:, T * 5 // 8:] = 0
    return v


UNEVEN = [
    (1, 512, 512, 2, 1, 0, 0, None),
    (2, 515, 515, 3, 1, 200, 1, [515, 290]),
    (1, 700, 700, 4, 2, 30, 70, None),
    (1, 400, 400, 1, 1, 40, 0, None),
    # shared tiles of queries, shared blocks of keys, the sinks' blocks in a launch of their own
    (1, 100, 2500, 2, 1, 0, 0, None),
    (1, 300, 2500, 1, 1, 900, 2, [2400]),
    (1, 1100, 1100, 8, 1, 0, 0, None),
    (1, 1500, 1500, 8, 1, 300, 3, None),
    # many sequences
    (40, 260, 260, 8, 4, 0, 0, None),
]


def uneven_gradients(env, d, pattern, B, Tq, Tk, H, KV, window, sinks, lengths):
    import torch

    q, k, v, g = tensors(46, torch.float32, B, Tq, Tk, H, KV, d)
    v = put(v, pattern)
    # (max |g| max |v| stays near 20, so that dS's smallest step after its power of two, 2^-28 of that product times the scale,
    # lies below the 2^-24 that the bound has for it)
    g = g * (2.0 ** -9 if pattern == "step" else 1.0)
    q = q * (8.0 if pattern == "small" else 1.0)
    q, k, v, g = (x.half() for x in (q, k, v, g))
    some = slice(None) if B < 10 else [0, B // 2, B - 1]
    want, bound = R.window_attention(q[some], k[some], v[some], window, sinks, lengths, d ** -0.5, g[some])
    out, lse = run_forward(env, q, k, v, window, sinks, lengths)
    check((out[some], lse[some]), want, bound, ("out", "lse"))
    return [x[some] for x in run_backward(env, q, k, v, out, lse, g, window, sinks, lengths)], want, bound


PATTERNS = ["first 64 zero", "first 128 zero", "middle zero", "zero but the last", "small", "step", "zero but a part"]


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("B,Tq,Tk,H,KV,window,sinks,lengths", UNEVEN)
def test_fp16_gradients_of_keys_with_uneven_values(env, d, pattern, B, Tq, Tk, H, KV, window, sinks, lengths):
    """dK of a block of keys whose values are zero or small: rowsum(dO o O) comes from other blocks' values and is not."""
    grads, want, bound = uneven_gradients(env, d, pattern, B, Tq, Tk, H, KV, window, sinks, lengths)
    check(grads[1:], want, bound, ("dk", "dv"))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("B,Tq,Tk,H,KV,window,sinks,lengths", UNEVEN)
def test_fp16_gradients_of_queries_with_uneven_values(env, d, pattern, B, Tq, Tk, H, KV, window, sinks, lengths):
    """dQ where the first tiles of keys, or those of a thread block that shares the keys, have values of zero or small ones."""
    grads, want, bound = uneven_gradients(env, d, pattern, B, Tq, Tk, H, KV, window, sinks, lengths)
    check(grads[:1], want, bound, ("dq",))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [60, 300])
def test_offsets_beyond_32_bits(env, T, d):
    """Rows so far apart that a sequence passes 2^32 elements: all tensors as columns of one of 10 GB."""
    import torch

    H, KV, n = 4, 2, 5 << 30
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("not enough memory")
    row = n // T // 8 * 8
    wide = torch.empty(n, dtype=torch.float16, device="cuda")
    at = 0

    def column(x):
        nonlocal at
        view = wide.as_strided(x.shape, (T * row, row, d, 1), at)
        view.copy_(x)
        at += x.shape[2] * d
        return view

    made = tensors(47, torch.float16, 1, T, T, H, KV, d)
    want, bound = R.window_attention(*made[:3], 50, 1, None, d ** -0.5, made[3])
    q, k, v, g = (column(x) for x in made)
    out, dq = (column(torch.full_like(made[0], MARK)) for _ in range(2))
    dk, dv = (column(torch.full_like(made[1], MARK)) for _ in range(2))
    lse, delta = torch.empty((1, H, T), device="cuda"), torch.empty((1, H, T), device="cuda")
    wa = env.pkg().WindowAttention(env.ctx(), 50, 1)
    wa.forward(q, k, v, out, lse)
    wa.backward(q, k, v, out, lse, g, dq, dk, dv, delta)
    env.ctx().sync()
    check((out, lse, dq, dk, dv), want, bound, ("out", "lse", "dq", "dk", "dv"))
