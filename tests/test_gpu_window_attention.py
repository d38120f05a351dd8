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
