"""The paged cache: appending, copying, attention of one new token, against plain forms in 64 bits, and all operators for long
contexts together as a program uses them."""
import math

import pytest

from tests import long_context_ref as R
from tests.test_gpu_rope import turned, types

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from tests import gpu_util as U

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return U


def pages_of(shape, dtype, seed, order="pshd"):
    """Two tensors [pages][size][heads][dim], in memory in the given order (`s`: places, `h`: heads)."""
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    p, s, h, d = shape
    make = lambda: torch.randn((p, h, s, d), device="cuda", generator=g).to(dtype).transpose(1, 2) if order == "phsd" else torch.randn(shape, device="cuda", generator=g).to(dtype)  # noqa: E731
    return make(), make()


def table_for(lengths, size, pages, seed, width=None, fill=-1):
    import torch

    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // size)) for n in lengths]
    order = torch.randperm(pages, generator=g).tolist()
    width = width or max(max(need), 1)
    t = torch.full((len(lengths), width), fill, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    assert at <= pages
    return t.cuda()


# ------------------------------------------------------------------------------------------------ append
@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["pshd", "phsd"])
@pytest.mark.parametrize("rope,size,kv,heads,dim", [(True, 16, 2, 4, 64), (True, 1, 1, 1, 64), (False, 24, 3, 0, 128), (True, 100, 8, 8, 128), (False, 7, 1, 2, 72)])
def test_append(env, kind, order, rope, size, kv, heads, dim):
    import torch

    U, pk = env, env.pkg()
    dtype = types()[kind]
    counts, had = [1, 0, 37, 5], [3, 2, 0, 2 * size - 1]
    lengths = [a + b for a, b in zip(counts, had)]
    pages = sum(-(-n // size) for n in lengths) + 2
    kp, vp = pages_of((pages, size, kv, dim), dtype, 1, order)
    before_k, before_v = kp.clone(), vp.clone()
    table = table_for(lengths, size, pages, 2)
    n = sum(counts)
    seqs = torch.tensor([s for s, c in enumerate(counts) for _ in range(c)], device="cuda").int()
    positions = torch.tensor([had[s] + i for s, c in enumerate(counts) for i in range(c)], device="cuda").int()
    mixed = torch.randperm(n, generator=torch.Generator().manual_seed(4)).cuda()
    seqs, positions = seqs[mixed].contiguous(), positions[mixed].contiguous()
    positions[n // 2] = -1  # padding
    row = torch.randn((n, heads + 2 * kv, dim), device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(dtype)
    q, k, v = row[:, :heads], row[:, heads:heads + kv], row[:, heads + kv:]
    q_out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda") if heads else None
    plan = pk.RopePlan(U.ctx(), dim) if rope else None
    cache = pk.PagedCache(U.ctx(), kp, vp)
    cache.append(k, v, positions, table, seqs=seqs, rope=plan, q=q if heads else None, q_out=q_out)
    U.ctx().sync()
    there = positions >= 0
    at = positions[there].long()
    page, place = table[seqs[there].long(), at // size].long(), at % size
    freq = plan.frequencies() if rope else [0.0] * (dim // 2)
    want, bound = turned(k[there], positions[there], freq, dim, False, 1.0, 1)
    assert R.worst(kp[page, place], want, bound) <= 1.0 and torch.equal(vp[page, place], v[there])
    if not rope:
        assert torch.equal(kp[page, place], k[there])
    before_k[page, place], before_v[page, place] = kp[page, place], vp[page, place]
    assert torch.equal(kp, before_k) and torch.equal(vp, before_v), "places that no token has were written"
    if heads:
        want, bound = turned(q[there], positions[there], freq, dim, False, 1.0, 1)
        assert R.worst(q_out[there], want, bound) <= 1.0
        assert (q_out[~there] == 7.0).all()


@gpu
def test_append_leaves_out_what_has_no_place(env):
    """Table entries and positions that lead nowhere: the other tokens are written, the next sync says so, once."""
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    kp, vp = pages_of((4, 4, 1, 64), torch.float16, 1)
    table = torch.tensor([[0, -1], [1, 4], [2, 3]], device="cuda").int()
    k = torch.randn((4, 1, 64), device="cuda").half()
    for seqs, positions, bad in (([0, 1, 2, 2], [5, 0, 1, 7], [0]), ([1, 1, 2, 2], [4, 0, 1, 7], [0]), ([0, 1, 2, 2], [0, 1, 8, 7], [2]), ([3, 1, -1, 2], [0, 1, 1, 7], [0, 2])):
        before = kp.clone()
        pk.PagedCache(ctx, kp, vp).append(k, k, torch.tensor(positions, device="cuda").int(), table, seqs=torch.tensor(seqs, device="cuda").int())
        with pytest.raises(pk.AigError) as e:
            ctx.sync()
        assert e.value.code == -1
        ctx.sync()
        for i, (s, p) in enumerate(zip(seqs, positions)):
            if i not in bad:
                before[table[s, p // 4].item(), p % 4] = k[i]
        assert torch.equal(kp, before)


# ------------------------------------------------------------------------------------------------ copies
@gpu
@pytest.mark.parametrize("order", ["pshd", "phsd"])
@pytest.mark.parametrize("pages,size,kv,dim,n", [(8, 1, 1, 8, 3), (64, 16, 8, 64, 20), (40, 100, 3, 128, 11), (2600, 2, 1, 64, 1203), (16, 16, 8, 64, 0), (5000, 1, 1, 8, 2101)])
def test_copy_pages(env, order, pages, size, kv, dim, n):
    import torch

    U, pk = env, env.pkg()
    kp, vp = pages_of((pages, size, kv, dim), torch.bfloat16, 3, order)
    wide_k, wide_v = (torch.randn((pages, size, kv + 1, dim), device="cuda").bfloat16() for _ in range(2))
    mixed = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = mixed[:n], mixed[n:2 * n]
    src = [src[0]] * (n // 2) + src[n // 2:] if n else src  # a page that several sequences forked from
    for a, b in ((kp, vp), (wide_k[:, :, :kv], wide_v[:, :, :kv])):
        want = [x.clone() for x in (a, b)]
        for w, x in zip(want, (a, b)):
            if n:
                w[dst] = x[src]
        rest = wide_k[:, :, kv].clone()
        pk.PagedCache(U.ctx(), a, b).copy_pages(src, dst)
        U.ctx().sync()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(wide_k[:, :, kv], rest)


@gpu
def test_copy_refusals(env):
    import torch

    U, pk = env, env.pkg()
    kp, vp = pages_of((8, 4, 2, 64), torch.float16, 3)
    cache = pk.PagedCache(U.ctx(), kp, vp)
    before = kp.clone()
    for src, dst in (([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0, 1], [1, 3]), ([0], [0]), ([8], [1]), ([-1], [1]), ([0], [8]), ([0], [-1])):
        with pytest.raises(pk.AigError):
            cache.copy_pages(src, dst)
    with pytest.raises(ValueError):
        cache.copy_pages([0, 1], [2])
    U.ctx().sync()
    assert torch.equal(kp, before)


# ------------------------------------------------------------------------------------------------ attention of one token
def attend_ref(q, kp, vp, table, lengths, window, sinks, scale):
    """(values, bounds): a rounding of the result; sums and weights in 32 bits."""
    import torch

    B, H, d = q.shape
    size, kv = kp.shape[1], kp.shape[2]
    G, u = H // kv, R.unit(q.dtype)
    out = torch.zeros((B, H, d), dtype=torch.float64, device="cuda")
    e = torch.full_like(out, 1e-30)
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        at = torch.arange(n, device="cuda")
        if 0 < window < n:
            at = at[(at >= n - window) | (at < sinks)]
        where = table[b, at // size].long(), at % size
        k, v = (x[where].double().repeat_interleave(G, 1) for x in (kp, vp))
        s = (k * q[b].double()).sum(-1) * scale
        big = ((k * q[b].double()).abs().sum(-1) * scale).amax(0) + 1
        w = torch.softmax(s, 0)[..., None]
        out[b] = (w * v).sum(0)
        # the weights enter as two 16-bit values: off by a step of a step, and by fp16's smallest
        e[b] = u * out[b].abs() + (2 * R.SLACK * big[:, None] + 2 * u * u) * (w * v.abs()).sum(0) + 2.0 ** -24 * v.abs().sum(0) / max(1, len(at)) * 2 + 2.0 ** -25
    return out, e


ATTEND = [
    # lengths, heads, kv_heads, page size, window, sinks
    ([1], 1, 1, 16, 0, 0),
    ([64], 8, 8, 16, 64, 0),
    ([0, 1, 2, 15, 16, 17], 4, 2, 16, 0, 0),
    ([300, 1, 77, 0, 129], 6, 2, 16, 50, 3),
    ([1000, 3], 8, 1, 1, 0, 0),
    ([513], 16, 1, 24, 100, 130),
    ([700, 699], 20, 1, 100, 0, 0),
    ([5000], 2, 2, 64, 0, 0),
    ([2100, 40], 36, 2, 64, 1, 1),
    ([90] * 70, 8, 8, 16, 33, 0),
]


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,heads,kv,size,window,sinks", ATTEND)
def test_attend(env, kind, d, lengths, heads, kv, size, window, sinks):
    import torch

    U, pk = env, env.pkg()
    dtype = types()[kind]
    need = sum(max(0, -(-n // size)) for n in lengths)
    kp, vp = pages_of((need + 3, size, kv, d), dtype, heads + d, "phsd" if heads % 4 else "pshd")
    table = table_for(lengths, size, need + 3, 6, width=max(max(-(-n // size) for n in lengths), 1) + 2, fill=-7)
    q = torch.randn((len(lengths), heads, d), device="cuda", generator=torch.Generator("cuda").manual_seed(8)).to(dtype)
    want, bound = attend_ref(q, kp, vp, table, lengths, window, sinks, d ** -0.5)
    # what no query sees may be anything: free pages, places behind the last position, positions that the window has left
    seen = torch.zeros(kp.shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        at = torch.arange(max(n, 0), device="cuda")
        at = at[(at >= n - window) | (at < sinks)] if window else at
        seen[table[b, at // size].long(), at % size] = True
    for x in (kp, vp):
        x[~seen] = torch.where(torch.rand((int((~seen).sum()), kv, d), device="cuda") < 0.5, math.nan, math.inf).to(dtype)
    for b, n in enumerate(lengths):  # entries of pages without a visible position
        for p in range(-(-n // size)):
            first, last = p * size, min(n, (p + 1) * size) - 1
            if window and last < n - window and first >= sinks:
                table[b, p] = [-1, 1 << 30][p % 2]
    n_dev = torch.tensor(lengths, device="cuda").int()
    cache = pk.PagedCache(U.ctx(), kp, vp)
    wide = torch.full((len(lengths), heads + 1, d), 7.0, dtype=dtype, device="cuda")
    for most in {max(lengths), 1, 10 ** 6}:  # the host's bound only splits the work
        cache.attend(q, wide[:, :heads], table, n_dev, most, window=window, sinks=sinks)
        U.ctx().sync()
        assert R.worst(wide[:, :heads], want, bound) <= 1.0, most
        assert (wide[:, heads] == 7.0).all()


@gpu
def test_attend_beyond_the_table_and_bad_pages(env):
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    kp, vp = pages_of((4, 4, 1, 64), torch.float16, 1)
    cache = pk.PagedCache(ctx, kp, vp)
    q = torch.randn((2, 1, 64), device="cuda").half()
    out = torch.empty_like(q)
    for table, lengths in (([[0, 1], [2, 3]], [9, 4]), ([[0, 4], [2, 3]], [8, 4]), ([[-1, 1], [2, 3]], [8, 4])):
        table, n = torch.tensor(table, device="cuda").int(), torch.tensor(lengths, device="cuda").int()
        cache.attend(q, out, table, n, 16)
        with pytest.raises(pk.AigError) as e:
            ctx.sync()
        assert e.value.code == -1
        ctx.sync()
        want, bound = attend_ref(q[1:], kp, vp, table[1:], [4], 0, 0, 0.125)
        assert R.worst(out[1:], want, bound) <= 1.0  # the other sequence has its result


@gpu
def test_offsets_beyond_32_bits(env):
    """A cache of 5 GB in each tensor: pages whose elements lie behind 2^31."""
    import torch

    U, pk = env, env.pkg()
    pages, size, kv, d = 20000, 16, 64, 128  # 2.6e9 elements
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("not enough memory")
    kp, vp = (torch.empty((pages, size, kv, d), dtype=torch.float16, device="cuda") for _ in range(2))
    use = [19999, 3, 19000, 16500]
    for x in (kp, vp):
        x[use] = torch.randn((4, size, kv, d), device="cuda").half()
    table = torch.tensor([use[:2], use[2:]], device="cuda").int()
    q = torch.randn((2, kv, d), device="cuda").half()
    out = torch.empty_like(q)
    cache = pk.PagedCache(U.ctx(), kp, vp)
    cache.attend(q, out, table, torch.tensor([32, 30], device="cuda").int(), 32)
    new = torch.randn((2, kv, d), device="cuda").half()
    cache.append(new, new, torch.tensor([15, 31], device="cuda").int(), table)
    U.ctx().sync()
    assert torch.equal(kp[19999, 15], new[0]) and torch.equal(vp[16500, 15], new[1])
    kp[19999, 15], vp[19999, 15] = kp[3, 0], vp[3, 0]
    cache.copy_pages([19999, 3], [17000, 19998])
    U.ctx().sync()
    assert torch.equal(kp[17000], kp[19999]) and torch.equal(vp[19998], vp[3])
    cache.attend(q, out, table, torch.tensor([32, 30], device="cuda").int(), 32)
    U.ctx().sync()
    want, bound = attend_ref(q, kp, vp, table, [32, 30], 0, 0, d ** -0.5)
    assert R.worst(out, want, bound) <= 1.0


@gpu
def test_attend_refusals(env):
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    kp, vp = pages_of((4, 4, 2, 64), torch.float16, 1)
    cache = pk.PagedCache(ctx, kp, vp)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    table, n = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for args in ((q.bfloat16(), q, table, n, 4), (q, q[:1], table, n, 4), (q, q, table[:1], n, 4), (q, q, table, n[:1], 4), (q, q, table.long(), n, 4), (q[..., :32], q[..., :32], table, n, 4)):
        with pytest.raises(ValueError):
            cache.attend(*args)
    for change in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(sinks=-1)):
        with pytest.raises(pk.AigError):
            cache.attend(q, q.clone(), table, n, 4, **change)
    odd = torch.zeros((2, 3, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(pk.AigError):
        cache.attend(odd, odd.clone(), table, n, 4)  # three query heads over two cached ones
    k80 = torch.zeros((4, 4, 2, 80), dtype=torch.float16, device="cuda")
    q80 = torch.zeros((2, 4, 80), dtype=torch.float16, device="cuda")
    with pytest.raises(pk.AigError) as e:
        pk.PagedCache(ctx, k80, k80.clone()).attend(q80, q80.clone(), table, n, 4)
    assert e.value.code == -4
    flat = torch.zeros(2 * 4 * 64 + 8, dtype=torch.float16, device="cuda")
    with pytest.raises(pk.AigError):
        cache.attend(flat[1:513].view(2, 4, 64), q, table, n, 4)  # off a 16-byte boundary
    for k, v in ((kp, vp.bfloat16()), (kp, vp[:3]), (kp.float(), vp.float()), (kp, vp.transpose(1, 2).contiguous().transpose(1, 2)), (kp[0], vp[0])):
        with pytest.raises(ValueError):
            pk.PagedCache(ctx, k, v)
    with pytest.raises(pk.AigError):
        pk.PagedCache(ctx, k80[..., :68], k80[..., :68]).copy_pages([0], [1])  # 68 is no multiple of 8
    ctx.sync()


# ------------------------------------------------------------------------------------------------ together
@gpu
def test_a_program_with_all_of_it(env):
    """Prompts through the windowed attention and into pages, then steps: sequences forked, trimmed behind their window, closed,
    the cache compacted.  Every step's output equals the windowed attention over the sequence as a whole."""
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    H, KV, d, size, window, sinks = 4, 2, 64, 8, 24, 3
    g = torch.Generator("cuda").manual_seed(0)
    pool, rope = pk.PagePool(64, size), pk.RopePlan(ctx, d, base=10000.0)
    kp, vp = pages_of((64, size, KV, d), torch.float16, 9)
    kp[:], vp[:] = math.nan, math.nan
    cache, attention = pk.PagedCache(ctx, kp, vp), pk.WindowAttention(ctx, window, sinks)
    width = 16
    history = {}  # sequence -> its rows [tokens][H + 2 KV][d] before they are turned

    def tables(seqs):
        return torch.tensor([pool.table(s, width) for s in seqs], device="cuda").int()

    def whole(rows):
        """The last row's output over all of them, and every row's."""
        n = rows.shape[0]
        q, k, v = rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:]
        at = torch.arange(n, device="cuda").int()
        qt, kt = torch.empty_like(q), torch.empty_like(k)
        rope.forward(at, q, qt, k, kt)
        out, lse = torch.empty((1, n, H, d), dtype=torch.float16, device="cuda"), torch.empty((1, H, n), device="cuda")
        attention.forward(qt[None], kt[None], v[None], out, lse)
        ctx.sync()
        want, bound = R.window_attention(qt[None], kt[None], v[None], window, sinks, None, d ** -0.5)
        assert R.worst(out, want["out"], bound["out"]) <= 1.0
        return want["out"][0, -1], bound["out"][0, -1]

    def step(seqs, counts):
        rows = [torch.randn((c, H + 2 * KV, d), device="cuda", generator=g).half() for c in counts]
        for s, c in zip(seqs, counts):
            pair = pool.grow(s, c)
            if pair:
                cache.copy_pages([pair[0]], [pair[1]])
        t = tables(seqs)
        row = torch.cat(rows)
        of = torch.tensor([i for i, c in enumerate(counts) for _ in range(c)], device="cuda").int()
        at = torch.tensor([len(history[s]) + i for s, c in zip(seqs, counts) for i in range(c)], device="cuda").int()
        q_out = torch.empty_like(row[:, :H])
        cache.append(row[:, H:H + KV], row[:, H + KV:], at, t, seqs=of, rope=rope, q=row[:, :H], q_out=q_out)
        for s, r in zip(seqs, rows):
            history[s] = torch.cat((history[s], r))
        last = (torch.tensor(counts).cumsum(0) - 1).cuda()
        lengths = torch.tensor([pool.length(s) for s in seqs], device="cuda").int()
        out = torch.empty((len(seqs), H, d), dtype=torch.float16, device="cuda")
        cache.attend(q_out[last].contiguous(), out, t, lengths, width * size, window=window, sinks=sinks)
        ctx.sync()
        for i, s in enumerate(seqs):
            want, bound = whole(history[s])
            assert R.worst(out[i], want, bound) <= 1.0
            pool.trim(s, window, sinks)

    none = torch.empty((0, H + 2 * KV, d), dtype=torch.float16, device="cuda")
    seqs = [pool.open() for _ in range(3)]
    history.update({s: none for s in seqs})
    step(seqs, [37, 5, 16])
    for i in range(6):
        step(seqs, [1, 1, 1])
    fork = pool.fork(seqs[0])
    history[fork] = history[seqs[0]]
    seqs.append(fork)
    for i in range(10):
        step(seqs, [1, 1, 1, 1])
    pool.close_sequence(seqs[1])
    del history[seqs[1]], seqs[1]
    src, dst = pool.compact(64)
    assert src
    cache.copy_pages(src, dst)
    for i in range(9):
        step(seqs, [1, 2, 1])
    pool.close()
    rope.close()


@gpu
def test_captured_steps_and_other_streams(env):
    """A step captured into two graphs that are replayed in turn, and calls on a context with a stream of its own."""
    import torch

    U, pk = env, env.pkg()
    main = U.ctx()
    for ctx in (main, pk.Context(0, use_torch_stream=False)):
        rope = pk.RopePlan(ctx, 64)
        kp, vp = pages_of((12, 16, 2, 64), torch.float16, 2)
        cache = pk.PagedCache(ctx, kp, vp)
        table = torch.arange(12, device="cuda").int().view(2, 6)
        row = torch.randn((2, 8, 64), device="cuda").half()
        q_out, out = torch.empty((2, 4, 64), dtype=torch.float16, device="cuda"), torch.empty((2, 4, 64), dtype=torch.float16, device="cuda")
        positions, lengths = torch.tensor([40, 70], device="cuda").int(), torch.tensor([41, 71], device="cuda").int()
        torch.cuda.synchronize()

        def step():
            cache.append(row[:, 4:6], row[:, 6:], positions, table, rope=rope, q=row[:, :4], q_out=q_out)
            cache.attend(q_out, out, table, lengths, 96, window=30, sinks=2)

        step()
        ctx.sync()
        graphs = []
        for _ in range(2):
            ctx.graph_begin()
            step()
            graphs.append(ctx.graph_end())
        for i in range(4):
            row.normal_()
            positions.add_(1)
            lengths.add_(1)
            torch.cuda.synchronize()
            ctx.graph_launch(graphs[i % 2])
            ctx.sync()
            want, bound = turned(row[:, :4], positions, rope.frequencies(), 64, False, 1.0, 1)
            assert R.worst(q_out, want, bound) <= 1.0
            want, bound = attend_ref(q_out, kp, vp, table, lengths.tolist(), 30, 2, 0.125)
            assert R.worst(out, want, bound) <= 1.0
        for g in graphs:
            pk.lib().aig_graph_destroy(g)
        rope.close()
        if ctx is not main:
            ctx.close()


def kept_ref(q, kp, vp, where, scale):
    """attend_ref of one sequence over these (page, place) pairs alone."""
    import torch

    n = len(where)
    page, place = (torch.tensor(x, device="cuda") for x in zip(*where))
    return attend_ref(q, kp[page, place][:, None], vp[page, place][:, None], torch.arange(n, device="cuda")[None], [n], 0, 0, scale)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("finite", [False, True])
@pytest.mark.parametrize("heads,kv", [(2, 2), (12, 1)])
@pytest.mark.parametrize("hidden", ["first", "last", "all but one", "between"])
def test_attend_scores_of_minus_infinity(env, hidden, heads, kv, finite, d):
    """Keys of minus infinity, or finite ones whose product passes 32 bits: weights of 0, wherever they lie; where no other key
    is visible the formula has no value."""
    import torch

    U, pk = env, env.pkg()
    size, n = 16, 700
    kp, vp = pages_of((60, size, kv, d), torch.bfloat16, 17)
    table = table_for([n, 40], size, 60, 18)
    q = torch.randn((2, heads, d), device="cuda", generator=torch.Generator("cuda").manual_seed(19)).bfloat16()
    q[:, :, 0] = 1e20 if finite else 1.0
    kp[..., 0] = 0
    gone = {"first": lambda t: t < 400, "last": lambda t: t >= 300, "all but one": lambda t: t != 555, "between": lambda t: t % 64 >= 16}[hidden]
    place = lambda t: (int(table[0, t // size]), t % size)  # noqa: E731
    for t in filter(gone, range(n)):
        kp[place(t)][:, 0] = -1e30 if finite else -math.inf
    for t in range(40):  # the other sequence has no other keys
        kp[int(table[1, t // size]), t % size][:, 0] = -1e30 if finite else -math.inf
    out = torch.empty_like(q)
    lengths = torch.tensor([n, 40], device="cuda").int()
    want, bound = kept_ref(q[:1], kp, vp, [place(t) for t in range(n) if not gone(t)], d ** -0.5)
    cache = pk.PagedCache(U.ctx(), kp, vp)
    for most in (1, n):
        cache.attend(q, out, table, lengths, most)
        U.ctx().sync()
        assert R.worst(out[:1], want, bound) <= 1.0
        assert out[1].isnan().all()


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size,bad", [(16, [0]), (16, [3, 40]), (7, [1, 2, 50]), (100, [2]), (16, list(range(43))), (16, list(range(44)))])
def test_attend_leaves_out_pages_that_are_none(env, size, bad, d):
    """Positions whose table entry names no page have no share in the softmax; with no other position the result is zeros."""
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    n, pages = 700, 110
    kp, vp = pages_of((pages, size, 2, d), torch.float16, 21)
    kp *= 3  # (a score of 0 would take a visible share)
    table = table_for([n], size, pages, 22)
    where = [(int(table[0, t // size]), t % size) for t in range(n) if t // size not in bad]
    for i, p in enumerate(bad):
        table[0, p] = [-1, pages, 1 << 30][i % 3]
    q = torch.randn((1, 8, d), device="cuda", generator=torch.Generator("cuda").manual_seed(23)).half()
    out = torch.full_like(q, 7.0)
    for most in (1, n):
        pk.PagedCache(ctx, kp, vp).attend(q, out, table, torch.tensor([n], device="cuda").int(), most)
        with pytest.raises(pk.AigError) as e:
            ctx.sync()
        assert e.value.code == -1
        if where:
            want, bound = kept_ref(q, kp, vp, where, d ** -0.5)
            assert R.worst(out, want, bound) <= 1.0
        else:
            assert not out.any()


@gpu
@pytest.mark.parametrize("heads", [2, 64])
def test_append_turns_queries_of_tokens_without_a_place(env, heads):
    """A place that is none leaves out the token's keys and values; its queries are turned like the others'."""
    import torch

    U, pk = env, env.pkg()
    ctx = U.ctx()
    n = 3000 if heads > 2 else 5  # (enough for several heads a thread, and few)
    kp, vp = pages_of((n, 1, 1, 64), torch.float16, 25)
    table = torch.arange(n, device="cuda").int()[None].contiguous()
    table[0, 1], table[0, 3] = -1, n
    positions = torch.arange(n, device="cuda").int()
    positions[4] = n  # beyond the table
    positions[2] = -1
    seqs = torch.zeros(n, dtype=torch.int32, device="cuda")
    seqs[0] = 1
    row = torch.randn((n, heads + 2, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(26)).half()
    q, k, v = row[:, :heads], row[:, heads:heads + 1], row[:, heads + 1:]
    q_out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    before_k, before_v = kp.clone(), vp.clone()
    rope = pk.RopePlan(ctx, 64)
    pk.PagedCache(ctx, kp, vp).append(k, v, positions, table, seqs=seqs, rope=rope, q=q, q_out=q_out)
    with pytest.raises(pk.AigError) as e:
        ctx.sync()
    assert e.value.code == -1
    there = positions >= 0
    want, bound = turned(q[there], positions[there], rope.frequencies(), 64, False, 1.0, 1)
    assert R.worst(q_out[there], want, bound) <= 1.0
    assert (q_out[2] == 7.0).all()
    want, bound = turned(k, positions, rope.frequencies(), 64, False, 1.0, 1)
    assert R.worst(kp[5:, 0], want[5:], bound[5:]) <= 1.0 and torch.equal(vp[5:, 0], v[5:])
    assert torch.equal(kp[:5], before_k[:5]) and torch.equal(vp[:5], before_v[:5])
    rope.close()
