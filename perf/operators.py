"""Attention over long contexts as measurable cases: rotary positions, a paged key/value cache with the attention of one new
token that reads it, and attention over whole sequences with a sliding window and first tokens that stay visible, forward
and backward.

Every case has a `kind`:

  rope     queries and keys turned by their positions, or gradients turned back (RopePlan.forward / backward)
  append   new keys and values written into their pages, keys and queries turned on the way (PagedCache.append)
  copy     pages of a cache copied: a forked sequence's last pages, a compaction (PagedCache.copy_pages)
  attend   one new token for each sequence over its pages (PagedCache.attend)
  forward  attention over whole sequences, or over a prompt's last part (WindowAttention.forward)
  train    the same with its gradients (WindowAttention.forward and backward)

With `own` false `run` computes the same values from elementary torch operations in 32 bits, angles in 64.
"""
import importlib
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_shared = {}


def _pkg():
    return importlib.import_module("ai-gamer_b200")


def _ctx():
    if "ctx" not in _shared:
        _shared["ctx"] = _pkg().Context(0)
    return _shared["ctx"]


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a training batch of the sequence head: 128 sequences of 64 frames, eight heads of 64
        {"name": "rope_b128_t64", "kind": "rope", "type": "f16", "tokens": 8192, "heads": 8, "kv_heads": 8, "dim": 64, "rot": 64,
         "interleaved": False, "base": 10000.0, "scaling": "plain", "factor": 1.0, "original": 0, "far": 64, "backward": False},
        # a long context's gradients: far positions, neighbouring pairs, three quarters of the head, frequencies scaled by parts
        {"name": "rope_far_backward", "kind": "rope", "type": "bf16", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 96,
         "interleaved": True, "base": 500000.0, "scaling": "ramp", "factor": 16.0, "original": 8192, "far": 1000000, "backward": True},
        # a handful of players: one token each into pages of 16
        {"name": "append_b6", "kind": "append", "type": "f16", "batch": 6, "new": 1, "most": 64, "heads": 8, "kv_heads": 8, "dim": 64, "page": 16},
        # prompts of eight requests, 500 to 4000 tokens, into pages of 64
        {"name": "append_prompts", "kind": "append", "type": "bf16", "batch": 8, "new": 4001, "most": 4001, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # six sequences forked: the page that each writes to next is copied
        {"name": "copy_fork6", "kind": "copy", "type": "f16", "pages": 512, "copied": 6, "kv_heads": 8, "dim": 64, "page": 16},
        # a cache compacted: a thousand pages move
        {"name": "copy_compact", "kind": "copy", "type": "bf16", "pages": 4096, "copied": 1021, "kv_heads": 8, "dim": 128, "page": 32},
        # a live player: one frame, 64 frames of context
        {"name": "attend_b1", "kind": "attend", "type": "f16", "batch": 1, "least": 64, "most": 64, "heads": 8, "kv_heads": 8, "dim": 64, "page": 16,
         "window": 64, "sinks": 0},
        # a server stepping 128 players who joined at different times, the last 512 frames and the first four visible
        {"name": "attend_b128", "kind": "attend", "type": "f16", "batch": 128, "least": 1, "most": 2000, "heads": 8, "kv_heads": 8, "dim": 64, "page": 16,
         "window": 512, "sinks": 4},
        # a few very long contexts of unequal length, four query heads to a cached one
        {"name": "attend_long", "kind": "attend", "type": "bf16", "batch": 8, "least": 1, "most": 65536, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "sinks": 0},
        # the sequence head's attention over whole recorded sequences
        {"name": "forward_b128_t64", "kind": "forward", "type": "f16", "batch": 128, "q_len": 64, "kv_len": 64, "ragged": False, "heads": 8, "kv_heads": 8,
         "dim": 64, "window": 0, "sinks": 0},
        # a long prompt with a window of half its length and four sinks
        {"name": "forward_t8192", "kind": "forward", "type": "bf16", "batch": 1, "q_len": 8192, "kv_len": 8192, "ragged": False, "heads": 16, "kv_heads": 4,
         "dim": 128, "window": 4096, "sinks": 4},
        # training on two recordings of unequal length, two query heads to a key head
        {"name": "train_b2_t4099", "kind": "train", "type": "f16", "batch": 2, "q_len": 4099, "kv_len": 4099, "ragged": True, "heads": 16, "kv_heads": 8,
         "dim": 64, "window": 1024, "sinks": 2},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= most]), kv


def draw(rng):
    kind = rng.choice(["rope", "append", "copy", "attend", "attend", "forward", "forward", "train", "train"])
    c = {"kind": kind, "type": rng.choice(["f16", "bf16"])}
    dim = rng.choice([64, 128])
    if kind == "rope":
        heads, kv = _heads(rng, 32)
        scaling = rng.choice(["plain", "linear", "ramp", "turns"])
        return {**c, "tokens": _log_int(rng, 1, 16384 * 4096 // (4096 + heads * dim)), "heads": heads, "kv_heads": kv, "dim": dim,
                "rot": rng.choice([dim, dim // 2, 2 * rng.randint(4, dim // 2)]), "interleaved": rng.random() < 0.5,
                "base": rng.choice([10000.0, 500000.0]), "scaling": scaling, "factor": 1.0 if scaling == "plain" else rng.choice([2.0, 8.0, 40.0]),
                "original": 0 if scaling == "plain" else rng.choice([2048, 8192]), "far": _log_int(rng, 64, 4000000), "backward": rng.random() < 0.5}
    if kind == "append":
        heads, kv = _heads(rng, 32)
        batch = _log_int(rng, 1, 128)
        most = _log_int(rng, 1, min(4001, 32768 // batch))
        return {**c, "batch": batch, "new": 1 if rng.random() < 0.5 else most, "most": most, "heads": heads, "kv_heads": kv, "dim": dim,
                "page": rng.choice([1, 16, 24, 64, 100])}
    if kind == "copy":
        page, kv = rng.choice([1, 16, 24, 64]), rng.choice([1, 2, 4, 8])
        pages = _log_int(rng, 8, min(20000, 4096 * 32 * 8 * 128 // (page * kv * dim)))
        return {**c, "pages": pages, "copied": _log_int(rng, 1, pages // 4), "kv_heads": kv, "dim": dim, "page": page}
    if kind == "attend":
        heads, kv = _heads(rng, 32)
        batch = _log_int(rng, 1, 128)
        most = _log_int(rng, 1, min(65536, 262144 // batch))
        window = 0 if rng.random() < 0.4 else _log_int(rng, 1, most)
        return {**c, "batch": batch, "least": rng.choice([0, 1, most]), "most": most, "heads": heads, "kv_heads": kv, "dim": dim,
                "page": rng.choice([1, 16, 24, 64, 100]), "window": window, "sinks": rng.choice([0, 1, 4, 64]) if window else 0}
    heads, kv = _heads(rng, 16)
    t = _log_int(rng, 1, 4099)
    window = 0 if rng.random() < 0.4 else _log_int(rng, 1, t)
    return {**c, "batch": _log_int(rng, 1, max(1, min(128, 2 * 16 * 4099 * 4099 // (heads * t * t)))), "q_len": t if rng.random() < 0.7 else rng.randint(1, t), "kv_len": t,
            "ragged": rng.random() < 0.5, "heads": heads, "kv_heads": kv, "dim": dim, "window": window, "sinks": rng.choice([0, 1, 4, 130]) if window else 0}


# ------------------------------------------------------------------------------------------------ lengths, known from the case alone
def _attend_lengths(c):
    """Lengths spread evenly from `least` to `most`."""
    n = c["batch"]
    return [c["most"] if n == 1 else c["least"] + (c["most"] - c["least"]) * i // (n - 1) for i in range(n)]


def _append_counts(c):
    """(tokens that each sequence gets, tokens that it had): one step on contexts of up to `most`, or prompts of up to `new`."""
    n = c["batch"]
    if c["new"] == 1:
        return [1] * n, [(c["most"] - 1) * (i + 1) // n for i in range(n)]
    return [max(1, c["new"] * (i + 1) // n) - (i % 3 if c["new"] > 3 * n else 0) for i in range(n)], [0] * n


def _sequence_lengths(c):
    n = c["batch"]
    return [c["kv_len"] - (c["kv_len"] * i // (2 * n) if c["ragged"] else 0) for i in range(n)]


def _visible(p, window, sinks):
    """Keys that a query at position p sees."""
    return min(p + 1, window) + min(sinks, max(0, p + 1 - window)) if window else p + 1


# ------------------------------------------------------------------------------------------------ states
class _State:
    pass


def _scaling(pkg, name):
    return {"plain": pkg.ROPE_PLAIN, "linear": pkg.ROPE_LINEAR, "ramp": pkg.ROPE_RAMP, "turns": pkg.ROPE_TURNS}[name]


def _prepare_rope(s, c, randn, g):
    dt, n = TYPES[c["type"]], c["tokens"]
    # queries and keys as a fused projection leaves them: columns of one row per token
    s.row = randn(n, c["heads"] + c["kv_heads"], c["dim"]).to(dt)
    s.q, s.k = s.row[:, :c["heads"]], s.row[:, c["heads"]:]
    s.q_out, s.k_out = torch.empty(s.q.shape, dtype=dt, device="cuda"), torch.empty(s.k.shape, dtype=dt, device="cuda")
    s.positions = torch.randint(0, c["far"], (n,), device="cuda", generator=g).int()
    if own:
        s.rope = _pkg().RopePlan(_ctx(), c["dim"], rot_dim=c["rot"], interleaved=c["interleaved"], base=c["base"], scaling=_scaling(_pkg(), c["scaling"]),
                                 factor=c["factor"], original_len=c["original"], low=1.0, high=4.0 if c["scaling"] == "turns" else 32.0)


def _pages(s, c, randn, pages):
    dt = TYPES[c["type"]]
    shape = (pages, c["page"], c["kv_heads"], c["dim"])
    s.k_pages, s.v_pages = randn(*shape).to(dt), randn(*shape).to(dt)
    if own:
        s.cache = _pkg().PagedCache(_ctx(), s.k_pages, s.v_pages)


def _table(s, c, lengths, g):
    """A page of the pool for each `page` tokens of a sequence, in no order; a cache has pages that nobody uses too."""
    need = [-(-n // c["page"]) for n in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, device="cuda", generator=g)[:sum(need)].int()
    width = max(max(need), 1)
    at = torch.arange(width, device="cuda")
    used = at[None] < torch.tensor(need, device="cuda")[:, None]
    s.table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    s.table[used] = order
    return total


def _prepare_append(s, c, randn, g):
    dt = TYPES[c["type"]]
    new, had = _append_counts(c)
    _pages(s, c, randn, _table(s, c, [a + b for a, b in zip(new, had)], g))
    n = sum(new)
    s.row = randn(n, c["heads"] + 2 * c["kv_heads"], c["dim"]).to(dt)
    s.q, s.k, s.v = s.row[:, :c["heads"]], s.row[:, c["heads"]:c["heads"] + c["kv_heads"]], s.row[:, c["heads"] + c["kv_heads"]:]
    s.q_out = torch.empty(s.q.shape, dtype=dt, device="cuda")
    counts = torch.tensor(new, device="cuda")
    s.seqs = torch.arange(len(new), device="cuda").repeat_interleave(counts).int()
    begin = (counts.cumsum(0) - counts - torch.tensor(had, device="cuda")).repeat_interleave(counts)
    s.positions = (torch.arange(n, device="cuda") - begin).int()
    if own:
        s.rope = _pkg().RopePlan(_ctx(), c["dim"], base=10000.0)


def _prepare_copy(s, c, randn, g):
    _pages(s, c, randn, c["pages"])
    order = torch.randperm(c["pages"], device="cuda", generator=g)
    s.src, s.dst = order[:c["copied"]].tolist(), order[c["copied"]:2 * c["copied"]].tolist()


def _prepare_attend(s, c, randn, g):
    lengths = _attend_lengths(c)
    mixed = torch.randperm(len(lengths), device="cuda", generator=g).tolist()
    lengths = [lengths[i] for i in mixed]
    _pages(s, c, randn, _table(s, c, lengths, g))
    s.lengths = torch.tensor(lengths, device="cuda").int()
    s.q = randn(c["batch"], c["heads"], c["dim"]).to(TYPES[c["type"]])
    s.out = torch.empty_like(s.q)


def _prepare_sequences(s, c, randn, g):
    dt, b, tq, tk, h, kv, d = TYPES[c["type"]], c["batch"], c["q_len"], c["kv_len"], c["heads"], c["kv_heads"], c["dim"]
    if tq == tk:  # as a fused projection leaves them
        row = randn(b, tk, h + 2 * kv, d).to(dt)
        s.q, s.k, s.v = row[:, :, :h], row[:, :, h:h + kv], row[:, :, h + kv:]
    else:
        s.q, s.k, s.v = randn(b, tq, h, d).to(dt), randn(b, tk, kv, d).to(dt), randn(b, tk, kv, d).to(dt)
    s.lengths = torch.tensor(_sequence_lengths(c), device="cuda").int() if c["ragged"] else None
    s.out = torch.zeros((b, tq, h, d), dtype=dt, device="cuda")
    s.lse = torch.zeros((b, h, tq), device="cuda")
    if c["kind"] == "train":
        s.dout = randn(b, tq, h, d).to(dt)
        s.dq, s.dk, s.dv = (torch.zeros(x.shape, dtype=dt, device="cuda") for x in (s.q, s.k, s.v))
        s.delta = torch.empty_like(s.lse)
    if own:
        s.attention = _pkg().WindowAttention(_ctx(), window=c["window"], sinks=c["sinks"])


_PREPARE = {"rope": _prepare_rope, "append": _prepare_append, "copy": _prepare_copy, "attend": _prepare_attend,
            "forward": _prepare_sequences, "train": _prepare_sequences}


def prepare(case, seed):
    if own:
        _ctx()
    g = torch.Generator("cuda").manual_seed(seed)
    s = _State()
    s.case = case
    _PREPARE[case["kind"]](s, case, lambda *shape: torch.randn(shape, device="cuda", generator=g), g)
    return s


# ------------------------------------------------------------------------------------------------ one pass: the plain forms
def _frequencies(c):
    """Radians per position of each pair, in 64 bits."""
    rot, base = c["rot"], c["base"]
    j = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    f = base ** (-2 * j / rot)
    if c["scaling"] == "linear":
        return f / c["factor"]
    if c["scaling"] == "turns":  # by the turns that a pair makes over the original length: 1 and fewer scaled, 4 and more kept
        keep = ((c["original"] * f / (2 * math.pi) - 1) / 3).clamp(0, 1)
        return f * keep + f / c["factor"] * (1 - keep)
    if c["scaling"] == "ramp":  # linear in the pair's index between the pairs that make 32 turns and one
        def at(turns):
            return rot * math.log(c["original"] / (2 * math.pi * turns)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
        scaled = ((j - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - scaled) + f / c["factor"] * scaled
    return f


def _turned(x, angle, rot, interleaved, sign):
    """x [tokens][heads][dim] in 32 bits, its first `rot` elements turned by `angle` [tokens][rot / 2]."""
    cos, sin = angle.cos().float()[:, None], (sign * angle.sin()).float()[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        t = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        t = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((t, x[..., rot:]), -1)


def _plain_rope(s, c):
    angle = s.positions.double()[:, None] * _frequencies(c)
    sign = -1.0 if c["backward"] else 1.0
    s.q_out.copy_(_turned(s.q.float(), angle, c["rot"], c["interleaved"], sign))
    s.k_out.copy_(_turned(s.k.float(), angle, c["rot"], c["interleaved"], sign))
    return s.q_out, s.k_out


def _plain_append(s, c):
    angle = s.positions.double()[:, None] * _frequencies({"rot": c["dim"], "base": 10000.0, "scaling": "plain"})
    s.q_out.copy_(_turned(s.q.float(), angle, c["dim"], False, 1.0))
    at = s.positions.long()
    page, slot = s.table[s.seqs.long(), at // c["page"]].long(), at % c["page"]
    s.k_pages[page, slot] = _turned(s.k.float(), angle, c["dim"], False, 1.0).to(s.k_pages.dtype)
    s.v_pages[page, slot] = s.v
    return s.q_out, s.k_pages, s.v_pages


def _plain_copy(s, c):
    src, dst = torch.tensor(s.src, device="cuda"), torch.tensor(s.dst, device="cuda")
    s.k_pages[dst] = s.k_pages[src]
    s.v_pages[dst] = s.v_pages[src]
    return s.k_pages, s.v_pages


def _plain_attend(s, c):
    b, kv, d = c["batch"], c["kv_heads"], c["dim"]
    group = c["heads"] // kv
    at = torch.arange(c["most"], device="cuda")
    n = s.lengths[:, None].long()
    seen = at < n
    if c["window"]:
        seen = seen & ((at >= n - c["window"]) | (at < c["sinks"]))
    page = s.table[:, at // c["page"]].long().clamp(min=0)
    k = s.k_pages[page, at % c["page"]].float()  # [batch][most][kv_heads][dim]
    score = torch.einsum("bkgd,btkd->bkgt", s.q.float().view(b, kv, group, d), k) / math.sqrt(d)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = s.v_pages[page, at % c["page"]].float().masked_fill(~seen[:, :, None, None], 0.0)
    o = torch.einsum("bkgt,btkd->bkgd", p, v) / torch.where(total > 0, total, 1.0)
    s.out.copy_(o.view(b, c["heads"], d))
    return s.out


def _sequence_mask(c, lengths):
    """(keys that each query sees [batch or 1][q][kv], queries that there are [batch or 1][q])."""
    i = torch.arange(c["q_len"], device="cuda")[:, None] + (c["kv_len"] - c["q_len"])
    j = torch.arange(c["kv_len"], device="cuda")
    seen = j <= i
    if c["window"]:
        seen = seen & ((j > i - c["window"]) | (j < c["sinks"]))
    if lengths is None:
        return seen[None], torch.ones((1, c["q_len"]), dtype=torch.bool, device="cuda")
    n = lengths.long()[:, None]
    return seen[None] & (j < n[:, :, None]), i[:, 0] < n


def _plain_forward(s, c, train):
    b, tq, h, kv, d = c["batch"], c["q_len"], c["heads"], c["kv_heads"], c["dim"]
    seen, there = _sequence_mask(c, s.lengths)
    q = s.q.float().reshape(b, tq, kv, h // kv, d)
    k, v = s.k.float(), s.v.float()
    score = torch.einsum("bqkgd,btkd->bkgqt", q, k).mul_(1 / math.sqrt(d))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    p.div_(total)
    o = torch.einsum("bkgqt,btkd->bqkgd", p, v).reshape(b, tq, h, d)
    s.out.copy_(torch.where(there[:, :, None, None], o, s.out.float()))
    s.lse.copy_(torch.where(there[:, None], (top + total.log()).reshape(b, h, tq), s.lse))
    if not train:
        return s.out, s.lse
    do = torch.where(there[:, :, None, None], s.dout.float(), 0.0).view(b, tq, kv, h // kv, d)
    dv = torch.einsum("bkgqt,bqkgd->btkd", p, do)
    dp = torch.einsum("bqkgd,btkd->bkgqt", do, v)
    ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(1 / math.sqrt(d))
    s.dq.copy_(torch.einsum("bkgqt,btkd->bqkgd", ds, k).reshape(b, tq, h, d))
    s.dk.copy_(torch.einsum("bkgqt,bqkgd->btkd", ds, q))
    s.dv.copy_(dv)
    return s.out, s.lse, s.dq, s.dk, s.dv


# ------------------------------------------------------------------------------------------------ one pass: the framework's calls
def _own(s, c):
    kind = c["kind"]
    if kind == "rope":
        (s.rope.backward if c["backward"] else s.rope.forward)(s.positions, s.q, s.q_out, s.k, s.k_out)
        return s.q_out, s.k_out
    if kind == "append":
        s.cache.append(s.k, s.v, s.positions, s.table, seqs=s.seqs, rope=s.rope, q=s.q, q_out=s.q_out)
        return s.q_out, s.k_pages, s.v_pages
    if kind == "copy":
        s.cache.copy_pages(s.src, s.dst)
        return s.k_pages, s.v_pages
    if kind == "attend":
        s.cache.attend(s.q, s.out, s.table, s.lengths, c["most"], window=c["window"], sinks=c["sinks"])
        return s.out
    s.attention.forward(s.q, s.k, s.v, s.out, s.lse, lengths=s.lengths)
    if kind == "forward":
        return s.out, s.lse
    s.attention.backward(s.q, s.k, s.v, s.out, s.lse, s.dout, s.dq, s.dk, s.dv, s.delta, lengths=s.lengths)
    return s.out, s.lse, s.dq, s.dk, s.dv


def run(s):
    c = s.case
    if own:
        return _own(s, c)
    kind = c["kind"]
    if kind == "rope":
        return _plain_rope(s, c)
    if kind == "append":
        return _plain_append(s, c)
    if kind == "copy":
        return _plain_copy(s, c)
    if kind == "attend":
        return _plain_attend(s, c)
    return _plain_forward(s, c, kind == "train")


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, kind, d = case, case["kind"], case["dim"]
    if kind == "rope":
        values = c["tokens"] * (c["heads"] + c["kv_heads"]) * d
        return {"bytes": 4.0 * values + 4.0 * c["tokens"], "flops": 3.0 * values * c["rot"] / d}
    if kind == "append":
        n = sum(_append_counts(c)[0])
        return {"bytes": n * (4.0 * (c["heads"] + 2 * c["kv_heads"]) * d + 12), "flops": 3.0 * n * (c["heads"] + c["kv_heads"]) * d}
    if kind == "copy":
        return {"bytes": 8.0 * c["copied"] * c["page"] * c["kv_heads"] * d, "flops": 0.0}
    if kind == "attend":
        seen = sum(_visible(n - 1, c["window"], c["sinks"]) if n else 0 for n in _attend_lengths(c))
        return {"bytes": 4.0 * seen * c["kv_heads"] * d + 4.0 * c["batch"] * c["heads"] * d, "flops": 4.0 * seen * c["heads"] * d}
    first = c["kv_len"] - c["q_len"]
    seen = rows = keys = 0
    for n in _sequence_lengths(c):
        seen += sum(_visible(p, c["window"], c["sinks"]) for p in range(first, n))
        rows += max(0, n - first)
        keys += n
    q_bytes, kv_bytes = 2.0 * rows * c["heads"] * d, 2.0 * keys * c["kv_heads"] * d
    forward = {"bytes": 2 * q_bytes + 2 * kv_bytes + 4.0 * rows * c["heads"], "flops": 4.0 * seen * c["heads"] * d}
    if kind == "forward":
        return forward
    # the gradients: q, k, v, the output, its gradient and the statistics read, three gradients written; five products
    return {"bytes": forward["bytes"] + 4 * q_bytes + 4 * kv_bytes + 4.0 * rows * c["heads"], "flops": forward["flops"] * 3.5}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _spin(x, positions, c, sign):
    """Each pair as a complex number times e^(i angle)."""
    rot, n = c["rot"], c["rot"] // 2
    rate = []
    for j in range(n):
        f = c["base"] ** (-2.0 * j / rot)
        turns = c["original"] * f / (2 * math.pi)
        if c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "turns":
            share = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            f = share * f + (1 - share) * f / c["factor"]
        elif c["scaling"] == "ramp":
            edge = [rot * math.log(c["original"] / (b * 2 * math.pi)) / (2 * math.log(c["base"])) for b in (32.0, 1.0)]
            lo, hi = max(0, math.floor(edge[0])), min(rot - 1, math.ceil(edge[1]))
            share = min(1.0, max(0.0, (j - lo) / (hi - lo if hi > lo else 0.001)))
            f = share * f / c["factor"] + (1 - share) * f
        rate.append(sign * f)
    phase = torch.outer(positions.double(), torch.tensor(rate, dtype=torch.float64, device="cuda"))[:, None]
    x = x.double()
    first, second = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["interleaved"] else (x[..., :n], x[..., n:rot])
    z = torch.complex(first.contiguous(), second.contiguous()) * torch.polar(torch.ones_like(phase), phase)
    out = x.clone()
    if c["interleaved"]:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        out[..., :n], out[..., n:rot] = z.real, z.imag
    return out


def _exact_attend(s, c):
    group, out = c["heads"] // c["kv_heads"], []
    for b, n in enumerate(s.lengths.tolist()):
        if n == 0:
            out.append(torch.zeros((c["heads"], c["dim"]), dtype=torch.float64, device="cuda"))
            continue
        at = torch.tensor(range(n), device="cuda")
        if c["window"] and n > c["window"]:
            at = torch.cat((at[:min(c["sinks"], n - c["window"])], at[n - c["window"]:]))
        where = s.table[b, at // c["page"]].long() * c["page"] + at % c["page"]
        k = s.k_pages.flatten(0, 1)[where].double().repeat_interleave(group, 1)
        v = s.v_pages.flatten(0, 1)[where].double().repeat_interleave(group, 1)
        w = torch.softmax((k * s.q[b].double()).sum(-1) * c["dim"] ** -0.5, 0)
        out.append((w[..., None] * v).sum(0))
    return torch.stack(out)


def _exact_sequences(s, c):
    b, tq, h, d = c["batch"], c["q_len"], c["heads"], c["dim"]
    group, first = h // c["kv_heads"], c["kv_len"] - c["q_len"]
    out, lse = s.out.double(), s.lse.double()
    if c["kind"] == "train":
        dq, dk, dv = s.dq.double(), s.dk.double(), s.dv.double()
    for i, n in enumerate(_sequence_lengths(c)):
        rows = n - first
        if rows <= 0:
            continue
        p = torch.arange(first, n, device="cuda")[:, None]
        t = torch.arange(n, device="cuda")[None]
        hidden = (t > p) | ((p - t >= c["window"]) & (t >= c["sinks"])) if c["window"] else t > p
        for x in range(h):
            q, k, v = s.q[i, :rows, x].double(), s.k[i, :n, x // group].double(), s.v[i, :n, x // group].double()
            score = (q @ k.T) * d ** -0.5
            score[hidden] = -math.inf
            lse[i, x, :rows] = torch.logsumexp(score, -1)
            w = torch.softmax(score, -1)
            out[i, :rows, x] = w @ v
            if c["kind"] == "train":
                g = s.dout[i, :rows, x].double()
                up = g @ v.T
                ds = w * (up - (g * out[i, :rows, x]).sum(-1, keepdim=True)) * d ** -0.5
                dv[i, :n, x // group] += w.T @ g
                dq[i, :rows, x] = ds @ k
                dk[i, :n, x // group] += ds.T @ q
    return (out, lse, dq, dk, dv) if c["kind"] == "train" else (out, lse)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    if kind == "rope":
        sign = -1 if c["backward"] else 1
        return _spin(s.q, s.positions, c, sign), _spin(s.k, s.positions, c, sign)
    if kind == "append":
        turn = {"rot": c["dim"], "base": 10000.0, "scaling": "plain", "original": 0, "interleaved": False}
        pages = s.table.tolist()
        where = torch.tensor([pages[b][p // c["page"]] * c["page"] + p % c["page"] for b, p in zip(s.seqs.tolist(), s.positions.tolist())], device="cuda")
        k, v = s.k_pages.double(), s.v_pages.double()
        k.view(-1, c["kv_heads"], c["dim"])[where] = _spin(s.k, s.positions, turn, 1)
        v.view(-1, c["kv_heads"], c["dim"])[where] = s.v.double()
        return _spin(s.q, s.positions, turn, 1), k, v
    if kind == "copy":
        k, v = s.k_pages.double(), s.v_pages.double()
        for a, b in zip(s.src, s.dst):
            k[b], v[b] = k[a], v[a]
        return k, v
    return _exact_attend(s, c) if kind == "attend" else _exact_sequences(s, c)
