"""The bookkeeping of a paged cache (aig_page_pool_*): no device involved.  A plain model beside it holds each sequence's
tokens, and what a cache would hold after the copies that the pool asks for."""
import ctypes
import random

import pytest

import __graft_entry__ as entry

NO_PAGES, INVALID = -6, -1


@pytest.fixture(scope="module")
def pkg():
    return entry.build()


class Model:
    """A pool and a cache of numbers kept by its tables and copies."""

    def __init__(self, pkg, pages, size):
        self.pool, self.size, self.width = pkg.PagePool(pages, size), size, pages
        self.cache = [[None] * size for _ in range(pages)]
        self.tokens, self.gone = {}, {}
        self.next = 0

    def copy(self, pairs):
        held = [list(self.cache[a]) for a, _ in pairs]
        for x, (_, b) in zip(held, pairs):
            self.cache[b] = x

    def open(self):
        s = self.pool.open()
        assert s not in self.tokens
        self.tokens[s], self.gone[s] = [], set()
        return s

    def grow(self, s, n):
        pair = self.pool.grow(s, n)
        if pair:
            self.copy([pair])
        t, begin = self.pool.table(s, self.width), len(self.tokens[s])
        for i in range(begin, begin + n):
            self.tokens[s].append(self.next)
            self.cache[t[i // self.size]][i % self.size] = self.next
            self.next += 1

    def fork(self, s):
        n = self.pool.fork(s)
        self.tokens[n], self.gone[n] = list(self.tokens[s]), set(self.gone[s])
        return n

    def trim(self, s, window, sinks):
        self.pool.trim(s, window, sinks)
        n = len(self.tokens[s])
        self.gone[s] |= {i for i in range(n) if sinks <= i < n - window}

    def close(self, s):
        self.pool.close_sequence(s)
        del self.tokens[s], self.gone[s]

    def check(self):
        used = {}
        for s, tokens in self.tokens.items():
            assert self.pool.length(s) == len(tokens)
            t = self.pool.table(s, self.width)
            need = -(-len(tokens) // self.size)
            assert all(p == -1 for p in t[need:])
            for p in t[:need]:
                if p >= 0:
                    used[p] = used.get(p, 0) + 1
            for i, x in enumerate(tokens):
                p = t[i // self.size]
                if i in self.gone[s]:
                    continue  # its page may be gone, or hold it still
                assert p >= 0 and self.cache[p][i % self.size] == x
        assert self.pool.free_pages == self.width - len(used)
        assert all(self.pool.shared(p) == used.get(p, 0) for p in range(self.width))


@pytest.mark.parametrize("pages,size,seed", [(1, 1, 0), (7, 1, 1), (12, 3, 2), (40, 16, 3), (64, 5, 4), (30, 2, 5)])
def test_random_histories(pkg, pages, size, seed):
    rng, m = random.Random(seed), Model(pkg, pages, size)
    refused = 0
    for _ in range(600):
        do = rng.choice(["open", "grow", "grow", "grow", "fork", "trim", "close", "compact"])
        s = rng.choice(list(m.tokens)) if m.tokens else None
        if do == "open" or s is None:
            if len(m.tokens) < 8:
                m.open()
        elif do == "grow":
            before = m.pool.free_pages, m.pool.table(s, pages)
            try:
                m.grow(s, rng.choice([0, 1, 1, 2, size, 2 * size + 1]))
            except pkg.AigError as e:
                assert e.code == NO_PAGES and before == (m.pool.free_pages, m.pool.table(s, pages))
                refused += 1
        elif do == "fork" and len(m.tokens) < 8:
            m.fork(s)
        elif do == "trim":
            m.trim(s, rng.choice([1, 2, size, 3 * size]), rng.choice([0, 1, size, size + 1]))
        elif do == "close" and rng.random() < 0.5:
            m.close(s)
        elif do == "compact":
            src, dst = m.pool.compact(rng.choice([0, 1, 3, pages]))
            assert not set(src) & set(dst) and len(set(dst)) == len(dst)
            m.copy(list(zip(src, dst)))
        m.check()
    assert refused or pages > 12  # the small pools run out
    m.pool.close()


def test_compaction_leaves_the_lowest_pages(pkg):
    m = Model(pkg, 10, 2)
    a, b = m.open(), m.open()
    for _ in range(5):
        m.grow(a, 2)
        m.grow(b, 2)
    m.close(a)
    src, dst = m.pool.compact(10)
    m.copy(list(zip(src, dst)))
    m.check()
    assert sorted(m.pool.table(b, 5)) == [0, 1, 2, 3, 4]
    assert m.pool.compact(10) == ([], [])
    m.pool.close()


def test_refusals(pkg):
    lib = pkg.lib()
    h, i = ctypes.c_void_p(), ctypes.c_int()
    for pages, size in ((0, 4), (4, 0), (-1, 4)):
        assert lib.aig_page_pool_create(pages, size, ctypes.byref(h)) == INVALID and not h
    assert lib.aig_page_pool_create(4, 4, None) == INVALID
    pool = pkg.PagePool(4, 4)
    a, b = ctypes.c_int(), ctypes.c_int()
    for seq in (-1, 0, 5):  # none is open yet
        assert lib.aig_page_pool_grow(pool.handle, seq, 1, ctypes.byref(a), ctypes.byref(b)) == INVALID
        assert lib.aig_page_pool_fork(pool.handle, seq, ctypes.byref(i)) == INVALID
        assert lib.aig_page_pool_trim(pool.handle, seq, 4, 0) == INVALID
        assert lib.aig_page_pool_close(pool.handle, seq) == INVALID
        assert lib.aig_page_pool_length(pool.handle, seq) == INVALID
        assert lib.aig_page_pool_table(pool.handle, seq, None, 0) == INVALID
    s = pool.open()
    assert lib.aig_page_pool_grow(pool.handle, s, -1, ctypes.byref(a), ctypes.byref(b)) == INVALID
    assert lib.aig_page_pool_grow(pool.handle, s, 2 ** 31 - 1, ctypes.byref(a), ctypes.byref(b)) == INVALID
    assert lib.aig_page_pool_grow(pool.handle, s, 17, ctypes.byref(a), ctypes.byref(b)) == NO_PAGES
    assert pool.length(s) == 0 and pool.free_pages == 4
    assert lib.aig_page_pool_grow(pool.handle, s, 1, None, ctypes.byref(b)) == INVALID
    assert lib.aig_page_pool_trim(pool.handle, s, 4, -1) == INVALID
    assert lib.aig_page_pool_compact(pool.handle, None, None, 1, ctypes.byref(i)) == INVALID
    assert lib.aig_page_pool_shared(pool.handle, 4) == INVALID
    for name in ("open", "length", "free_pages"):
        assert getattr(lib, "aig_page_pool_" + name)(*([None] + ([ctypes.byref(i)] if name == "open" else [0] if name == "length" else []))) == INVALID
    assert lib.aig_page_pool_destroy(None) == 0
    pool.close()


def test_rotary_frequencies(pkg):
    """The frequencies of every scaling against their definitions, computed on the host."""
    import math

    for rot, base, scaling, factor, length, low, high in [(64, 1e4, 0, 1.0, 0, 1.0, 32.0), (2, 5e5, 1, 4.0, 0, 1.0, 32.0), (96, 5e5, 2, 16.0, 8192, 1.0, 32.0),
                                                          (128, 1e4, 2, 2.0, 64, 1.0, 32.0), (64, 5e5, 3, 8.0, 8192, 1.0, 4.0)]:
        desc = pkg.RopeDesc(128, rot, 0, scaling, base, factor, length, low, high, 1.0)
        got = (ctypes.c_double * (rot // 2))()
        assert pkg.lib().aig_rope_frequencies(ctypes.byref(desc), ctypes.cast(got, ctypes.c_void_p), rot // 2) == 0
        for j in range(rot // 2):
            f = base ** (-2 * j / rot)
            if scaling == 1:
                f /= factor
            if scaling == 2:
                pair = lambda t: rot * math.log(length / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
                a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
                share = min(1, max(0, (j - a) / max(b - a, 0.001)))
                f = f * (1 - share) + f / factor * share
            if scaling == 3:
                share = 1 - min(1, max(0, (length * f / (2 * math.pi) - low) / (high - low)))
                f = f * (1 - share) + f / factor * share
            assert abs(got[j] - f) <= 1e-14 * f
    bad = [dict(head_dim=63), dict(rot_dim=130), dict(rot_dim=3), dict(rot_dim=0), dict(base=1.0), dict(base=float("inf")), dict(scaling=4), dict(scaling=1, factor=0.5),
           dict(scaling=2, original_len=0), dict(scaling=3, original_len=8, low=4.0, high=4.0), dict(magnitude=float("nan")), dict(head_dim=2048)]
    for change in bad:
        desc = pkg.RopeDesc(128, 128, 0, 0, 1e4, 1.0, 0, 1.0, 32.0, 1.0)
        for k, v in change.items():
            setattr(desc, k, v)
        got = (ctypes.c_double * 64)()
        assert pkg.lib().aig_rope_frequencies(ctypes.byref(desc), ctypes.cast(got, ctypes.c_void_p), 64) == INVALID, change


def test_calls_without_a_context_are_refused(pkg):
    lib = pkg.lib()
    assert lib.aig_rope_plan_create(None, None, None) == INVALID
    assert lib.aig_rope_forward(None, 0, None, 0, None, None, None, None) == INVALID
    assert lib.aig_rope_plan_destroy(None) == 0
    assert lib.aig_kv_append(None, None, None, None, None, None, None, None, None, 0, None, 0, 0) == INVALID
    assert lib.aig_kv_copy_pages(None, None, None, None, 0) == INVALID
    assert lib.aig_paged_attention(None, None, None, None, None, 0, None, 0, 0, 1.0, 0, 0) == INVALID
    assert lib.aig_window_attention_forward(None, None, None, None, None, None, None, None) == INVALID
    assert lib.aig_window_attention_backward(*[None] * 13) == INVALID
