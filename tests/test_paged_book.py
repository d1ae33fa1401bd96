"""The paged cache's bookkeeping, without a GPU, against a restatement of its rules: pages and numbers lowest first, shared
full pages, what is refused and that a refusal changes nothing."""
import ctypes
import random
from ctypes import c_int, c_int32, c_int64

import pytest

from infllm_b200 import _lib as L


class Cache:
    def __init__(self, n_pages=40, page=16, max_sequences=12, max_pages=10):
        cfg = L.PagesConfig(1, 2, 64, page, n_pages, max_sequences, max_pages, L.BF16, -1, 0, None, None)
        self.h = ctypes.c_void_p()
        L.check(L.lib.infllm_pages_create(ctypes.byref(cfg), ctypes.byref(self.h)))

    def __del__(self):
        L.lib.infllm_pages_destroy(self.h)

    def ids(self, x):
        return (c_int32 * len(x))(*x)

    def open(self, n=1):
        out = (c_int32 * n)()
        L.check(L.lib.infllm_pages_open(self.h, n, out))
        return list(out)

    def fork(self, seqs, n):
        out = (c_int32 * (len(seqs) * n))()
        L.check(L.lib.infllm_pages_fork(self.h, self.ids(seqs), len(seqs), n, out, None))
        return list(out)

    def copy(self, seqs, into):
        out = (c_int32 * len(seqs))()
        L.check(L.lib.infllm_pages_copy(self.h, self.ids(seqs), len(seqs), into.h, out, None))
        return list(out)

    def extend(self, seqs, counts):
        b = ctypes.c_void_p()
        L.check(L.lib.infllm_page_batch_create(self.h, self.ids(seqs), len(seqs), ctypes.byref(b)))
        try:
            L.check(L.lib.infllm_page_batch_extend(b, self.ids(counts), 0, None, None))
        finally:
            L.lib.infllm_page_batch_destroy(b)

    def truncate(self, seqs, lengths):
        L.check(L.lib.infllm_pages_truncate(self.h, self.ids(seqs), (c_int64 * len(lengths))(*lengths), len(seqs)))

    def free(self, seqs):
        L.check(L.lib.infllm_pages_free(self.h, self.ids(seqs), len(seqs)))

    def compact(self, seqs, keep):
        flat = [x for spans in keep for s in spans for x in s]
        L.check(L.lib.infllm_pages_compact(self.h, self.ids(seqs), len(seqs), (c_int64 * len(flat))(*flat),
                                           self.ids([len(k) for k in keep]), None))

    def row(self, s):
        n, out = c_int(), (c_int32 * 64)()
        L.check(L.lib.infllm_pages_row(self.h, s, out, 64, ctypes.byref(n)))
        return list(out[:n.value])

    def info(self, s):
        a, b = c_int64(), c_int64()
        L.check(L.lib.infllm_pages_info(self.h, s, ctypes.byref(a), ctypes.byref(b)))
        return a.value, b.value

    @property
    def n_free(self):
        return L.lib.infllm_pages_free_count(self.h)


class Model:
    """The rules, as plainly as they can be said; a page also knows which tokens are in it, so that moves can be followed."""

    def __init__(self, n_pages=40, page=16, max_sequences=12, max_pages=10):
        self.page, self.n_pages, self.max_pages, self.max_sequences = page, n_pages, max_pages, max_sequences
        self.uses = [0] * n_pages
        self.seqs = {}  # number -> [pages, length, position]

    def free_pages(self):
        return [i for i in range(self.n_pages) if not self.uses[i]]

    def take(self):
        p = self.free_pages()[0]
        self.uses[p] = 1
        return p

    def numbers(self, n):
        got = [i for i in range(self.max_sequences) if i not in self.seqs][:n]
        return got if len(got) == n else None

    def pages_of(self, n):
        return -(-n // self.page)

    def open(self, n=1):
        got = self.numbers(n)
        if got is None:
            return None
        for g in got:
            self.seqs[g] = [[], 0, 0]
        return got

    def extend(self, seqs, counts):
        need = 0
        for s, c in zip(seqs, counts):
            pages, length, _ = self.seqs[s]
            if length + c > self.max_pages * self.page:
                return None
            need += self.pages_of(length + c) - len(pages)
            need += bool(c and length % self.page and self.uses[pages[-1]] > 1)
        if need > len(self.free_pages()):
            return None
        for s, c in zip(seqs, counts):
            q = self.seqs[s]
            if c and q[1] % self.page and self.uses[q[0][-1]] > 1:
                old, q[0][-1] = q[0][-1], self.take()
                self.uses[old] -= 1
            q[1] += c
            q[2] += c
            while len(q[0]) < self.pages_of(q[1]):
                q[0].append(self.take())
        return True

    def fork(self, seqs, n):
        got = self.numbers(len(seqs) * n)
        if got is None or sum(n * bool(self.seqs[s][1] % self.page) for s in seqs) > len(self.free_pages()):
            return None
        at = iter(got)
        for s in seqs:
            pages, length, position = self.seqs[s]
            full = pages[:length // self.page]
            for _ in range(n):
                for p in full:
                    self.uses[p] += 1
                self.seqs[next(at)] = [full + ([self.take()] if length % self.page else []), length, position]
        return got

    def cut(self, s, length):
        q = self.seqs[s]
        q[2] -= q[1] - length
        q[1] = length
        while len(q[0]) > self.pages_of(length):
            self.uses[q[0].pop()] -= 1

    def compact(self, seqs, keep):
        plans, need = [], 0
        for s, spans in zip(seqs, keep):
            place = [i for a, b in spans for i in range(a, b)]
            stay = 0
            while (stay + 1) * self.page <= len(place) and place[(stay + 1) * self.page - 1] == (stay + 1) * self.page - 1:
                stay += 1
            need += self.pages_of(len(place)) - stay
            plans.append((len(place), stay))
        if need > len(self.free_pages()):
            return None
        gone = []
        for s, (n, stay) in zip(seqs, plans):
            q = self.seqs[s]
            gone += q[0][stay:]
            q[0] = q[0][:stay] + [self.take() for _ in range(self.pages_of(n) - stay)]
            q[1] = n
        for g in gone:
            self.uses[g] -= 1
        return True


def same(c, m):
    assert c.n_free == len(m.free_pages())
    for s, (pages, length, position) in m.seqs.items():
        assert c.row(s) == pages and c.info(s) == (length, position), s


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page,n_pages", [(16, 40), (32, 9)])
def test_random_steps_follow_the_rules(seed, page, n_pages):
    r = random.Random(seed)
    c, m = Cache(n_pages, page), Model(n_pages, page)
    refused = done = 0
    for _ in range(400):
        live = sorted(m.seqs)
        what = r.choice(["open", "extend", "extend", "fork", "cut", "free", "compact"])
        some = r.sample(live, r.randint(1, min(3, len(live)))) if live else []
        if what != "open" and not live:
            continue
        if what == "open":
            want, call = m.open(2), lambda: c.open(2)
        elif what == "extend":
            counts = [r.choice([0, 1, 3, page, 2 * page + 1]) for _ in some]
            want, call = m.extend(some, counts), lambda: c.extend(some, counts)
        elif what == "fork":
            n = r.randint(0, 3)
            want, call = m.fork(some, n), lambda: c.fork(some, n)
        elif what == "cut":
            lengths = [r.randint(0, m.seqs[s][1]) for s in some]
            for s, n in zip(some, lengths):
                m.cut(s, n)
            want, call = True, lambda: c.truncate(some, lengths)
        elif what == "free":
            for s in some:
                m.cut(s, 0)
                del m.seqs[s]
            want, call = True, lambda: c.free(some)
        else:
            keep = []
            for s in some:
                cuts = sorted(r.sample(range(m.seqs[s][1] + 1), min(m.seqs[s][1] + 1, 2 * r.randint(0, 3)) // 2 * 2))
                keep.append(list(zip(cuts[::2], cuts[1::2])))
            want, call = m.compact(some, keep), lambda: c.compact(some, keep)
        if want is None:
            with pytest.raises(L.InfLLMCapacityError):
                call()
            refused += 1
        else:
            got = call()
            assert got is None or got == want
            done += 1
        same(c, m)
    assert done > 100 and refused > 5


def test_copies_share_nothing():
    a, b = Cache(), Cache(n_pages=7)
    s = a.open()[0]
    a.extend([s], [35])
    k = a.fork([s], 1)[0]
    t = a.copy([k, s], a)
    assert len(set(a.row(t[0]) + a.row(t[1])) & set(a.row(s) + a.row(k))) == 0 and not set(a.row(t[0])) & set(a.row(t[1]))
    assert [a.info(x) for x in t] == [(35, 35)] * 2
    u = b.copy([], b) + a.copy([s, k], b)
    assert b.row(u[0]) == [0, 1, 2] and b.row(u[1]) == [3, 4, 5] and b.n_free == 1
    with pytest.raises(L.InfLLMCapacityError):
        a.copy([s], b)
    assert b.n_free == 1 and b.info(u[0]) == (35, 35)


def test_refusals():
    c = Cache()
    s = c.open()[0]
    c.extend([s], [20])
    for call in (lambda: c.free([5]), lambda: c.free([s, s]), lambda: c.free([-1]), lambda: c.fork([3], 1), lambda: c.truncate([s], [21]),
                 lambda: c.truncate([s], [-1]), lambda: c.extend([s], [-1]), lambda: c.compact([s], [[(0, 21)]]),
                 lambda: c.compact([s], [[(5, 7), (6, 9)]]), lambda: c.compact([s], [[(5, 4)]]), lambda: c.row(99)):
        with pytest.raises(L.InfLLMError) as e:
            call()
        assert e.value.code == L.E_BADARG
        assert c.info(s) == (20, 20) and c.n_free == 38
    b = ctypes.c_void_p()
    L.check(L.lib.infllm_page_batch_create(c.h, c.ids([s]), 1, ctypes.byref(b)))
    c.free([s])
    assert c.open() == [s]  # the same number, another sequence
    assert L.lib.infllm_page_batch_extend(b, None, 1, None, None) == L.E_BADARG and b"freed" in L.lib.infllm_last_error()
    L.lib.infllm_page_batch_destroy(b)
    out = ctypes.c_void_p()
    for change in (dict(head_dim=96), dict(page_size=48), dict(dtype=2), dict(n_pages=0), dict(max_pages=1 << 30)):
        cfg = L.PagesConfig(n_layers=1, n_kv_heads=2, head_dim=64, page_size=16, n_pages=4, max_sequences=4, max_pages=4, dtype=0, device=-1)
        for k, v in change.items():
            setattr(cfg, k, v)
        assert L.lib.infllm_pages_create(ctypes.byref(cfg), ctypes.byref(out)) in (L.E_BADARG, L.E_UNSUPPORTED)
    assert L.lib.infllm_pages_create(None, None) == L.E_BADARG


@pytest.mark.parametrize("seed", range(12))
def test_plan_of_a_batch_that_has_lived(seed):
    """What a batch keeps of its sequences' order is made anew where what they share has changed: its plan has the size of a new batch's."""
    r = random.Random(seed)
    c = Cache(n_pages=4000, max_sequences=100, max_pages=300)

    def batch(seqs):
        b = ctypes.c_void_p()
        L.check(L.lib.infllm_page_batch_create(c.h, c.ids(seqs), len(seqs), ctypes.byref(b)))
        return b

    def plan(b, new):
        if L.lib.infllm_page_batch_select(b, None, new, None) != 0:  # (one of them has fewer)
            L.check(L.lib.infllm_page_batch_select(b, None, 0, None))
        size = c_int64()
        L.check(L.lib.infllm_page_batch_plan(b, 8, ctypes.byref(size)))
        return size.value

    seqs = c.open(r.randint(1, 2))
    for _ in range(3):
        b = batch(seqs)
        L.check(L.lib.infllm_page_batch_extend(b, None, r.choice([5, 16, 100, 800]), None, None))
        L.lib.infllm_page_batch_destroy(b)
        seqs += c.fork([r.choice(seqs)], r.randint(1, 10))
    b = batch(seqs)
    for _ in range(20):
        what = r.randrange(4)
        if what == 0:
            L.check(L.lib.infllm_page_batch_extend(b, c.ids([r.choice([0, 1, 3, 16, 40]) for _ in seqs]), 0, None, None))
        elif what == 1:
            n = r.choice([1, 16, 33])
            L.check(L.lib.infllm_page_batch_extend(b, None, n, None, None))
            plan(b, 1)
            L.check(L.lib.infllm_page_batch_select(b, None, n, None))
            L.check(L.lib.infllm_page_batch_retract(b, None, r.randint(0, n)))
        elif what == 2:
            for q in r.sample(seqs, r.randint(1, len(seqs))):
                L.lib.infllm_pages_truncate(c.h, c.ids([q]), (c_int64 * 1)(r.choice([0, 16, 17, 100, 160, 800])), 1)  # (or refused)
        else:
            L.check(L.lib.infllm_pages_free(c.h, c.ids(c.fork([r.choice(seqs)], 1)), 1))
        new = r.choice([1, 4])
        fresh = batch(seqs)
        assert plan(b, new) == plan(fresh, new)
        L.lib.infllm_page_batch_destroy(fresh)
    L.lib.infllm_page_batch_destroy(b)


@pytest.mark.parametrize("what", ["truncate", "truncate a little", "compact", "retract of another batch", "extend of another batch", "free pages"])
def test_write_is_refused_where_the_step_is_another(what):
    """A step's counts are of the sequences as they were when it began.  A sequence that was cut since would be written in front of its
    pages, one that was cut by less, or has grown, where other tokens are."""
    c = Cache()
    s, t = c.open(2)
    b, other = ctypes.c_void_p(), ctypes.c_void_p()
    L.check(L.lib.infllm_page_batch_create(c.h, c.ids([s, t]), 2, ctypes.byref(b)))
    L.check(L.lib.infllm_page_batch_create(c.h, c.ids([t]), 1, ctypes.byref(other)))

    def write():
        rc = L.lib.infllm_page_batch_write(b, 0, None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, None, 0, None, None, 0, None)
        assert rc == L.E_BADARG  # (at the latest because there is no device)
        return L.lib.infllm_last_error().decode()

    L.check(L.lib.infllm_page_batch_extend(b, c.ids([3, 40]), 0, None, None))
    assert "without a device" in write()
    if what == "truncate":
        c.truncate([t], [2])
    elif what == "truncate a little":
        c.truncate([t], [39])
    elif what == "compact":
        c.compact([t], [[(0, 1), (7, 9)]])
    elif what == "retract of another batch":
        L.check(L.lib.infllm_page_batch_select(other, None, 0, None))
        L.check(L.lib.infllm_page_batch_retract(other, None, 40))
    elif what == "extend of another batch":
        L.check(L.lib.infllm_page_batch_extend(other, None, 1, None, None))
    else:  # (what changes no token of theirs is no reason to refuse)
        c.truncate([s, t], [3, 40])
        c.compact([t], [[(0, 40)]])
        L.check(L.lib.infllm_page_batch_extend(other, None, 0, None, None))
        c.free(c.fork([s], 2))
    got = write()
    if what == "free pages":
        assert "without a device" in got
    else:
        assert f"sequence {t}" in got and "step" in got
        # a step that is about fewer sequences, or a new one, is not refused for it
        L.check(L.lib.infllm_page_batch_select(b, c.ids([3, 0]), 0, None))
        L.check(L.lib.infllm_page_batch_extend(other, None, 1, None, None))
        assert "without a device" in write()
        L.check(L.lib.infllm_page_batch_extend(b, None, 2, None, None))
        assert "without a device" in write()
    for x in (b, other):
        L.lib.infllm_page_batch_destroy(x)


def test_a_plan_that_found_no_memory_is_not_used_with_the_last_ones(monkeypatch):
    """Where the workspace of a new plan cannot be had, the call fails, and the next one asks for it again: it is never made in the
    last plan's memory, which may be too small.  (The library is stood in for by the rules of its attend and plan calls.)"""
    import types

    import torch

    from infllm_b200.attention import paged_cache as M

    class Library:
        planned, need, seen = False, 1 << 12, []

        def infllm_page_batch_create(self, *a):
            return 0

        infllm_page_batch_destroy = infllm_page_batch_extend = infllm_page_batch_create

        def infllm_page_batch_plan(self, handle, heads, size):
            size._obj.value, self.planned = self.need, True
            return 0

        def infllm_page_batch_attend(self, handle, layer, q, bs, hs, ts, out, lse, heads, scale, work, stream):
            if not self.planned:
                return L.PAGES_NO_PLAN
            self.seen.append(work)
            return 0 if work else L.E_BADARG

    lib = Library()
    monkeypatch.setattr(M, "_lib_call", lib)
    monkeypatch.setattr(M._lib, "raw_stream", lambda device: 0)
    cache = types.SimpleNamespace(handle=None, head_dim=64, dtype=torch.bfloat16, device=torch.device("cpu"), n_kv_heads=1)
    empty, sizes, short = torch.empty, {}, [False]

    def take(size, *a, **k):
        if k.get("dtype") is not torch.uint8:
            return empty(size, *a, **k)
        if short[0]:
            raise torch.cuda.OutOfMemoryError("no memory")
        t = empty(size, *a, **k)
        sizes[t.data_ptr()] = t.numel()
        return t

    monkeypatch.setattr(torch, "empty", take)
    q = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16)
    for before in (False, True):  # the batch's first plan, or a later one
        b = M.PagedBatch(cache, [0])
        b.extend(1)
        lib.planned, lib.need = False, 1 << 12
        if before:
            b.attend(0, q)
        lib.planned, lib.need, short[0] = False, 1 << 16, True
        with pytest.raises(torch.cuda.OutOfMemoryError):
            b.attend(0, q)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            b.attend(0, q)
        short[0] = False
        lib.seen.clear()
        b.attend(0, q)
        b.attend(1, q)
        assert len(lib.seen) == 2 and all(sizes[w] >= 1 << 16 for w in lib.seen)


def test_numbers_beyond_the_library_s_are_refused(monkeypatch):
    """Not cut to 32 or 64 bits, where they would name another sequence or count."""
    import torch

    from infllm_b200.attention import paged_cache as M

    monkeypatch.setattr(M._lib, "raw_stream", lambda device: None)
    book = Cache()
    c = M.PagedCache.__new__(M.PagedCache)
    c.handle, c.device, c.head_dim, c.table = book.h, None, 64, torch.zeros((12, 10))
    s = c.open()[0]
    b = c.batch([s])
    b.extend(20)
    far = s + (1 << 32)
    try:
        for call in (lambda: c.free([far]), lambda: c.fork([far], 1), lambda: c.copy([far]), lambda: c.truncate([far], [3]), lambda: c.truncate([s], [1 << 64]),
                     lambda: c.compact([far], [[]]), lambda: c.compact([s], [[(0, (1 << 64) + 4)]]), lambda: c.batch([far]), lambda: c.length(far),
                     lambda: c.position(far), lambda: c.page_ids(far), lambda: b.extend((1 << 32) + 1), lambda: b.extend([(1 << 32) + 1]),
                     lambda: b.plan(1 << 32), lambda: b.retract((1 << 32) + 1), lambda: b.retract([(1 << 32) + 1])):
            with pytest.raises(OverflowError):
                call()
            assert c.length(s) == 20 and b.tokens == 20 and c.free_pages == 38 and c.open() == [s + 1]
            c.free([s + 1])
    finally:
        c.handle = None  # (the book's)
