"""The packed cache's bookkeeping and refusals, without a GPU: lengths and positions, what is refused and that a refusal changes nothing."""
import ctypes
import random
from ctypes import c_int32, c_int64

import numpy as np
import pytest
import torch

from infllm_b200 import _lib as L
from infllm_b200.attention import PackedCache, packed_cache


class Calls:
    """The library, of which calls that launch something are noted and not made."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        if "book" in name or name == "infllm_last_error":
            return getattr(L.lib, name)

        def call(*args):
            self.seen.append((name, args))
            return 0

        return call


@pytest.fixture
def cache(monkeypatch):
    def make(n_sequences=4, max_tokens=20):
        c = PackedCache.__new__(PackedCache)
        c.n_layers, c.n_kv_heads, c.head_dim, c.n_sequences, c.max_tokens = 2, 2, 64, n_sequences, max_tokens
        c.dtype, c.device, c._ref = torch.bfloat16, torch.device("cpu"), None
        c._begin()
        c.calls = Calls()
        monkeypatch.setattr(packed_cache, "_lib_call", c.calls)
        monkeypatch.setattr(L, "raw_stream", lambda device: 0)
        return c

    return make


def test_a_cpu_device_is_refused():
    with pytest.raises(ValueError, match="CUDA"):
        PackedCache(1, 1, 64, 1, 16, device="cpu")


def state(c):
    return list(c._state)


def fresh(c, s):  # newest tokens that are known to lie in a row
    return c._state[5 * s + 3]


def test_lowest_numbers_and_capacity(cache):
    c = cache()
    assert c.open(3) == [0, 1, 2]
    c.free([1])
    assert c.open() == [1] and c.open() == [3]
    before = state(c)
    with pytest.raises(L.InfLLMCapacityError):
        c.open()
    b = c.batch([0, 1])
    b.extend([20, 3])
    before = state(c)
    with pytest.raises(L.InfLLMCapacityError):
        b.extend([0, 18])
    with pytest.raises(L.InfLLMCapacityError):
        b.extend(1)
    for n in (1 << 40, [0, 1 << 62]):
        with pytest.raises(L.InfLLMCapacityError):
            b.extend(n)
    for n in (1 << 63, [0, 1 << 64]):
        with pytest.raises(OverflowError):
            b.extend(n)
    assert state(c) == before


@pytest.mark.parametrize("call", [
    lambda c, b: c.batch([0, 0]), lambda c, b: c.batch([3]), lambda c, b: c.batch([-1]), lambda c, b: c.batch([9]), lambda c, b: c.free([0, 0]),
    lambda c, b: c.length(3), lambda c, b: c.position(-2), lambda c, b: c.open(-1), lambda c, b: b.extend(-1), lambda c, b: b.extend([1]),
    lambda c, b: b.extend([1, -1]), lambda c, b: b.plan([11, 1]), lambda c, b: b.retract(7), lambda c, b: c.evict([0, 0], 4), lambda c, b: c.evict([0], -1),
    lambda c, b: c.evict([0], 4, 3, 2), lambda c, b: c.evict([0], 4, -1), lambda c, b: c.evict([0], 4, 0, -1), lambda c, b: c.evict([0, 1], 4, into=[1, 2]),
    lambda c, b: c.evict([0, 1], 4, into=[2]), lambda c, b: c.evict([0], 4, into=[3]), lambda c, b: c.evict([0], 4, into=[0])])
def test_refusals_change_nothing(cache, call):
    c = cache()
    b = c.batch(c.open(3)[:2])
    b.extend([10, 6])
    before = state(c)
    with pytest.raises(ValueError):
        call(c, b)
    assert state(c) == before and not [n for n, _ in c.calls.seen if "evict" in n]


def test_numbers_that_do_not_fit_are_refused_not_cut(cache):
    c = cache()
    b = c.batch(c.open())
    b.extend(5)
    before = state(c)
    for args in ((1 << 64,), (1 << 63,), (5, 1 << 64), (5, 0, -(1 << 64))):
        with pytest.raises(OverflowError):
            c.evict([0], *args)
    for seqs in ([1 << 32], [-1 << 40]):
        with pytest.raises((OverflowError, ValueError)):
            c.evict(seqs, 3)
        with pytest.raises(ValueError):
            c.batch(seqs)
    with pytest.raises(ValueError):
        b.values(1 << 32)
    assert state(c) == before


def test_positions_go_on_behind_an_eviction(cache):
    c = cache()
    s, t = c.open(2)
    b = c.batch([s])
    b.extend(18)
    c.evict([s], 8, sink=1, recent=3)
    assert (c.length(s), c.position(s)) == (8, 18)
    assert [n for n, _ in c.calls.seen] == ["infllm_packed_evict"]
    with pytest.raises(ValueError, match="changed"):
        b.values(0)
    with pytest.raises(ValueError):
        b.retract(4)  # the newest three are the only ones that are known to lie in a row
    b.retract(2)
    assert (c.length(s), c.position(s)) == (6, 16)
    b.extend(5)
    assert list(b._table)[:4] == [s, 11, 5, 16] and b._info[1] == 21
    b.plan(11)
    with pytest.raises(ValueError, match="eviction"):
        b.write(0, None, None)
    c.evict([s], 30)  # nothing to do
    assert (c.length(s), c.position(s)) == (11, 21)
    c.evict([s], 4, recent=4, into=[t])
    assert (c.length(s), c.length(t), c.position(t), fresh(c, t)) == (11, 4, 21, 4)
    c.evict([s], 40, into=[t])
    assert (c.length(t), c.position(t)) == (11, 21)


def test_a_step_is_its_batchs(cache):
    c = cache()
    seqs = c.open(2)
    a, b = c.batch(seqs), c.batch(seqs[:1])
    with pytest.raises(ValueError, match="no step"):
        a.values()
    a.extend(2)
    b.extend(1)
    with pytest.raises(ValueError, match="changed"):
        a.values()
    a.plan(0)
    a.plan([3, 2])
    a.retract(1)
    with pytest.raises(ValueError, match="no step"):
        a.values()
    c.free(seqs)
    c.open(2)
    for call in (a.extend, a.plan, a.retract):
        with pytest.raises(ValueError, match="freed"):
            call(0)


def test_random_books_agree_with_a_restatement(cache):
    rng = random.Random(3)
    c = cache(6, 50)
    held = {}  # sequence: its tokens' positions
    for _ in range(3000):
        what = rng.choice(["open", "extend", "extend", "retract", "evict", "free"])
        if what == "open" and len(held) < 6:
            s = c.open()[0]
            assert s == min(set(range(6)) - set(held))
            held[s] = ([], 0, 0)
        elif held:
            s = rng.choice(sorted(held))
            rows, pos, new = held[s]
            n = rng.randint(0, 12)
            if what == "extend" and len(rows) + n <= 50:
                c.batch([s]).extend(n)
                held[s] = (rows + list(range(pos, pos + n)), pos + n, new + n)
            elif what == "retract" and n <= new:
                c.batch([s]).retract(n)
                held[s] = (rows[:len(rows) - n], pos - n, new - n)
            elif what == "evict":
                recent = rng.randint(0, 10)
                budget = recent + rng.randint(0, 20)
                c.evict([s], budget, recent=recent)
                if len(rows) > budget:
                    held[s] = (rows[:budget - recent] + rows[len(rows) - recent:], pos, min(new, recent))
            elif what == "free":
                c.free([s])
                del held[s]
        for s, (rows, pos, new) in held.items():
            assert (c.length(s), c.position(s), fresh(c, s)) == (len(rows), pos, new)
            assert not new or rows[-new:] == list(range(pos - new, pos))


# ------------------------------------------------------------------------------------------------- the C entry points
AT = 1 << 20  # an address that nothing is launched with


def packed(**more):
    a = dict(n_layers=2, n_kv_heads=2, head_dim=64, n_sequences=4, max_tokens=100, dtype=L.BF16, device=-1, pad=0, d_codes=AT, d_scales=AT,
             d_weights=AT, d_places=AT)
    a.update(more)
    return L.Packed(**a)


def rows(*r):
    return (c_int32 * (4 * len(r)))(*[x for row in r for x in row])


GOOD = (1, 10, 3, 7)


def write(c=None, layer=0, seqs=(GOOD,), most=3, k=AT, ks=(64, 64, 64), q=AT, q_out=AT, heads=4, cos=None, sin=None, table=0):
    c = packed() if c is None else c
    return L.lib.infllm_packed_write(ctypes.byref(c), layer, rows(*seqs), len(seqs), most, k, *ks, AT, 64, 64, 64, q, 64, 64, 64, q_out, heads, cos,
                                     sin, table, None)


def attend(c=None, layer=0, seqs=(GOOD,), most=3, q=AT, qs=(64, 64, 64), out=AT, heads=4, scale=0.1, weigh=0, decay=1.0, work=AT, size=1 << 40):
    c = packed() if c is None else c
    return L.lib.infllm_packed_attend(ctypes.byref(c), layer, rows(*seqs), len(seqs), most, q, *qs, out, None, heads, scale, weigh, decay, work, size,
                                      None)


def values(c=None, layer=0, n_layers=1, seqs=(GOOD,), most=3, k=AT):
    c = packed() if c is None else c
    return L.lib.infllm_packed_values(ctypes.byref(c), layer, n_layers, rows(*seqs), len(seqs), most, k, AT, None)


def evict(c=None, seqs=(GOOD,), into=None, budget=5, sink=1, recent=2, work=AT, size=1 << 40):
    c = packed() if c is None else c
    return L.lib.infllm_packed_evict(ctypes.byref(c), rows(*seqs), len(seqs), None if into is None else (c_int32 * len(into))(*into), budget, sink,
                                     recent, work, size, None)


def room(c=None, seqs=(GOOD,), most=3, heads=4, weigh=0):
    c, n = packed() if c is None else c, c_int64(-1)
    return L.lib.infllm_packed_room(ctypes.byref(c), rows(*seqs), len(seqs), most, heads, weigh, ctypes.byref(n))


BAD_CACHES = [dict(n_layers=0), dict(n_kv_heads=0), dict(head_dim=96), dict(n_sequences=0), dict(max_tokens=0), dict(max_tokens=1 << 29), dict(dtype=7),
              dict(d_codes=0), dict(d_scales=AT + 8), dict(d_weights=AT + 4), dict(d_places=0), dict(n_layers=20000), dict(n_kv_heads=9000)]
BAD_SEQS = [((4, 10, 3, 7),), ((-1, 10, 3, 7),), ((1, 101, 3, 7),), ((1, 10, 4, 7),), ((1, 2, 3, 7),), ((1, 10, -1, 7),), ((1, -1, 0, 7),),
            ((1, 10, 3, -1),), ((1, 10, 3, 0x7fffffff),), (GOOD, (1, 5, 1, 4))]


@pytest.mark.parametrize("call", [write, attend, values, room, evict])
@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_that_are_none(call, bad):
    assert call(packed(**bad)) in (L.E_BADARG, L.E_UNSUPPORTED)
    assert L.lib.infllm_last_error()


@pytest.mark.parametrize("call", [write, attend, values, room])
@pytest.mark.parametrize("seqs", BAD_SEQS)
def test_sequences_that_are_none(call, seqs):
    assert call(seqs=seqs) == L.E_BADARG


@pytest.mark.parametrize("rc", [
    lambda: write(layer=2), lambda: write(layer=-1), lambda: write(most=101), lambda: write(most=-1), lambda: write(k=None), lambda: write(k=AT + 2),
    lambda: write(ks=(64, 60, 64)), lambda: write(q_out=None), lambda: write(heads=0), lambda: write(cos=AT), lambda: write(cos=AT, sin=AT, table=9),
    lambda: attend(layer=2), lambda: attend(q=None), lambda: attend(q=AT + 8), lambda: attend(qs=(4, 64, 64)), lambda: attend(out=None),
    lambda: attend(heads=3), lambda: attend(heads=0), lambda: attend(scale=-1.0), lambda: attend(scale=float("nan")), lambda: attend(scale=float("inf")),
    lambda: attend(weigh=-1), lambda: attend(weigh=1, decay=-1.0), lambda: attend(weigh=1, decay=float("nan")), lambda: attend(work=None),
    lambda: attend(work=AT + 4), lambda: attend(size=16), lambda: values(layer=1, n_layers=2), lambda: values(n_layers=0), lambda: values(k=None),
    lambda: values(k=AT + 4), lambda: evict(budget=-1), lambda: evict(sink=-1), lambda: evict(recent=-1), lambda: evict(sink=4), lambda: evict(work=None),
    lambda: evict(work=AT + 4), lambda: evict(size=2 * 2 * 4 * 8 - 1), lambda: evict(into=[1]), lambda: evict(into=[4]), lambda: evict(seqs=(GOOD, (2, 3, 0, 0)), into=[0, 0]),
    lambda: evict(seqs=(GOOD, GOOD)), lambda: room(heads=5), lambda: room(weigh=-1)])
def test_arguments_that_are_none(rc):
    assert rc() == L.E_BADARG


def test_calls_without_work():
    for call in (write, attend, values, evict):
        assert call(seqs=()) == L.OK
    assert write(seqs=((1, 10, 0, 7),), most=0) == attend(seqs=((1, 10, 0, 7),), most=0) == values(seqs=((1, 10, 0, 7),), most=0) == L.OK
    assert evict(budget=10) == evict(seqs=((1, 0, 0, 0),), budget=0, sink=0, recent=0, into=[2]) == L.OK


@pytest.mark.parametrize("number", [np.int64, np.int32, torch.tensor, np.array])
def test_numbers_of_other_kinds(cache, number):
    """A count that numpy or torch made is one for every sequence, an array of them one for each."""
    c = cache()
    b = c.batch(c.open(2))
    b.extend(number(5))
    assert [c.length(0), c.length(1)] == [5, 5] and b.tokens == 5
    b.extend(np.array([3, 1]))
    b.plan(torch.tensor([2, 1]))
    assert [c.length(0), c.length(1)] == [8, 6] and b.tokens == 2
    b.retract(number(1))
    c.evict([0], number(4), number(1))
    assert [c.length(0), c.length(1)] == [4, 5]
    for n in (1.0, np.float64(1), torch.tensor(1.0), None):
        with pytest.raises(TypeError):
            b.extend(n)
    one = c.batch([1])
    one.extend(torch.tensor([2]))
    with pytest.raises(ValueError):
        b.extend(torch.tensor([2]))
    assert [c.length(0), c.length(1)] == [4, 7]
