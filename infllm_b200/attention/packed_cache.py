"""A key/value cache in 4 bits, attention over it, and eviction of what attention does not look at.

The reference keeps a long stream on the device by moving what it does not attend to to the host (inf_llm/attention/context_manager.py:
196-816) or by dropping all but a sink and a window (stream_llm.py:6-111).  This cache holds a token's keys and values in 80 bytes
instead of 256 (per KV head of 128 dimensions, each), and can drop tokens by the attention that they have had:

    cache = PackedCache(n_layers, n_kv_heads, head_dim, n_sequences, max_tokens)
    batch = cache.batch(cache.open(8))
    batch.extend(len_prompt)                               # once per step ...
    q = batch.write(layer, k, v, q, rope)                  # ... then in every layer
    o = batch.attend(layer, q, weigh=True)
    cache.evict(batch.seqs, budget=2048, sink=128, recent=512)

Of each 32 neighbouring numbers x of a key (rotated to its position) or value, in the cache's 16-bit type T, it holds m = min x, a step
s = T((max x - m) / 15) and of each number 4 bits, c, the nearest of 0 .. 15 to (x - m) / s.  They stand for T(m + s c).  (Where
T(m + 15 s) were infinite, s is the next smaller number.)  Where one of 32 numbers is not finite, or where the step is not, or in bf16 is 2^122 or more, none is a number: of
a value, these dimensions of the rows that see it are none, and nothing else is.

Tensors are (batch, heads, tokens, head_dim) views with any strides whose rows are 16-byte aligned, as the other attention types take
them.  Work goes to the current stream; all calls on a cache belong on one stream, or are ordered by the caller.  Inside a CUDA
graph's capture, write, attend, values and evict are launches like others: a replay does them again for the lengths of the
capture, while extend, retract and what evict does to lengths happen on the host, once.  A graph reads the cache's tensors and, of
a write with `rope`, the tables of positions that were there, which the cache keeps for it."""
import ctypes
import math
import operator
from array import array
from ctypes import c_int32, c_int64

import torch

from .. import _lib
from .rope import RotaryEmbeddingESM

_lib_call = _lib.lib
GROUP = 32  # numbers that share a least one and a step


class PackedCache:
    """Room for `n_sequences` sequences of up to `max_tokens` tokens.  head_dim is 64 or 128, dtype bfloat16 or float16.

    `codes` (n_layers, 2, n_sequences, n_kv_heads, max_tokens, head_dim / 8) int32 has the 4-bit codes, eight to a word (number 2i of the
    eight at bit 4i, number 2i + 1 at bit 16 + 4i); `scales` (.., head_dim / 32, 2) the least number and the step of each 32;
    `weights` (n_layers, n_sequences, n_kv_heads, max_tokens) fp32 what attend(weigh=..) has added up of each token, and `places` int32
    its position.  Sequences are named by their place in these, the lowest that is free.  What does not fit raises
    InfLLMCapacityError and changes nothing."""

    def __init__(self, n_layers, n_kv_heads, head_dim, n_sequences, max_tokens, dtype=torch.bfloat16, device=None):
        self.device = torch.device("cuda") if device is None else torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"a CUDA device is needed, got {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_layers, self.n_kv_heads, self.head_dim = int(n_layers), int(n_kv_heads), int(head_dim)
        self.n_sequences, self.max_tokens, self.dtype = int(n_sequences), int(max_tokens), dtype
        if min(self.n_layers, self.n_kv_heads, self.n_sequences, self.max_tokens) < 1:
            raise ValueError("sizes of a packed cache are positive")
        if self.head_dim not in (64, 128):
            raise ValueError(f"head_dim {self.head_dim} (64 and 128 are built)")
        code = _lib.dtype_code(dtype)
        rows = (self.n_sequences, self.n_kv_heads, self.max_tokens)
        self.codes = torch.zeros((self.n_layers, 2, *rows, self.head_dim // 8), dtype=torch.int32, device=self.device)
        self.scales = torch.zeros((self.n_layers, 2, *rows, self.head_dim // GROUP, 2), dtype=dtype, device=self.device)
        self.weights = torch.zeros((self.n_layers, *rows), dtype=torch.float32, device=self.device)
        self.places = torch.zeros((self.n_layers, *rows), dtype=torch.int32, device=self.device)
        self._c = _lib.Packed(self.n_layers, self.n_kv_heads, self.head_dim, self.n_sequences, self.max_tokens, code, self.device.index, 0,
                              self.codes.data_ptr(), self.scales.data_ptr(), self.weights.data_ptr(), self.places.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._captured = []  # rotary tables that captured writes read
        self._begin()

    def _begin(self):
        n = self.n_sequences
        self._state = (c_int64 * (5 * n))()  # of each sequence: opened, length, position, newest in a row, change
        self._book = _lib.PackedBook(n, self.max_tokens, 0, ctypes.addressof(self._state))
        self._book_ref = ctypes.byref(self._book)

    # -- sequences
    def _known(self, seqs):
        seqs = [int(s) for s in seqs]
        for s in seqs:
            if not 0 <= s < self.n_sequences or self._state[5 * s] % 2 == 0:
                raise ValueError(f"there is no sequence {s}")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence twice")
        return seqs

    def open(self, n=1):
        """n new, empty sequences: their numbers, the lowest that are not in use."""
        if n < 0:
            raise ValueError(f"{n} sequences")
        free = [s for s in range(self.n_sequences) if self._state[5 * s] % 2 == 0][:n]
        if len(free) < n:
            raise _lib.InfLLMCapacityError(_lib.E_CAPACITY, f"{n} sequences, where {len(free)} of {self.n_sequences} are free")
        for s in free:
            self._set(s)
        return free

    def _set(self, s):  # opened, or freed, and empty
        self._book.changes += 1
        self._state[5 * s:5 * s + 5] = self._state[5 * s] + 1, 0, 0, 0, self._book.changes

    def free(self, seqs):
        """Ends sequences."""
        for s in self._known(seqs):
            self._set(s)

    def length(self, seq):
        """Tokens that a sequence holds."""
        return self._state[5 * self._known([seq])[0] + 1]

    def position(self, seq):
        """The position that its next token is rotated to: the tokens that it has had (evict() takes none of them back)."""
        return self._state[5 * self._known([seq])[0] + 2]

    def batch(self, seqs):
        return PackedBatch(self, seqs)

    def check(self):
        """Waits for the device, and raises InfLLMError (E_TIMEOUT) where an attention kernel on it has given up a wait and left rows
        unwritten."""
        with torch.cuda.device(self.device):
            code, where = _lib.device_error()
        if code:
            raise _lib.InfLLMError(_lib.E_TIMEOUT, f"a bounded wait of an attention kernel ran out in a call before (code {code}, wait {where}): the "
                                   "rows that the block was to write are not valid")

    def evict(self, seqs, budget, sink=0, recent=0, into=None):
        """In every layer, each KV head of a sequence of more than `budget` tokens keeps that many, in their order: the first `sink`, the
        newest `recent`, and of the others those of the largest weights (of equal ones the earlier).  Which ones differs from head
        to head: `places` says it.  Keys keep the rotation that they were written with, and position() goes on from where it was.
        `into`: sequences of this cache that get what stays (all of a shorter sequence) in place of what they hold; `seqs` then
        stay as they are."""
        budget, sink, recent = (operator.index(x) for x in (budget, sink, recent))
        for x in (budget, sink, recent):
            if not -1 << 63 <= x < 1 << 63:
                raise OverflowError(f"{x} is beyond 64 bits")
        n, ids, to = len(seqs), _ids(seqs), None
        if into is not None:
            if len(into) != n:
                raise ValueError(f"{n} sequences into {len(into)}")
            to = _ids(into)
        table, most = (c_int32 * (4 * max(n, 1)))(), c_int64()
        _checked(_lib_call.infllm_packed_book_evict(self._book_ref, ids, n, to, budget, sink, recent, table, ctypes.byref(most), 0))
        size = self.n_layers * n * self.n_kv_heads * (-(-most.value // 4) * 4) * 4
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=self.device)
        _lib.check(_lib_call.infllm_packed_evict(self._ref, table, n, to, budget, sink, recent, work.data_ptr(), work.numel(),
                                                 _lib.raw_stream(self.device)))
        _lib.check(_lib_call.infllm_packed_book_evict(self._book_ref, ids, n, to, budget, sink, recent, None, None, 1))


def _checked(rc):
    """What there is not, and what does not fit, as Python's own errors."""
    if rc == _lib.E_BADARG:
        raise ValueError(_lib_call.infllm_last_error().decode("utf-8", "replace"))
    if rc:
        _lib.check(rc)


# (ctypes cuts what does not fit: array raises OverflowError)
def _ids(values):
    return (c_int32 * len(values)).from_buffer(array("i", values)) if len(values) else (c_int32 * 1)()


def _long(values):
    return (c_int64 * len(values)).from_buffer(array("q", values)) if len(values) else (c_int64 * 1)()


def _one(n):
    """Whether n, which is no int, is one number and not several: numpy's, a tensor's without dimensions."""
    try:
        len(n)
    except TypeError:
        return True
    return False


class PackedBatch:
    """Sequences that take a step together.  extend(), or plan(), says how many of each one's newest tokens the step is about;
    write() and attend() are then called in every layer.  Tensors have as many tokens as the largest of those counts; a
    sequence with fewer has its own at the end, and what is before them is not read, and zero in what is returned.  What the
    step is about is refused once one of its sequences was changed by another call."""

    def __init__(self, cache, seqs):
        self.cache, self.seqs = cache, cache._known(seqs)
        self._n = len(self.seqs)
        self._ids = _ids(self.seqs)
        self._opened = _long([cache._state[5 * s] for s in self.seqs])
        self.tokens = 0  # of the step's tensors
        self._table = (c_int32 * (4 * max(self._n, 1)))()  # of the step's sequences: slot, length, count, position
        self._as_of = (c_int64 * max(self._n, 1))()  # the last changes of the sequences when the step began,
        self._at = None  # and of the book; None: there is no step
        self._info = (c_int64 * 3)()  # tokens, rows that a rotary table has to have, whether all tokens' positions are known
        self._rooms = {}  # of workspaces, by heads and counted tokens
        self._scale = 1.0 / math.sqrt(cache.head_dim)

    def _step(self, what, n):
        c, counts, same = self.cache, None, n
        if not isinstance(n, int) and not _one(n):
            if len(n) != self._n:
                raise ValueError(f"{self._n} sequences and {len(n)} counts")
            counts, same = _long(n), 0
        else:
            n = same = operator.index(n)
        if counts is None and not -1 << 63 <= n < 1 << 63:
            raise OverflowError(f"{n} is beyond 64 bits")
        rc = _lib_call.infllm_packed_book_step(c._book_ref, what, self._ids, self._opened, self._n, counts, same, self._table, self._as_of,
                                               self._info)
        if rc:
            _checked(rc)
        if what == _lib.PACKED_RETRACT:
            self.tokens, self._at = 0, None
        else:
            self.tokens, self._at, self._rooms = self._info[0], c._book.changes, {}

    def _layer(self, layer):
        c = self.cache
        if not 0 <= layer < c.n_layers:
            raise ValueError(f"layer {layer} of {c.n_layers}")
        if self._at == c._book.changes:
            return
        if self._at is None:
            raise ValueError("no step: extend() or plan() says what it is about")
        for s, x in zip(self.seqs, self._as_of):
            if c._state[5 * s + 4] != x:
                raise ValueError(f"sequence {s} has been changed since the step began")
        self._at = c._book.changes

    def extend(self, n):
        """Room for n more tokens of every sequence, or for n[i]: they are the step's."""
        self._step(_lib.PACKED_EXTEND, n)

    def plan(self, n):
        """The newest n tokens of every sequence, or n[i], that are there already, are the step's."""
        self._step(_lib.PACKED_PLAN, n)

    def retract(self, n):
        """Takes the newest n tokens of every sequence, or n[i], back, as a speculative decoder does with drafts.  They are tokens
        that were written since the last eviction, or that it kept as `recent`.  (What their queries have added to the weights of
        others stays.)"""
        self._step(_lib.PACKED_RETRACT, n)

    def _rows(self, t, heads, what):
        """A tensor (batch, heads, tokens, head_dim) with 16-byte aligned rows, copied if it has others; address and strides."""
        c = self.cache
        if t.shape != (self._n, heads, self.tokens, c.head_dim):
            raise ValueError(f"{what} is {tuple(t.shape)}, not {(self._n, heads, self.tokens, c.head_dim)}")
        if t.dtype != c.dtype:
            raise TypeError(f"{what} is {t.dtype}, the cache {c.dtype}")
        if t.device != c.device:
            raise RuntimeError(f"{what} must be on {c.device}: infllm_b200 has no CPU path")
        bs, hs, ts, ds = t.stride()
        at = t.data_ptr()
        if ds != 1 or (bs | hs | ts) % 8 or at % 16:
            t = t.clone(memory_format=torch.contiguous_format)
            bs, hs, ts, _ = t.stride()
            at = t.data_ptr()
        return t, at, bs, hs, ts

    def _out(self, like, heads):
        """(batch, heads, tokens, head_dim) over memory of (batch, tokens, heads, head_dim)."""
        if self.tokens == 1:
            return like.new_empty((self._n, heads, 1, self.cache.head_dim))
        return like.new_empty((self._n, self.tokens, heads, self.cache.head_dim)).permute(0, 2, 1, 3)

    def write(self, layer, k, v, q=None, rope=None):
        """The step's keys and values (batch, n_kv_heads, tokens, head_dim) into a layer of the cache, with weights of 0.  With `rope`,
        a RotaryEmbeddingESM, keys and queries are rotated to their positions.  Returns the queries (None without q)."""
        c = self.cache
        self._layer(layer)
        if not self._info[2]:
            raise ValueError("tokens that an eviction has come after are not written again")
        k, k_at, k_bs, k_hs, k_ts = self._rows(k, c.n_kv_heads, "k")
        v, v_at, v_bs, v_hs, v_ts = self._rows(v, c.n_kv_heads, "v")
        out = q_at = at = cos = sin = None
        q_bs = q_hs = q_ts = heads = rows = 0
        if q is not None:
            heads = q.size(1)
            q, q_at, q_bs, q_hs, q_ts = self._rows(q, heads, "q")
            out = self._out(q, heads)
            at = out.data_ptr()
        if rope is not None:
            if not isinstance(rope, RotaryEmbeddingESM) or rope.dim != c.head_dim:
                raise ValueError(f"rope must be a RotaryEmbeddingESM of {c.head_dim} dimensions")
            need, captured = max(self._info[1], 1), _lib.capturing(c.device)
            if captured and (rope._cos is None or rope._cos.device != c.device or need > rope._seq_len_cached):
                raise RuntimeError(f"a rotary table of {need} positions is not there, and is not made inside a capture: write once outside of it")
            tables = rope._tables(need, c.device)
            if captured and all(x[0] is not tables[0] for x in c._captured):
                c._captured.append(tables)  # (the graph goes on reading these, also when longer ones have taken their place)
            rows, cos, sin = tables[0].size(0), tables[0].data_ptr(), tables[1].data_ptr()
        rc = _lib_call.infllm_packed_write(c._ref, layer, self._table, self._n, self.tokens, k_at, k_bs, k_hs, k_ts, v_at, v_bs, v_hs, v_ts,
                                           q_at, q_bs, q_hs, q_ts, at, heads, cos, sin, rows, _lib.raw_stream(c.device))
        if rc:
            _lib.check(rc)
        return out

    def values(self, layer=None):
        """What the cache holds of the step's tokens, in its 16-bit type: keys and values (batch, n_kv_heads, tokens, head_dim) of a layer,
        or (n_layers, batch, ..) of all."""
        c = self.cache
        self._layer(0 if layer is None else layer)
        first, n = (0, c.n_layers) if layer is None else (layer, 1)
        size = (self._n, c.n_kv_heads, self.tokens, c.head_dim)
        if layer is None:
            size = (n, *size)
        k = torch.empty(size, dtype=c.dtype, device=c.device)
        v = torch.empty(size, dtype=c.dtype, device=c.device)
        _lib.check(_lib_call.infllm_packed_values(c._ref, first, n, self._table, self._n, self.tokens, k.data_ptr(), v.data_ptr(),
                                                  _lib.raw_stream(c.device)))
        return k, v

    def attend(self, layer, q, scale=None, return_lse=False, weigh=False, decay=1.0):
        """Attention of the step's queries (batch, n_heads, tokens, head_dim) to their sequences' keys up to their own places.
        `scale` of the scores, not negative: 1 / sqrt(head_dim) if not given.  Returns (batch, n_heads, tokens, head_dim), a view of
        (batch, tokens, n_heads, head_dim); with return_lse also the scores' log-sum-exps (batch, n_heads, tokens), fp32.
        weigh: the layer's `weights` of the sequences that have tokens in the step become decay * weights + the probabilities that
        the tokens' queries give them, summed over the queries and the query heads of a KV head: all queries' (True), or those of
        each sequence's newest `weigh` tokens of the step.  Each such call adds."""
        c = self.cache
        self._layer(layer)
        heads = q.size(1)
        q, at, bs, hs, ts = self._rows(q, heads, "q")
        out = self._out(q, heads)
        lse = lse_at = None
        if return_lse:
            lse = torch.empty((self._n, self.tokens, heads), dtype=torch.float32, device=c.device)
            lse_at = lse.data_ptr()
        weigh = self.tokens if weigh is True else min(int(weigh), self.tokens)
        if weigh < 0:
            raise ValueError(f"the weights of {weigh} tokens")
        size = self._rooms.get((heads, weigh))
        if size is None:  # the first layer of a step
            size = c_int64()
            _lib.check(_lib_call.infllm_packed_room(c._ref, self._table, self._n, self.tokens, heads, weigh, ctypes.byref(size)))
            size = self._rooms[heads, weigh] = size.value
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=c.device)
        rc = _lib_call.infllm_packed_attend(c._ref, layer, self._table, self._n, self.tokens, at, bs, hs, ts, out.data_ptr(), lse_at, heads,
                                            self._scale if scale is None else scale, weigh, decay, work.data_ptr(), work.numel(),
                                            _lib.raw_stream(c.device))
        if rc:
            _lib.check(rc)
        return (out, lse.permute(0, 2, 1)) if return_lse else out


class PackedLayer:
    """What ATTN_FORWRAD["packed"] takes and returns as past_key_value: a layer of a step's sequences.  weigh, decay: attend()'s."""

    def __init__(self, batch, layer, weigh=False, decay=1.0):
        self.batch, self.layer, self.weigh, self.decay = batch, layer, weigh, decay


def packed_forward(*args, **kwargs):
    """ATTN_FORWRAD["packed"]: causal attention of several sequences over a PackedCache, behind the same forward(self, query,
    key_value, position_bias, use_cache, past_key_value, project_q, project_k, project_v, attention_out, dim_head, num_heads,
    num_heads_kv) as the other types (inf_llm/attention/inf_llm.py:20-32).  past_key_value is a PackedLayer; its batch was
    extended by the step's tokens before the first layer."""

    def forward(self, query, key_value, position_bias, use_cache, past_key_value, project_q, project_k, project_v,
                attention_out, dim_head, num_heads, num_heads_kv):
        if not isinstance(past_key_value, PackedLayer):
            raise TypeError('attention type "packed" needs a PackedLayer as past_key_value')
        n, tokens = query.size(0), query.size(1)
        q, k, v = (project(x).view(n, tokens, heads, dim_head).permute(0, 2, 1, 3) for project, x, heads in (
            (project_q, query, num_heads), (project_k, key_value, num_heads_kv), (project_v, key_value, num_heads_kv)))
        past = past_key_value
        q = past.batch.write(past.layer, k, v, q, position_bias)
        o = past.batch.attend(past.layer, q, weigh=past.weigh, decay=past.decay)
        o = attention_out(o.permute(0, 2, 1, 3).reshape(n, tokens, num_heads * dim_head))
        return (o, past_key_value) if use_cache else o

    return forward
