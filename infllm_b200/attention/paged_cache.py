"""A paged key/value cache for several continuations of one prompt, and attention that reads shared pages once.

The reference's caches hold one stream each (inf_llm/attention/context_manager.py:196-816, stream_llm.py:6-111); this
one is for a program that samples many answers to a long prompt, keeps beams, or puts many questions to one document:

    cache = PagedCache(n_layers, n_kv_heads, head_dim, n_pages)
    root = cache.open()[0]
    prompt = cache.batch([root])
    prompt.extend(len_prompt)                              # once per step ...
    q = prompt.write(layer, k, v, q, rope)                 # ... then in every layer
    o = prompt.attend(layer, q)
    answers = cache.batch(cache.fork([root], 64))          # 64 sequences that share the prompt's pages
    answers.extend(1); ...

Tensors are (batch, heads, tokens, head_dim) views with any strides whose rows are 16-byte aligned, as the other
attention types take them.  Work goes to the current stream; all calls on a cache belong on one stream, or are ordered by
the caller."""
import ctypes
import math
from array import array
from ctypes import c_int32, c_int64

import torch

from .. import _lib
from .rope import RotaryEmbeddingESM

_lib_call = _lib.lib


# ctypes cuts what does not fit, which would name another sequence or count: OverflowError instead.  (Of a few numbers one by one, as
# an array costs 0.4 us more than that; of 64 it takes a third of the time.)
def _one(n):
    if not -0x80000000 <= n <= 0x7fffffff:
        raise OverflowError(f"{n} is beyond 32 bits")
    return n


def _ids(seqs):
    n = len(seqs)
    if n < 8:
        for x in seqs:
            if not -0x80000000 <= x <= 0x7fffffff:
                raise OverflowError(f"{x} is beyond 32 bits")
        return (c_int32 * n)(*seqs)
    return (c_int32 * n).from_buffer(array("i", seqs))


def _long(values):
    n = len(values)
    if n < 8:
        for x in values:
            if not -1 << 63 <= x < 1 << 63:
                raise OverflowError(f"{x} is beyond 64 bits")
        return (c_int64 * n)(*values)
    return (c_int64 * n).from_buffer(array("q", values))


class PagedCache:
    """`n_pages` pages of `page_size` tokens (16, 32, 64 or 128), each with the keys and values of all layers, and up to
    `max_sequences` sequences of up to `max_tokens` tokens over them.  head_dim is 64 or 128, dtype bfloat16 or float16.

    `pages` (n_layers, 2, n_pages, n_kv_heads, page_size, head_dim) and `table` (max_sequences, max_pages) are the device's
    memory of it.  Sequences are named by small numbers.  What does not fit raises InfLLMCapacityError and changes nothing."""

    def __init__(self, n_layers, n_kv_heads, head_dim, n_pages, page_size=128, max_sequences=256, max_tokens=131072,
                 dtype=torch.bfloat16, device=None):
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"a CUDA device is needed, got {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_layers, self.n_kv_heads, self.head_dim = int(n_layers), int(n_kv_heads), int(head_dim)
        self.n_pages, self.page_size, self.max_sequences = int(n_pages), int(page_size), int(max_sequences)
        self.dtype = dtype
        if min(self.n_layers, self.n_kv_heads, self.head_dim, self.n_pages, self.page_size, self.max_sequences, int(max_tokens)) < 1:
            raise ValueError("sizes of a paged cache are positive")
        max_pages = -(-int(max_tokens) // self.page_size)
        self.pages = torch.zeros((self.n_layers, 2, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim), dtype=dtype,
                                 device=self.device)
        self.table = torch.zeros((self.max_sequences, max_pages), dtype=torch.int32, device=self.device)
        cfg = _lib.PagesConfig(self.n_layers, self.n_kv_heads, self.head_dim, self.page_size, self.n_pages, self.max_sequences,
                               max_pages, _lib.dtype_code(dtype), self.device.index, 0, self.pages.data_ptr(), self.table.data_ptr())
        self.handle = ctypes.c_void_p()
        _lib.check(_lib_call.infllm_pages_create(ctypes.byref(cfg), ctypes.byref(self.handle)))

    def __del__(self):
        try:
            if self.handle:
                _lib_call.infllm_pages_destroy(self.handle)
        except Exception:
            pass
        self.handle = None

    # -- sequences
    def open(self, n=1):
        """n new, empty sequences: their numbers, the lowest that are not in use."""
        out = (c_int32 * n)()
        _lib.check(_lib_call.infllm_pages_open(self.handle, n, out))
        return list(out)

    def fork(self, seqs, n=1):
        """n continuations of each of `seqs`, one sequence's after the other's.  They share its full pages; a last page that is not
        full is copied, in all layers."""
        out = (c_int32 * (len(seqs) * n))()
        _lib.check(_lib_call.infllm_pages_fork(self.handle, _ids(seqs), len(seqs), n, out, _lib.raw_stream(self.device)))
        return list(out)

    def copy(self, seqs, into=None):
        """Copies of `seqs` that share no pages, here or `into` another PagedCache with pages of the same shape."""
        into = self if into is None else into
        out = (c_int32 * len(seqs))()
        _lib.check(_lib_call.infllm_pages_copy(self.handle, _ids(seqs), len(seqs), into.handle, out, _lib.raw_stream(self.device)))
        return list(out)

    def truncate(self, seqs, lengths):
        """Cuts each sequence to a length."""
        if len(seqs) != len(lengths):
            raise ValueError(f"{len(seqs)} sequences and {len(lengths)} lengths")
        _lib.check(_lib_call.infllm_pages_truncate(self.handle, _ids(seqs), _long(lengths), len(seqs)))

    def free(self, seqs):
        """Ends sequences; pages that no other one shares are free."""
        _lib.check(_lib_call.infllm_pages_free(self.handle, _ids(seqs), len(seqs)))

    def compact(self, seqs, keep):
        """Of each sequence only the tokens of keep[i], a list of ascending (start, stop), stay, and close up.  Keys keep the
        rotation that they were written with, and position() goes on from where it was.  Pages at the front that stay whole
        are kept, and stay shared; the other tokens move to pages of the sequence's own."""
        if len(seqs) != len(keep):
            raise ValueError(f"{len(seqs)} sequences and {len(keep)} lists of spans")
        flat = [x for spans in keep for span in spans for x in span]
        counts = [len(spans) for spans in keep]
        if len(flat) != 2 * sum(counts):
            raise ValueError("spans are pairs (start, stop)")
        _lib.check(_lib_call.infllm_pages_compact(self.handle, _ids(seqs), len(seqs), _long(flat), (c_int32 * len(keep))(*counts),
                                                  _lib.raw_stream(self.device)))

    def batch(self, seqs):
        return PagedBatch(self, seqs)

    def check(self):
        """Waits for the current stream, and raises InfLLMError (E_TIMEOUT) where an attention kernel has given up a wait and left
        rows unwritten.  attend() reports that too, but of calls whose kernels have run by then."""
        _lib.check(_lib_call.infllm_pages_check(self.handle, _lib.raw_stream(self.device)))

    # -- what there is
    def _info(self, seq):
        length, position = c_int64(), c_int64()
        _lib.check(_lib_call.infllm_pages_info(self.handle, _one(seq), ctypes.byref(length), ctypes.byref(position)))
        return length.value, position.value

    def length(self, seq):
        """Tokens of a sequence."""
        return self._info(seq)[0]

    def position(self, seq):
        """The position that its next token is rotated to: the tokens that it has had (compact() takes none of them back)."""
        return self._info(seq)[1]

    def page_ids(self, seq):
        n = ctypes.c_int()
        out = (c_int32 * self.table.size(1))()
        _lib.check(_lib_call.infllm_pages_row(self.handle, _one(seq), out, len(out), ctypes.byref(n)))
        return out[:n.value]

    @property
    def free_pages(self):
        return _lib_call.infllm_pages_free_count(self.handle)


class PagedBatch:
    """Sequences that take a step together.  extend(), or plan(), says how many of each one's newest tokens the step is about;
    write() and attend() are then called in every layer.  Tensors have as many tokens as the largest of those counts; a
    sequence with fewer has its own at the end, and what is before them is not read, and zero in what is returned."""

    def __init__(self, cache, seqs):
        self.cache, self.seqs = cache, list(seqs)
        self._n = len(self.seqs)
        self.tokens = 0  # of the step's tensors
        self._work, self._work_at = None, 0  # the plan on the device, and room for partial results
        self._work_stream = None  # that its memory is of
        self._reach = c_int64()  # rows that a rotary table has to have
        self._reach_ref = ctypes.byref(self._reach)
        self._scale = 1.0 / math.sqrt(cache.head_dim)
        self.handle = ctypes.c_void_p()
        _lib.check(_lib_call.infllm_page_batch_create(cache.handle, _ids(self.seqs), self._n, ctypes.byref(self.handle)))

    def __del__(self):
        try:
            if self.handle:
                _lib_call.infllm_page_batch_destroy(self.handle)
        except Exception:
            pass
        self.handle = None

    def _counts(self, n):
        if isinstance(n, int):
            return None, _one(n), n
        if len(n) != self._n:
            raise ValueError(f"{self._n} sequences and {len(n)} counts")
        return _ids(n), 0, max(n)

    def extend(self, n):
        """Room for n more tokens of every sequence, or for n[i]: they are the step's."""
        counts, same, most = self._counts(n)
        rc = _lib_call.infllm_page_batch_extend(self.handle, counts, same, self._reach_ref, _lib.raw_stream(self.cache.device))
        if rc:
            _lib.check(rc)
        self.tokens = most

    def plan(self, n):
        """The newest n tokens of every sequence, or n[i], that are there already, are the step's."""
        counts, same, most = self._counts(n)
        _lib.check(_lib_call.infllm_page_batch_select(self.handle, counts, same, self._reach_ref))
        self.tokens = most

    def retract(self, n):
        """Takes the newest n tokens of every sequence, or n[i], back, as a speculative decoder does with drafts."""
        counts, same, _ = self._counts(n)
        rc = _lib_call.infllm_page_batch_retract(self.handle, counts, same)
        if rc:
            _lib.check(rc)
        self.tokens = 0

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
        """The step's keys and values (batch, n_kv_heads, tokens, head_dim) into a layer's pages.  With `rope`, a
        RotaryEmbeddingESM, keys and queries are rotated to their positions.  Returns the queries (None without q).  Refused where one
        of the sequences was cut, compacted or extended by another call since the step began."""
        c = self.cache
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
            cos, sin = rope._tables(max(self._reach.value, 1), c.device)
            rows, cos, sin = cos.size(0), cos.data_ptr(), sin.data_ptr()
        rc = _lib_call.infllm_page_batch_write(self.handle, layer, k_at, k_bs, k_hs, k_ts, v_at, v_bs, v_hs, v_ts, q_at, q_bs, q_hs, q_ts,
                                               at, heads, cos, sin, rows, _lib.raw_stream(c.device))
        if rc:
            _lib.check(rc)
        return out

    def attend(self, layer, q, scale=None, return_lse=False):
        """Attention of the step's queries (batch, n_heads, tokens, head_dim) to their sequences' keys up to their own places.
        `scale` of the scores, not negative: 1 / sqrt(head_dim) if not given.  Returns (batch, n_heads, tokens, head_dim), a view of
        (batch, tokens, n_heads, head_dim); with return_lse also the scores' log-sum-exps (batch, n_heads, tokens), fp32.  A batch's
        calls share a workspace: on several streams, one waits for the other as for any tensor that both use.  A step's first call is
        refused while a CUDA graph is captured; later ones may be, for replays within the step."""
        c = self.cache
        heads = q.size(1)
        q, at, bs, hs, ts = self._rows(q, heads, "q")
        out = self._out(q, heads)
        lse = lse_at = None
        if return_lse:
            lse = torch.empty((self._n, self.tokens, heads), dtype=torch.float32, device=c.device)
            lse_at = lse.data_ptr()
        scale = self._scale if scale is None else scale
        stream = _lib.raw_stream(c.device)
        rc = _lib.PAGES_NO_PLAN
        if self._work_at:
            rc = _lib_call.infllm_page_batch_attend(self.handle, layer, at, bs, hs, ts, out.data_ptr(), lse_at, heads, scale, self._work_at,
                                                    stream)
        if rc == _lib.PAGES_NO_PLAN:  # the first layer of a step
            size = c_int64()
            # a plan goes with the memory that was made for it, or with none: the last one's may be too small for it
            self._work, self._work_at = None, 0
            _lib.check(_lib_call.infllm_page_batch_plan(self.handle, heads, ctypes.byref(size)))
            self._work = torch.empty(max(size.value, 16), dtype=torch.uint8, device=c.device)
            self._work_at, self._work_stream = self._work.data_ptr(), stream
            rc = _lib_call.infllm_page_batch_attend(self.handle, layer, at, bs, hs, ts, out.data_ptr(), lse_at, heads, scale, self._work_at,
                                                    stream)
            if rc:  # (memory of a graph that is captured is not for calls outside it)
                self._work, self._work_at = None, 0
        elif stream != self._work_stream and self._work is not None:  # it is not to be given away before this stream is done with it
            self._work.record_stream(torch.cuda.current_stream(c.device))
        if rc:
            _lib.check(rc)
        return (out, lse.permute(0, 2, 1)) if return_lse else out


class PagedLayer:
    """What ATTN_FORWRAD["paged"] takes and returns as past_key_value: a layer of a step's sequences."""

    def __init__(self, batch, layer):
        self.batch, self.layer = batch, layer


def paged_forward(*args, **kwargs):
    """ATTN_FORWRAD["paged"]: full causal attention of several sequences over a PagedCache, behind the same
    forward(self, query, key_value, position_bias, use_cache, past_key_value, project_q, project_k, project_v, attention_out,
    dim_head, num_heads, num_heads_kv) as the other types (inf_llm/attention/inf_llm.py:20-32).  past_key_value is a
    PagedLayer; its batch was extended by the step's tokens before the first layer."""

    def forward(self, query, key_value, position_bias, use_cache, past_key_value, project_q, project_k, project_v,
                attention_out, dim_head, num_heads, num_heads_kv):
        if not isinstance(past_key_value, PagedLayer):
            raise TypeError('attention type "paged" needs a PagedLayer as past_key_value')
        n, tokens = query.size(0), query.size(1)
        q, k, v = (project(x).view(n, tokens, heads, dim_head).permute(0, 2, 1, 3) for project, x, heads in (
            (project_q, query, num_heads), (project_k, key_value, num_heads_kv), (project_v, key_value, num_heads_kv)))
        batch, layer = past_key_value.batch, past_key_value.layer
        o = batch.attend(layer, batch.write(layer, k, v, q, position_bias))
        o = attention_out(o.permute(0, 2, 1, 3).reshape(n, tokens, num_heads * dim_head))
        return (o, past_key_value) if use_cache else o

    return forward
