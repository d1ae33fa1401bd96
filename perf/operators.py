"""Workloads of the paged key/value cache: several continuations of one long prompt, which share its pages.

Kinds of work (the "kind" of a case):

attend    attention of the newest `new` tokens of `batch` sequences, which are forks of one prompt of `prefix` tokens with
          up to `tail` tokens of their own behind it: one token each is a decode step, more are questions put to a long
          document, or (batch 1) a chunk of a prompt
write     one layer's keys and values of `new` tokens of every sequence into its pages, keys and queries rotated to the
          tokens' positions; pages are taken for them, and given back at the end of the pass
fork      `children` continuations of a sequence: shared pages, and a copy of the page that is not full, in every layer
compact   a copy of `batch` sequences with only some stretches of their tokens: the first ones and the newest ones (sink
          and window), or every other memory unit

Where `own` is false, a pass is elementary torch operations in 32 bits on the same pages.  Pages are taken lowest number
first, for one sequence after the other; so both forms put the same things into the same pages.

Sizes are those of the repository's benchmark configurations (32 query heads over 8 or 32 KV heads of 128 dimensions, units
of 128 tokens, chunks of 8192 tokens, contexts up to 131072 tokens) and odd ones of the same kind.
"""
import heapq
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BASE = 1e6  # of the rotary embedding
UNIT = 128  # tokens of a memory unit


def _attend(batch, prefix, tail, new=1, heads=32, kv_heads=8, dim=128, page=128, dtype="bf16", **more):
    return dict(kind="attend", batch=batch, prefix=prefix, tail=tail, new=new, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype, **more)


def _write(batch, past, new, heads=32, kv_heads=8, dim=128, page=128, dtype="bf16", **more):
    return dict(kind="write", batch=batch, past=past, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, **more)


def _fork(children, length, layers, kv_heads=8, dim=128, page=128, dtype="bf16", **more):
    return dict(kind="fork", children=children, length=length, layers=layers, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, **more)


def _compact(batch, length, policy, layers, kv_heads=8, dim=128, page=128, dtype="bf16", **more):
    return dict(kind="compact", batch=batch, length=length, policy=policy, layers=layers, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype, **more)


def listed():
    return [
        # a decode step of four answers to a short prompt: the smallest call of a generation loop
        _attend(4, 1024, 40, page=16, name="tokens_4_on_1k"),
        # the same of 32 samples of an answer over a 32K-token document
        _attend(32, 32768, 300, name="tokens_32_on_32k"),
        # many samples over the longest context of the benchmark configurations
        _attend(128, 131072, 800, name="tokens_128_on_128k"),
        # 28 query heads over 4 KV heads of 64 dimensions, fp16, small pages, a prompt that ends inside a page
        _attend(13, 5003, 700, heads=28, kv_heads=4, dim=64, page=32, dtype="fp16", name="tokens_13_odd_fp16"),
        # eight questions of 48 tokens to one document, each read at once
        _attend(8, 16384, 48, new=48, page=64, name="questions_8_on_16k"),
        # a chunk of a prompt: 2048 tokens behind 28000
        _attend(1, 28000, 2048, new=2048, name="chunk_2048_on_28k"),
        # a decode step's token of each of 64 sequences
        _write(64, 5000, 1, name="write_64_tokens"),
        # the chunk in which prompts are read, fp16, as many KV heads as query heads
        _write(1, 8192, 8192, kv_heads=32, dtype="fp16", name="write_chunk_8192"),
        # four answers to a short prompt are begun
        _fork(4, 1000, 2, page=32, name="fork_4_of_1k"),
        # 64 samples over a 32K-token document, eight layers
        _fork(64, 32749, 8, name="fork_64_of_32k"),
        # a sequence is cut down to its first and its newest tokens
        _compact(1, 3001, "window", 2, page=16, name="compact_window_3k"),
        # half the memory units of two long sequences are dropped, four layers
        _compact(2, 65536, "units", 4, name="compact_units_64k"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "fork", "compact"])
    dim = rng.choice([64, 128, 128])
    kv, group = rng.choice([(1, 8), (2, 2), (4, 7), (8, 1), (8, 4), (8, 4), (32, 1)])
    more = dict(kv_heads=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 128]), dtype=rng.choice(["bf16", "fp16"]))
    if kind == "attend":
        c = _attend(_log(rng, 1, 128), rng.choice([0, 1, 1, 1, 1, 1]) * _log(rng, 100, 131072), _log(rng, 1, 2000), heads=kv * group, **more)
        if rng.random() < 0.4:
            c["new"] = _log(rng, 2, 2048)
            c["tail"] = max(c["tail"], c["new"])
        most = 128 * 32 * 131072 * 0.9  # query rows by keys, and the sequences' own pages in 32 bits
        while c["batch"] * c["new"] * c["heads"] * (c["prefix"] + c["tail"]) > most or c["batch"] * c["tail"] * kv * dim > 1 << 28:
            c["batch"] = (c["batch"] + 1) // 2
            c["prefix"] = c["prefix"] * 2 // 3
            c["new"] = (c["new"] + 1) // 2
        return c
    if kind == "write":
        new = rng.choice([1, _log(rng, 1, 8192)])
        return _write(max(1, min(_log(rng, 1, 128), 16384 // new)), _log(rng, 1, 20000), new, heads=kv * group, **more)
    layers = rng.randint(1, 8)
    if kind == "fork":
        c = _fork(_log(rng, 1, 64), _log(rng, 10, 33000), layers, **more)
        while c["layers"] > 1 and c["layers"] * kv * dim * (2 * c["length"] + c["children"] * c["page"]) > 1 << 29:
            c["layers"] = (c["layers"] + 1) // 2
        return c
    c = _compact(rng.randint(1, 3), _log(rng, 300, 65536), rng.choice(["window", "units", "ragged"]), layers, **more)
    while c["layers"] * kv * dim * c["batch"] * c["length"] > 1 << 28:
        if c["layers"] > 1:
            c["layers"] = (c["layers"] + 1) // 2
        else:
            c["length"] = (c["length"] + 1) // 2
    return c


def _pages_of(tokens, page):
    return -(-tokens // page)


class _Book:
    """Which pages a sequence has: the rows of the page table, lengths, and how many sequences use a page."""

    def __init__(self, n_pages, page):
        self.page, self.free, self.uses, self.rows, self.lens = page, list(range(n_pages)), [0] * n_pages, [], []

    def take(self):
        p = heapq.heappop(self.free)
        self.uses[p] = 1
        return p

    def drop(self, p):
        self.uses[p] -= 1
        if self.uses[p] == 0:
            heapq.heappush(self.free, p)

    def open(self):
        self.rows.append([])
        self.lens.append(0)
        return len(self.rows) - 1

    def extend(self, s, n):
        self.lens[s] += n
        while len(self.rows[s]) < _pages_of(self.lens[s], self.page):
            self.rows[s].append(self.take())

    def truncate(self, s, n):
        self.lens[s] = n
        while len(self.rows[s]) > _pages_of(n, self.page):
            self.drop(self.rows[s].pop())

    def fork(self, s):
        """A child, and the pages (from, to) that have to be copied for it."""
        c = self.open()
        n, full = self.lens[s], self.lens[s] // self.page
        self.lens[c], self.rows[c] = n, self.rows[s][:full]
        for p in self.rows[c]:
            self.uses[p] += 1
        if n % self.page == 0:
            return c, []
        self.rows[c].append(self.take())
        return c, [(self.rows[s][full], self.rows[c][full])]

    def close(self, s):  # the last one that was opened
        assert s == len(self.rows) - 1
        self.truncate(s, 0)
        self.rows.pop()
        self.lens.pop()


def _tails(case):
    """Tokens that each sequence of an attend case has of its own, the newest included: from one to `tail`."""
    r = random.Random("%(batch)d %(prefix)d %(tail)d %(new)d" % case)
    return [r.randint(case["new"], max(case["new"], case["tail"])) for _ in range(case["batch"])]


def _pasts(case):
    r = random.Random("%(batch)d %(past)d" % case)
    return [r.randint(max(1, case["past"] // 2), case["past"]) for _ in range(case["batch"])]


def _keep(case):
    """The stretches of tokens that stay of a sequence of a compact case."""
    n = case["length"]
    if case["policy"] == "window":
        return [(0, min(UNIT, n // 8)), (n - n // 3, n)]
    if case["policy"] == "units":
        return [(a, min(a + UNIT, n)) for a in range(0, n, 2 * UNIT)]
    r, spans, at = random.Random(n), [], 0
    while at < n:  # stretches of any length at any place
        stop = min(n, at + r.randint(1, 300))
        spans.append((at, stop))
        at = stop + r.randint(1, 200)
    return spans


def _kept(case):
    return sum(b - a for a, b in _keep(case))


def _script(case, cache):
    """Brings a cache or a book to where the pass begins, by the same steps; returns the sequences."""
    kind = case["kind"]
    if kind == "attend":
        root = cache.open()
        cache.extend(root, case["prefix"])
        seqs = [cache.fork(root)[0] for _ in range(case["batch"])]
        for s, n in zip(seqs, _tails(case)):
            cache.extend(s, n)
        return seqs
    if kind == "write":
        seqs = [cache.open() for _ in range(case["batch"])]
        pasts = _pasts(case)
        for part in (2, 1):  # in two steps, so that the pages of a sequence are not in order
            for s, n in zip(seqs, pasts):
                cache.extend(s, n // 2 if part == 2 else n - n // 2)
        return seqs
    seqs = [cache.open() for _ in range(case.get("batch", 1))]
    other = cache.open()
    left = case["length"]
    while left:  # another sequence has grown beside them, and is gone: their pages lie among free ones
        n = min(left, 5 * case["page"] + 3)
        for s in seqs:
            cache.extend(s, n)
        if cache.lens[other] < 2000:
            cache.extend(other, case["page"])
        left -= n
    cache.close(other)
    return seqs


class _Framework:
    """The framework's cache behind the names that _script uses."""

    def __init__(self, cache):
        self.cache, self.lens = cache, {}

    def open(self):
        s = self.cache.open()[0]
        self.lens[s] = 0
        return s

    def extend(self, s, n):
        if n:
            self.cache.batch([s]).extend(n)
        self.lens[s] += n

    def fork(self, s):
        kids = self.cache.fork([s], 1)
        self.lens[kids[0]] = self.lens[s]
        return kids

    def close(self, s):
        self.cache.free([s])


def _pool(case):
    """Pages of the pool: what the case uses at its largest, and some more."""
    page, kind = case["page"], case["kind"]
    if kind == "attend":
        return _pages_of(case["prefix"], page) + sum(1 + _pages_of(n + page, page) for n in _tails(case)) + 3
    if kind == "write":
        return sum(_pages_of(n + case["new"], page) + 1 for n in _pasts(case)) + 3
    if kind == "fork":
        return _pages_of(case["length"], page) + case["children"] + _pages_of(2000, page) + 3
    return case["batch"] * (_pages_of(case["length"], page) + _pages_of(_kept(case), page) + 1) + _pages_of(2000, page) + 3


def _longest(case):
    kind = case["kind"]
    if kind == "attend":
        return case["prefix"] + max(_tails(case))
    return max(_pasts(case)) + case["new"] if kind == "write" else case["length"]


def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kv, dim, page, layers = _DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"], case.get("layers", 1)
    n_pages = _pool(case)
    # the whole pool, so that what lies behind a sequence's end is what another one left there
    pages = torch.empty((layers, 2, n_pages, kv, page, dim), dtype=dtype, device="cuda")
    for layer in pages:
        for part in layer:
            part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float32))
    max_sequences = case.get("batch", 1) + case.get("children", 1) + 130
    if own:
        from infllm_b200.attention import PagedCache, RotaryEmbeddingESM

        cache = PagedCache(layers, kv, dim, n_pages, page_size=page, max_sequences=max_sequences, max_tokens=_longest(case),
                           dtype=dtype)
        seqs = _script(case, _Framework(cache))
        cache.pages.copy_(pages)
        pages = cache.pages
        state = {"case": case, "cache": cache, "seqs": seqs, "pages": pages}
        rows = [cache.page_ids(s) for s in seqs]
    else:
        book = _Book(n_pages, page)
        seqs = _script(case, book)
        table = torch.zeros((max_sequences, _pages_of(_longest(case), page)), dtype=torch.int32)
        for s, row in enumerate(book.rows):
            table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        state = {"case": case, "book": book, "seqs": seqs, "pages": pages, "table": table.cuda()}
        rows = [book.rows[s] for s in seqs]
    if case["kind"] == "attend":
        b, h, n = case["batch"], case["heads"], case["new"]
        q = _randn(g, torch.float32, b, n, h, dim)
        # every sequence's first tokens draw some of all its heads' attention; the rest is spread
        lean = _randn(g, torch.float32, kv, dim)
        lean /= lean.norm(dim=-1, keepdim=True)
        q += 3 * lean.repeat_interleave(h // kv, 0)
        pages[0, 0, rows[0][0], :, :4] += (6 * lean[:, None]).to(dtype)
        state["q"] = q.to(dtype).permute(0, 2, 1, 3)  # (batch, heads, tokens, dim), as a projection's view
        # the sequences' pages and lengths are laid out once a step, for the calls of all layers
        if own:
            batch = state["batch"] = cache.batch(seqs)
            batch.plan(n)
        else:
            state["lens"] = torch.tensor([book.lens[s] for s in seqs], device="cuda")
            state["rows"] = state["table"][torch.tensor(seqs, device="cuda")].long()
            state["shared"] = case["prefix"] // page if b > 1 else 0  # pages
    if case["kind"] == "write":
        b, h, n = case["batch"], case["heads"], case["new"]
        state["q"] = _randn(g, dtype, b, n, h, dim).permute(0, 2, 1, 3)
        state["k"] = _randn(g, dtype, b, n, kv, dim).permute(0, 2, 1, 3)
        state["v"] = _randn(g, dtype, b, n, kv, dim).permute(0, 2, 1, 3)
        if own:
            state["rope"], state["batch"] = RotaryEmbeddingESM(dim, BASE, 1.0), cache.batch(seqs)
        else:
            angle = torch.arange(_longest(case), dtype=torch.float32)[:, None] * (1.0 / BASE ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))
            state["cos"], state["sin"] = angle.cos().cuda(), angle.sin().cuda()
    if case["kind"] == "compact":
        state["keep"] = [_keep(case)] * case["batch"]
    return state


# ------------------------------------------------------------------------------------------------- plain forms
def _rows32(pages, ids):
    """(..., n) page numbers -> (..., kv, n * page, dim) rows in 32 bits."""
    x = pages[ids].float()  # (..., n, kv, page, dim)
    x = x.movedim(-3, -4)
    return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], x.shape[-1])


def _plain_attend(s):
    """out = softmax(q k^T / sqrt(dim)) v: the scores of the shared pages, read once for all, beside those of each sequence's
    own; a query sees the keys up to its own place."""
    case, q, lens = s["case"], s["q"], s["lens"]
    b, h, n, dim = q.shape
    kv, shared = case["kv_heads"], s["shared"]
    table = s["rows"]
    x = q.float().reshape(b, kv, h // kv * n, dim)
    k0, v0 = (_rows32(s["pages"][0, i], table[0, :shared]) for i in (0, 1))   # (kv, keys, dim)
    k1, v1 = (_rows32(s["pages"][0, i], table[:, shared:]) for i in (0, 1))   # (b, kv, keys, dim)
    ours = torch.matmul(x, k1.transpose(-1, -2))
    # all sequences' queries of a KV head are the rows of one product
    theirs = torch.matmul(x.transpose(0, 1).reshape(kv, b * h // kv * n, dim), k0.transpose(-1, -2))
    scores = torch.cat((theirs.view(kv, b, h // kv * n, k0.shape[1]).transpose(0, 1), ours), dim=-1) / math.sqrt(dim)
    place = lens[:, None] - n + torch.arange(n, device="cuda")  # (b, n)
    seen = torch.arange(scores.shape[-1], device="cuda") <= place[:, None, :, None]
    scores = scores.view(b, h, n, -1).masked_fill_(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    p = (p / p.sum(dim=-1, keepdim=True)).view(b, kv, h // kv * n, -1)
    at = shared * case["page"]
    out = torch.matmul(p[..., at:], v1)
    out += torch.matmul(p[..., :at].transpose(0, 1).reshape(kv, b * h // kv * n, at), v0).view(kv, b, h // kv * n, dim).transpose(0, 1)
    return out.view(b, h, n, dim).to(q.dtype)


def _rotate32(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)


def _plain_write(s):
    case, book, seqs, n = s["case"], s["book"], s["seqs"], s["case"]["new"]
    past = [book.lens[i] for i in seqs]
    for i in seqs:
        book.extend(i, n)
    width = max(len(book.rows[i]) for i in seqs)
    rows = torch.tensor([book.rows[i] + [0] * (width - len(book.rows[i])) for i in seqs]).cuda()
    s["table"][torch.tensor(seqs).cuda(), :width] = rows.int()
    place = torch.tensor(past).cuda()[:, None] + torch.arange(n, device="cuda")  # (b, n)
    cos, sin = s["cos"][place][:, None], s["sin"][place][:, None]
    at, offset = torch.gather(rows, 1, place // case["page"]), place % case["page"]
    pages = s["pages"][0]
    pages[0, at, :, offset] = _rotate32(s["k"], cos, sin).transpose(1, 2)
    pages[1, at, :, offset] = s["v"].transpose(1, 2)
    q = _rotate32(s["q"], cos, sin)
    for i, m in zip(seqs, past):
        book.truncate(i, m)
    return q, s["pages"]


def _plain_fork(s):
    case, book, seq = s["case"], s["book"], s["seqs"][0]
    kids, copies = zip(*(book.fork(seq) for _ in range(case["children"])))
    copies = [c for one in copies for c in one]
    if copies:
        at = torch.tensor(copies).cuda()
        s["pages"][:, :, at[:, 1]] = s["pages"][:, :, at[:, 0]]
    width = len(book.rows[seq])
    s["table"][torch.tensor(kids).cuda(), :width] = torch.tensor([book.rows[k] for k in kids], dtype=torch.int32).cuda()
    got = s["pages"], s["table"][kids[0]:kids[-1] + 1, :width], len(book.free)
    for k in reversed(kids):
        book.close(k)
    return got


def _plain_compact(s):
    case, book, page = s["case"], s["book"], s["case"]["page"]
    kids = []
    copies = []
    for seq in s["seqs"]:
        kid, more = book.fork(seq)
        kids.append(kid)
        copies += more
    if copies:
        at = torch.tensor(copies).cuda()
        s["pages"][:, :, at[:, 1]] = s["pages"][:, :, at[:, 0]]
    kept, gone = _kept(case), []
    for kid, keep in zip(kids, s["keep"]):
        place = torch.cat([torch.arange(a, b) for a, b in keep])
        stay = 0  # pages at the front that nothing is dropped from
        while (stay + 1) * page <= kept and place[(stay + 1) * page - 1] == (stay + 1) * page - 1:
            stay += 1
        old = book.rows[kid]
        book.rows[kid] = old[:stay] + [book.take() for _ in range(_pages_of(kept, page) - stay)]
        book.lens[kid] = kept
        src, dst = place[stay * page:], torch.arange(stay * page, kept)
        a, b = torch.tensor(old)[src // page].cuda(), torch.tensor(book.rows[kid])[dst // page].cuda()
        s["pages"][:, :, b, :, (dst % page).cuda()] = s["pages"][:, :, a, :, (src % page).cuda()]
        gone += old[stay:]
    for p in gone:
        book.drop(p)
    width = _pages_of(kept, page)
    s["table"][torch.tensor(kids).cuda(), :width] = torch.tensor([book.rows[k] for k in kids], dtype=torch.int32).cuda()
    got = s["pages"], s["table"][kids[0]:kids[-1] + 1, :width], len(book.free)
    for k in reversed(kids):
        book.close(k)
    return got


# ------------------------------------------------------------------------------------------- one pass through an operator
def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"attend": _plain_attend, "write": _plain_write, "fork": _plain_fork, "compact": _plain_compact}[kind](s)
    if kind == "attend":
        return s["batch"].attend(0, s["q"])
    cache, seqs = s["cache"], s["seqs"]
    if kind == "write":
        batch = s["batch"]
        batch.extend(s["case"]["new"])
        q = batch.write(0, s["k"], s["v"], s["q"], s["rope"])
        batch.retract(s["case"]["new"])
        return q, s["pages"]
    if kind == "fork":
        kids = cache.fork(seqs, s["case"]["children"])
    else:
        kids = cache.fork(seqs, 1)
        cache.compact(kids, s["keep"])
    width = _pages_of(cache.length(kids[0]), s["case"]["page"])
    got = s["pages"], cache.table[kids[0]:kids[-1] + 1, :width], cache.free_pages
    cache.free(kids)
    return got


def work(case):
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    token = 2 * kv * dim * 2  # bytes of a token's keys and values in one layer
    if case["kind"] == "attend":
        b, h, n, tails = case["batch"], case["heads"], case["new"], _tails(case)
        keys = case["prefix"] + sum(tails)
        pairs = sum(n * (case["prefix"] + t) - n * (n - 1) / 2 for t in tails)
        return {"bytes": keys * token + 2 * b * h * n * dim * 2, "flops": 4.0 * h * dim * pairs}
    if case["kind"] == "write":
        tokens = case["batch"] * case["new"]
        values = tokens * (case["heads"] + kv) * dim
        return {"bytes": tokens * (2 * token + 4 * case["heads"] * dim), "flops": 3.0 * values}
    if case["kind"] == "fork":
        part = case["length"] % page * token * case["layers"]
        rows = (1 + case["children"]) * _pages_of(case["length"], page) * 4
        return {"bytes": part * (1 + case["children"]) + rows, "flops": 0}
    moved = sum(b - a for a, b in _keep(case) if a) * case["batch"]  # (the first stretch stays where it is, but for a page's end)
    return {"bytes": 2 * moved * token * case["layers"] + case["batch"] * _pages_of(_kept(case), page) * 4, "flops": 0}


# --------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    kind, page = case["kind"], case["page"]
    s = prepare(case, seed)
    book, pages, seqs = s["book"], s["pages"], s["seqs"]

    def tokens(seq, part, layer=0):  # (kv, length, dim), one sequence at a time
        x = pages[layer, part, torch.tensor(book.rows[seq], device="cuda")].double()
        return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :book.lens[seq]]

    if kind == "attend":
        out, n, kv = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), case["new"], case["kv_heads"]
        group = case["heads"] // kv
        for i, seq in enumerate(seqs):
            k, v = tokens(seq, 0), tokens(seq, 1)
            hidden = torch.ones((n, k.shape[1]), dtype=torch.bool, device="cuda").triu(k.shape[1] - n + 1)
            for j in range(kv):
                x = torch.einsum("gnd,kd->gnk", s["q"][i, j * group:(j + 1) * group].double(), k[j]) / math.sqrt(case["dim"])
                out[i, j * group:(j + 1) * group] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v[j]
        return out
    if kind == "write":
        half = case["dim"] // 2
        freq = BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        pool, turned = pages.double(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, seq in enumerate(seqs):
            past = book.lens[seq]
            place = torch.arange(past, past + case["new"], device="cuda")
            wave = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), place[:, None].double() * freq)

            def turn(x):
                z = torch.complex(x[..., :half].double(), x[..., half:].double()) * wave
                return torch.cat((z.real, z.imag), dim=-1)

            turned[i] = turn(s["q"][i])
            k, v = turn(s["k"][i]), s["v"][i].double()
            book.extend(seq, case["new"])
            for p in range(past // page, len(book.rows[seq])):
                a, b = max(past, p * page), min(past + case["new"], (p + 1) * page)
                pool[0, 0, book.rows[seq][p], :, a - p * page:b - p * page] = k[:, a - past:b - past]
                pool[0, 1, book.rows[seq][p], :, a - p * page:b - p * page] = v[:, a - past:b - past]
        return turned, pool
    return None  # copies: equal to the plain form's
