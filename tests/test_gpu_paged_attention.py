"""PagedBatch.attend and write against the formulas in 64 bits.

Tolerances, per output: u of |o| for the rounding to the 16-bit type (u = 2^-8 for bf16, 2^-11 for fp16), u of
sum_j p_j |v_j| for the probabilities, which are 16-bit operands of the product, and for what is held in 32 bits 2^-16 of that
sum (a dot product of 128 terms, and sums over 4096 keys in parts).  Of a log-sum-exp: 2^-16 of the largest sum_d |q_d k_d| of a row, scaled."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAN = float("nan")


def make(n_pages, page, kv, dim, dtype=torch.bfloat16, layers=1, **more):
    from infllm_b200.attention import PagedCache

    c = PagedCache(layers, kv, dim, n_pages, page_size=page, dtype=dtype, **more)
    c.pages.fill_(NAN)  # what no token was written to is not read
    return c


def rand(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


class Kept:
    """A cache, and the keys and values of every sequence as one tensor each."""

    def __init__(self, cache, seed):
        self.c, self.g, self.k, self.v = cache, torch.Generator(device="cuda").manual_seed(seed), {}, {}

    def open(self):
        s = self.c.open()[0]
        self.k[s] = self.v[s] = torch.empty((self.c.n_kv_heads, 0, self.c.head_dim), dtype=self.c.dtype, device="cuda")
        return s

    def grow(self, seqs, counts):
        b, most = self.c.batch(seqs), max(counts)
        b.extend(counts)
        k, v = (rand(self.g, len(seqs), self.c.n_kv_heads, most, self.c.head_dim, dtype=self.c.dtype) for _ in range(2))
        b.write(0, k, v)
        for i, (s, n) in enumerate(zip(seqs, counts)):
            self.k[s] = torch.cat((self.k[s], k[i, :, most - n:]), 1)
            self.v[s] = torch.cat((self.v[s], v[i, :, most - n:]), 1)
        return b

    def fork(self, s, n):
        kids = self.c.fork([s], n)
        for x in kids:
            self.k[x], self.v[x] = self.k[s], self.v[s]
        return kids

    def check(self, b, counts, heads, scale=None, lean=1.0):
        c, most = self.c, max(counts)
        q = rand(self.g, len(b.seqs), heads, most, c.head_dim, dtype=c.dtype, scale=lean)
        out, lse = b.attend(0, q, scale=scale, return_lse=True)
        alone = b.attend(0, q, scale=scale)
        assert torch.equal(out, alone)
        scale = 1 / math.sqrt(c.head_dim) if scale is None else scale
        u, group = U[c.dtype], heads // c.n_kv_heads
        assert out.shape == q.shape and out.dtype == c.dtype and lse.shape == q.shape[:3]
        from infllm_b200._lib import device_error

        assert device_error() == (0, 0)
        for i, (s, n) in enumerate(zip(b.seqs, counts)):
            assert (out[i, :, :most - n] == 0).all() and (lse[i, :, :most - n] == -math.inf).all()
            if n == 0:
                continue
            k, v = (x[s].double().repeat_interleave(group, 0) for x in (self.k, self.v))
            length = k.size(1)
            x = q[i, :, most - n:].double()
            sc = x @ k.transpose(1, 2) * scale
            hidden = torch.ones((n, length), dtype=torch.bool, device="cuda").triu(length - n + 1)
            sc = sc.masked_fill(hidden, -math.inf)
            p = torch.softmax(sc, -1)
            want, mass = p @ v, p @ v.abs()
            err = (out[i, :, most - n:].double() - want).abs()
            tol = u * want.abs() + (u + 2.0 ** -16) * mass
            assert (err <= tol).all(), (i, s, n, (err / tol).max().item())
            big = (x.abs() @ k.abs().transpose(1, 2)).amax() * abs(scale)
            assert ((lse[i, :, most - n:].double() - torch.logsumexp(sc, -1)).abs() <= 2.0 ** -16 * (1 + big)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,kv,group", [(16, 128, 2, 4), (128, 128, 8, 4), (32, 64, 4, 7), (64, 64, 1, 16), (128, 128, 3, 1), (64, 128, 2, 24)])
@pytest.mark.parametrize("prefix,tails", [(0, (1,)), (1, (1, 1)), (15, (2, 1, 17)), (300, (1, 5, 129, 64)), (1024, (1,) * 5), (2000, (3, 200) * 20)])
def test_one_token_each(dtype, page, dim, kv, group, prefix, tails):
    total = prefix + sum(t + 2 * page for t in tails)
    x = Kept(make(total // page + 2, page, kv, dim, dtype, max_tokens=8192), prefix + len(tails))
    root = x.open()
    if prefix:
        x.grow([root], [prefix])
    seqs = x.fork(root, len(tails))
    x.grow(seqs, list(tails))
    b = x.grow(seqs, [1] * len(tails))
    x.check(b, [1] * len(tails), kv * group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,kv,group", [(16, 128, 2, 4), (128, 128, 4, 1), (32, 64, 2, 7), (64, 128, 1, 8)])
@pytest.mark.parametrize("prefix,counts", [(0, (1000,)), (700, (33,)), (129, (7, 1, 0, 40)), (1500, (48,) * 6), (40, (300, 2, 129)), (2500, (128, 128))])
def test_several_tokens_each(dtype, page, dim, kv, group, prefix, counts):
    total = prefix + sum(t + 2 * page for t in counts)
    x = Kept(make(total // page + 2, page, kv, dim, dtype, max_tokens=8192), prefix + sum(counts))
    root = x.open()
    if prefix:
        x.grow([root], [prefix])
    seqs = x.fork(root, len(counts))
    b = x.grow(seqs, list(counts))
    x.check(b, list(counts), kv * group)
    some = [min(n, 5) for n in counts]
    b.plan(some)  # the newest tokens, asked again
    x.check(b, some, kv * group)


@pytest.mark.parametrize("page", [16, 128])
def test_a_tree_of_forks_and_strangers(page):
    _tree(page, 1)


@pytest.mark.parametrize("page", [16, 64, 128])
def test_a_tree_of_long_forks(page):
    """The same tree with 40 times the prompt: its nodes are the tensor-core kernel's."""
    _tree(page, 40 * 128 // page)


def _tree(page, long):
    x = Kept(make(4000 // page + 60 + 3 * long, page, 2, 128), 3)
    a, other, empty = x.open(), x.open(), x.open()
    x.grow([a, other], [page * 3 * long + 5, 77])
    kids = x.fork(a, 3)
    x.grow(kids, [page * 2, page * 2 + 1, 9])
    grand = x.fork(kids[0], 2) + x.fork(kids[1], 3)
    x.grow(grand, [1, 300, 2, page, 5])
    seqs = [grand[3], other, kids[2], empty, grand[0], a, grand[4], kids[1], grand[1], grand[2], kids[0]]
    b = x.c.batch(seqs)
    counts = [1, 1, 1, 0, 1, 1, 1, 1, 1, 1, 1]
    b.plan(counts)
    x.check(b, counts, 8)
    counts = [min(n, x.c.length(s)) for n, s in zip([3, 70, 9, 0, 150, 2, 5, 1, 33, 2, 2], seqs)]  # newest tokens that lie in shared pages
    b.plan(counts)
    x.check(b, counts, 8)
    ends = page * 3 * long + 9, page * (3 * long + 1)
    x.c.truncate([kids[1], grand[2]], ends)  # inside a page that others share
    for s, n in ((kids[1], ends[0]), (grand[2], ends[1])):
        x.k[s], x.v[s] = x.k[s][:, :n], x.v[s][:, :n]
    counts = [1, 1, 1, 0, 1, 1, 1, 2, 1, 2, 1]
    b.plan(counts)
    x.check(b, counts, 8)
    b = x.grow([kids[1], grand[2], kids[0]], [1, 2, 3])  # written into a copy of it
    x.check(b, [1, 2, 3], 8)
    b = x.c.batch(seqs)
    b.plan(counts)
    x.check(b, counts, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,kv,group", [(16, 128, 2, 4), (128, 128, 4, 1), (32, 64, 2, 7), (64, 64, 1, 16), (64, 128, 1, 24)])
@pytest.mark.parametrize("prefix,counts,tail", [(9000, (1,) * 40, 30), (16000, (1,) * 33, 0), (9001, (17, 0, 40, 33), 100), (0, (2000,), 0), (5000, (700, 3), 1),
                                                (12345, (1,) * 70, 3), (3000, (65,) * 9, 0), (20000, (5,), 0)])
def test_many_rows(dtype, page, dim, kv, group, prefix, counts, tail):
    """Sizes of the tensor-core kernel: nodes of one and of several row tiles and units, whole and ragged last tiles of keys, leaves
    of few rows beside them."""
    total = prefix + sum(t + tail + 2 * page for t in counts)
    x = Kept(make(total // page + 2, page, kv, dim, dtype, max_tokens=32768), prefix + sum(counts))
    root = x.open()
    if prefix:
        x.grow([root], [prefix])
    seqs = x.fork(root, len(counts))
    if tail:
        x.grow(seqs, [1 + (tail + 7 * i) % tail for i in range(len(seqs))])
    b = x.grow(seqs, list(counts))
    x.check(b, list(counts), kv * group)


@pytest.mark.parametrize("lean", [0.0, 8.0, 60.0])
def test_flat_and_peaked_scores(lean):
    x = Kept(make(200, 32, 2, 128), 5)
    root = x.open()
    x.grow([root], [3000])
    seqs = x.fork(root, 40)
    b = x.grow(seqs, [4] * 40)
    x.check(b, [4] * 40, 8, lean=lean)
    x.check(b, [4] * 40, 8, scale=0.01, lean=lean)


def test_strided_queries_and_another_layer():
    c = make(40, 16, 2, 128, layers=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    s = c.open(2)
    b = c.batch(s)
    b.extend([100, 30])
    qkv = rand(g, 2, 100, 12 * 128 + 8)  # one projection of all heads
    q, k, v = (qkv[..., a * 128:e * 128].view(2, 100, e - a, 128).permute(0, 2, 1, 3) for a, e in ((0, 8), (8, 10), (10, 12)))
    b.write(2, k, v)
    o = b.attend(2, q)
    b.write(1, k.contiguous(), v.contiguous())
    assert torch.equal(o, b.attend(1, q.contiguous()))
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)  # not 16-byte aligned
    odd.copy_(q)
    assert torch.equal(o, b.attend(1, odd))
    torch.cuda.synchronize()
    assert torch.isnan(c.pages[0]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,page,kv,heads", [(128, 16, 2, 8), (64, 64, 4, 4), (128, 128, 1, 0)])
def test_write_rotates_to_the_tokens_positions(dtype, dim, page, kv, heads):
    """Bit for bit the rotary embedding of the other attention types, at the tokens' places; nothing else is touched."""
    from infllm_b200.attention import RotaryEmbeddingESM

    c = make(60, page, kv, dim, dtype)
    rope, g = RotaryEmbeddingESM(dim, 1e4, 1.0), torch.Generator(device="cuda").manual_seed(dim)
    s = c.open(3)
    b = c.batch(s)
    pasts = [0, 21, page]
    b.extend(pasts)
    counts = [5, 37, 0]
    b.extend(counts)
    k, v = (rand(g, 3, kv, 37, dim, dtype=dtype) for _ in range(2))
    q = rand(g, 3, heads, 37, dim, dtype=dtype) if heads else None
    got = b.write(0, k, v, q, rope)
    assert (got is None) == (heads == 0)
    touched = torch.zeros_like(c.pages, dtype=torch.bool)
    for i, (n, past) in enumerate(zip(counts, pasts)):
        if n == 0:
            continue
        turned = rope.apply_rotary_pos_emb(k[i, :, 37 - n:], n, past + n)
        row = c.page_ids(s[i])
        for t in range(n):
            p, o = row[(past + t) // page], (past + t) % page
            assert torch.equal(c.pages[0, 0, p, :, o], turned[:, t]) and torch.equal(c.pages[0, 1, p, :, o], v[i, :, 37 - n + t])
            touched[0, :, p, :, o] = True
        if heads:
            assert torch.equal(got[i, :, 37 - n:], rope.apply_rotary_pos_emb(q[i, :, 37 - n:], n, past + n))
            assert (got[i, :, :37 - n] == 0).all()
    assert torch.isnan(c.pages[~touched]).all()


def test_positions_go_on_after_compaction():
    from infllm_b200.attention import RotaryEmbeddingESM

    c = make(20, 16, 1, 64)
    rope = RotaryEmbeddingESM(64, 1e4, 1.0)
    s = c.open()
    b = c.batch(s)
    b.extend(50)
    c.compact(s, [[(0, 3), (30, 50)]])
    assert (c.length(s[0]), c.position(s[0])) == (23, 50)
    b.extend(2)
    k = rand(torch.Generator(device="cuda").manual_seed(0), 1, 1, 2, 64)
    b.write(0, k, k, None, rope)
    at = c.page_ids(s[0])[1]
    assert torch.equal(c.pages[0, 0, at, :, 7:9], rope.apply_rotary_pos_emb(k[0], 2, 52))


@pytest.mark.parametrize("page,layers,kv,dim", [(16, 2, 2, 64), (128, 3, 1, 128), (32, 1, 4, 128)])
def test_fork_copy_and_compact_move_what_they_say(page, layers, kv, dim):
    from infllm_b200.attention import PagedCache

    c = make(100 * 128 // page, page, kv, dim, layers=layers)
    g = torch.Generator(device="cuda").manual_seed(page)
    c.pages.copy_(rand(g, *c.pages.shape))
    s = c.open(2)
    c.batch(s).extend([5 * page + 3, 2 * page])

    def tokens(cache, seq):
        ids = torch.tensor(cache.page_ids(seq), device="cuda", dtype=torch.long)
        assert cache.table[seq, :len(ids)].tolist() == ids.tolist()
        x = cache.pages[:, :, ids].movedim(3, 2)
        return x.reshape(layers, 2, kv, -1, dim)[:, :, :, :cache.length(seq)]

    before, was = [tokens(c, x).clone() for x in s], c.pages.clone()
    kids = c.fork(s, 70)  # more changes than a small launch takes
    for i, k in enumerate(kids):
        assert torch.equal(tokens(c, k), before[i // 70])
    assert c.page_ids(kids[0])[:5] == c.page_ids(s[0])[:5] and c.page_ids(kids[0])[5] != c.page_ids(s[0])[5]
    spans = [[(0, page), (page + 3, 2 * page + 1), (4 * page, 5 * page + 3)], [(1, 2), (3, 3), (5, 2 * page)]]
    c.compact([kids[3], kids[75]], spans)
    for k, i, sp in ((kids[3], 0, spans[0]), (kids[75], 1, spans[1])):
        assert torch.equal(tokens(c, k), torch.cat([before[i][:, :, :, a:b] for a, b in sp], 3))
    assert c.page_ids(kids[3])[0] == c.page_ids(s[0])[0]
    for i, k in enumerate(s):
        assert torch.equal(tokens(c, k), before[i])
    other = PagedCache(layers, kv, dim, 30, page_size=page, max_sequences=4, max_tokens=6 * page)
    moved = c.copy([kids[3], s[1]], into=other)
    assert torch.equal(tokens(other, moved[0]), tokens(c, kids[3])) and torch.equal(tokens(other, moved[1]), before[1])
    again = c.copy([s[0]])[0]
    assert torch.equal(tokens(c, again), before[0]) and not set(c.page_ids(again)) & set(c.page_ids(s[0]))
    c.compact([again], [[]])
    assert c.length(again) == 0 and c.page_ids(again) == []
    c.free(kids + [again])
    assert torch.equal(was[:, :, c.page_ids(s[0])], c.pages[:, :, c.page_ids(s[0])])
    assert c.free_pages == c.n_pages - 8


def test_refusals():
    from infllm_b200 import _lib as L
    from infllm_b200.attention import PagedCache, RotaryEmbeddingESM

    c = make(6, 16, 2, 64, max_sequences=4, max_tokens=64)
    s = c.open(2)
    b = c.batch(s)
    b.extend([20, 4])
    k = torch.zeros((2, 2, 20, 64), dtype=torch.bfloat16, device="cuda")
    b.write(0, k, k)
    with pytest.raises(L.InfLLMCapacityError):
        b.extend(40)  # pages
    with pytest.raises(L.InfLLMCapacityError):
        b.extend([45, 0])  # the row of the table
    assert c.length(s[0]) == 20 and c.free_pages == 3
    q = torch.zeros((2, 4, 20, 64), dtype=torch.bfloat16, device="cuda")
    for call, error in ((lambda: b.write(1, k, k), L.InfLLMError), (lambda: b.attend(-1, q), L.InfLLMError), (lambda: b.attend(0, q[:, :3]), L.InfLLMError),
                        (lambda: b.attend(0, q[:, :, :3]), ValueError), (lambda: b.attend(0, q.half()), TypeError), (lambda: b.attend(0, q.cpu()), RuntimeError),
                        (lambda: b.attend(0, q, scale=-1.0), L.InfLLMError), (lambda: b.attend(0, q, scale=NAN), L.InfLLMError),
                        (lambda: b.write(0, k, k[..., :32]), ValueError), (lambda: b.write(0, k, k, q, RotaryEmbeddingESM(128)), ValueError),
                        (lambda: c.batch([s[0], s[0]]), L.InfLLMError), (lambda: c.batch([]), L.InfLLMError), (lambda: b.plan([30, 1]), L.InfLLMError),
                        (lambda: b.plan([1]), ValueError), (lambda: b.retract([21, 0]), L.InfLLMError), (lambda: c.truncate(s, [1]), ValueError),
                        (lambda: c.compact(s, [[(0, 1)]]), ValueError), (lambda: c.compact(s, [[(0, 1, 2)], []]), ValueError),
                        (lambda: PagedCache(1, 2, 96, 4), L.InfLLMError), (lambda: PagedCache(1, 2, 64, 4, page_size=24), L.InfLLMError),
                        (lambda: PagedCache(1, 2, 64, 4, dtype=torch.float32), TypeError), (lambda: PagedCache(1, 2, 64, 4, device="cpu"), ValueError),
                        (lambda: PagedCache(0, 2, 64, 4), ValueError)):
        with pytest.raises(error):
            call()
    kid = c.fork([s[0]], 1)
    both = c.batch([s[0], kid[0]])
    both.plan([20, 20])
    with pytest.raises(L.InfLLMError):  # shared pages are not written
        both.write(0, k, k)
    b.plan(1)
    assert b.attend(0, q[:, :, :1]).shape == (2, 4, 1, 64)
    c.free([s[1]])
    with pytest.raises(L.InfLLMError):
        b.attend(0, q[:, :, :1])
    b = c.batch([s[0]])
    b.extend(1)
    b.retract(1)
    assert b.attend(0, q[:1, :, :0]).shape == (1, 4, 0, 64)  # no token is newest


def test_drafts_are_taken_back():
    x = Kept(make(60, 16, 2, 128), 9)
    root = x.open()
    x.grow([root], [100])
    seqs = x.fork(root, 3)
    x.grow(seqs, [5, 6, 7])
    b = x.c.batch(seqs)
    free = x.c.free_pages
    b.extend(30)
    junk = rand(x.g, 3, 2, 30, 128)
    b.write(0, junk, junk)
    b.retract(30)
    assert x.c.free_pages == free
    b = x.grow(seqs, [2, 2, 2])
    x.check(b, [2, 2, 2], 8)


def test_another_stream_than_the_default():
    x = Kept(make(60, 16, 2, 128), 11)
    root = x.open()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x.grow([root], [500])
        seqs = x.fork(root, 6)
        b = x.grow(seqs, [1] * 6)
        x.check(b, [1] * 6, 8)


@pytest.mark.parametrize("n_seqs,n,prefix", [(3, 1, 900), (40, 1, 900), (3, 30, 900), (40, 1, 9000), (3, 30, 9000)])
@pytest.mark.parametrize("what", [NAN, math.inf])
def test_what_is_no_number_stays_in_its_row(n_seqs, n, prefix, what):
    """A query that is no number, and a key of a sequence's own that is none, reach that row and that sequence alone."""
    c = make(prefix // 16 + 400, 16, 2, 128)
    g = torch.Generator(device="cuda").manual_seed(2)
    root = c.open()
    b = c.batch(root)
    b.extend(prefix)
    b.write(0, rand(g, 1, 2, prefix, 128), rand(g, 1, 2, prefix, 128))
    seqs = c.fork(root, n_seqs)
    b = c.batch(seqs)
    b.extend(n)
    k, v, q = (rand(g, n_seqs, h, n, 128) for h in (2, 2, 8))
    b.write(0, k, v)
    fine = b.attend(0, q)
    odd = q.clone()
    odd[1, 5, 0, 3] = what
    got = b.attend(0, odd)
    bad = torch.zeros_like(fine, dtype=torch.bool)
    bad[1, 5, 0] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], fine[~bad])
    k[2, 1, 0, 7] = what
    b.write(0, k, v)
    got = b.attend(0, q)
    bad = torch.zeros_like(fine, dtype=torch.bool)
    bad[2, 4:] = True  # the KV head's query heads
    assert torch.equal(got[~bad], fine[~bad])
    assert (torch.isnan(got[bad]).any() if what == math.inf else torch.isnan(got[bad]).all())


def test_pages_far_into_a_large_pool():
    """Offsets past 32 bits, in bytes and in elements: the last pages of 9 GB, of the second of two layers."""
    n_pages = 9000
    x = Kept(make(n_pages, 128, 8, 128, layers=2, max_tokens=n_pages * 128), 13)
    c = x.c
    filler = c.open()
    c.batch(filler).extend((n_pages - 100) * 128)
    root = x.open()
    x.grow([root], [4000])
    seqs = x.fork(root, 12)
    b = x.grow(seqs, [1] * 12)
    assert min(c.page_ids(seqs[0])) >= n_pages - 100
    x.check(b, [1] * 12, 32)
    b = x.c.batch(seqs[:2])
    b.extend(40)
    k, v, q = (rand(x.g, 2, h, 40, 128) for h in (8, 8, 32))
    b.write(0, k, v)
    b.write(1, k, v)
    at = torch.tensor(c.page_ids(root), device="cuda")
    c.pages[1, :, at] = c.pages[0, :, at]  # (the forks' shared and own pages, in the other layer too)
    for s in seqs[:2]:
        own = torch.tensor(c.page_ids(s)[31:], device="cuda")
        c.pages[1, :, own] = c.pages[0, :, own]
    assert torch.equal(b.attend(0, q), b.attend(1, q))
    small = c.copy(seqs[:1])
    ids = [torch.tensor(c.page_ids(s), device="cuda") for s in (seqs[0], small[0])]
    n = c.length(seqs[0])
    one, other = (c.pages[:, :, i].movedim(3, 2).reshape(2, 2, 8, -1, 128)[:, :, :, :n] for i in ids)
    assert torch.equal(one, other)


def test_batch_goes_while_another_stream_reads_its_plan():
    """The plan is made on one stream and read on another, which is held up meanwhile: its memory is not given away before."""
    kept = Kept(make(200, 16, 2, 64), 77)
    seqs = [kept.open()]
    kept.grow(seqs, [700])
    seqs += kept.fork(seqs[0], 5)
    kept.grow(seqs, [3, 20, 1, 40, 9, 17])
    b = kept.c.batch(seqs)
    b.plan(1)
    q = rand(kept.g, len(seqs), 8, 1, 64)
    want = b.attend(0, q)
    torch.cuda.synchronize()
    stream, size = torch.cuda.Stream(), b._work.numel()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)  # (some 50 ms)
        got = b.attend(0, q)
    del b
    filled = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(not x.any() for x in filled)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("what", ["truncate", "compact", "retract"])
def test_a_write_after_a_cut_touches_nothing(page, what):
    """The step's tokens are gone, and their places in front of the sequence's pages another's: the write is refused."""
    from infllm_b200 import _lib as L
    from infllm_b200.attention import RotaryEmbeddingESM

    c = make(12, page, 2, 64)
    s = c.open(2)
    c.batch(s[:1]).extend(page)
    b = c.batch(s)
    b.extend([1, 40])
    k = torch.zeros((2, 2, 40, 64), dtype=torch.bfloat16, device="cuda")
    if what == "truncate":
        c.truncate(s[1:], [2])
    elif what == "compact":
        c.compact(s[1:], [[(3, 5)]])
    else:
        other = c.batch(s[1:])
        other.plan(1)
        other.retract(39)
    for rope in (None, RotaryEmbeddingESM(64, 1e4, 1.0)):
        with pytest.raises(L.InfLLMError, match="since the step began"):
            b.write(0, k, k, None, rope)
    torch.cuda.synchronize()
    assert torch.isnan(c.pages).sum() == c.pages.numel()
    b.extend(2)
    b.write(0, k[:, :, :2], k[:, :, :2])
    assert (~torch.isnan(c.pages)).sum() == 2 * 2 * 2 * 2 * 64


def test_attend_again_after_its_workspace_found_no_memory(monkeypatch):
    """The next call plans anew, with memory of the size that the longer sequences need."""
    x = Kept(make(300, 16, 2, 128), 21)
    root = x.open()
    x.grow([root], [40])
    b = x.grow([root], [1])
    x.check(b, [1], 8)
    x.grow([root], [3000])
    b.plan(200)
    q = rand(x.g, 1, 8, 200, 128)
    empty, small = torch.empty, b._work.numel()

    def none(*a, **k):
        if k.get("dtype") is torch.uint8:
            raise torch.cuda.OutOfMemoryError("no memory")
        return empty(*a, **k)

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", none)
        for _ in range(2):
            with pytest.raises(torch.cuda.OutOfMemoryError):
                b.attend(0, q)
    x.check(b, [200], 8)
    assert b._work.numel() > small


@pytest.mark.parametrize("scale", [0.0, 1e-50, 1e-42, 1e-30])
@pytest.mark.parametrize("prefix,counts", [(9000, (1,) * 40), (9001, (17, 0, 40, 33)), (0, (2000,)), (300, (1, 1)), (5000, (700, 3))])
def test_scales_of_nearly_nothing(scale, prefix, counts):
    """Every key that a row sees has the same share: the mean of the values, by the kernel of few rows and by the tensor cores' one."""
    x = Kept(make((prefix + 40 * 60 + 2000) // 16, 16, 2, 128, max_tokens=32768), prefix)
    root = x.open()
    if prefix:
        x.grow([root], [prefix])
    seqs = x.fork(root, len(counts))
    b = x.grow(seqs, list(counts))
    x.check(b, list(counts), 8, scale=scale)


def test_scales_that_are_none_to_base_2():
    """Scores are scaled by scale * log2(e): where that is no number in 32 bits, neither is what would come out."""
    from infllm_b200 import _lib as L

    c = make(300, 16, 2, 128)
    s = c.open()
    b = c.batch(s)
    b.extend(4)
    k = torch.zeros((1, 2, 4, 128), dtype=torch.bfloat16, device="cuda")
    b.write(0, k, k)
    q = torch.zeros((1, 8, 4, 128), dtype=torch.bfloat16, device="cuda")
    for scale in (2.4e38, 3e38, 1e39, math.inf):
        with pytest.raises(L.InfLLMError):
            b.attend(0, q, scale=scale)
    assert (b.attend(0, q, scale=2.3e38) == 0).all()


def test_a_plan_is_not_uploaded_by_a_graph():
    """The copy of a plan would not run while a graph is captured, and would read another plan when it is replayed; a step's later calls
    can be captured, and are replayed within it."""
    from infllm_b200 import _lib as L

    x = Kept(make(900, 16, 2, 128), 31)
    root = x.open()
    x.grow([root], [9000])
    seqs = x.fork(root, 40)
    b = x.grow(seqs, [2] * 40)
    q = rand(x.g, 40, 8, 2, 128)
    torch.cuda.synchronize()
    with pytest.raises(L.InfLLMError, match="captures"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.attend(0, q)
    want = b.attend(0, q)
    x.check(b, [2] * 40, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b.attend(0, q)
    for _ in range(3):
        got.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_pages_do_not_change_in_a_graph():
    """The device's copy of the table would be changed by replays alone, while the host goes on at once: refused, and nothing changes.
    A step within pages that are there can be captured."""
    from infllm_b200 import _lib as L

    c, g = make(40, 16, 2, 128), torch.Generator(device="cuda").manual_seed(4)
    s = c.open(2)
    b = c.batch(s)
    b.extend([20, 16])
    k = rand(g, 2, 2, 1, 128)
    torch.cuda.synchronize()
    for call in (lambda: b.extend(1), lambda: c.fork(s, 1), lambda: c.copy(s), lambda: c.compact(s[:1], [[(3, 20)]])):
        with pytest.raises(L.InfLLMError, match="captures"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        assert c.free_pages == 37 and [c.length(x) for x in s] == [20, 16] and c.open() == [2]
        c.free([2])
    graph = torch.cuda.CUDAGraph()
    b = c.batch(s[:1])
    with torch.cuda.graph(graph):
        b.extend(1)
        b.write(0, k[:1], k[:1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.pages[0, 0, c.page_ids(s[0])[1], :, 4], k[0, :, 0]) and torch.isnan(c.pages).sum() == c.pages.numel() - 512


@pytest.mark.parametrize("how", ["attend", "check"])
def test_a_wait_that_ran_out_is_reported(how):
    """By the cache whose kernel gave it up, once.  (Set from the host: nothing is made to time out on the GPU.)"""
    from infllm_b200 import _lib as L

    c, other = make(40, 16, 2, 128), make(40, 16, 2, 128)
    b, of_other = (x.batch(x.open()) for x in (c, other))
    for x in (b, of_other):
        x.extend(20)
        k = torch.zeros((1, 2, 20, 128), dtype=torch.bfloat16, device="cuda")
        x.write(0, k, k)
    q = torch.zeros((1, 8, 20, 128), dtype=torch.bfloat16, device="cuda")
    L.check(L.lib.infllm_pages_error_set(c.handle, 1, 712))
    assert not torch.isnan(of_other.attend(0, q)).any()
    other.check()
    with pytest.raises(L.InfLLMError, match="wait 712") as e:
        b.attend(0, q) if how == "attend" else c.check()
    assert e.value.code == L.E_TIMEOUT
    c.check()
    assert not torch.isnan(b.attend(0, q)).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,kv,group", [(128, 2, 4), (64, 2, 7), (128, 1, 16)])
@pytest.mark.parametrize("prefix,tails", [(0, (24,)), (0, (1, 3, 70)), (32, (5, 9)), (300, (20, 1, 64))])
def test_few_rows_round_their_output_alone(dtype, dim, kv, group, prefix, tails):
    """The kernel of few rows holds a probability as two 16-bit numbers, so that the rounding of the output is the only one of 16 bits:
    the output lies between the roundings of (o - rest) and of (o + rest), where `rest` has no rounding to 16 bits in it.

    rest: of sum_j p_j |v_j| 2^-16 for what is held in 32 bits, and u^2 (2^-16, 2^-22) for what the second number leaves of p_j; fp16 has
    a least step of 2^-24, by half of which a p_j may be off: 2^-25 sum_j |v_j| over the sum of the unnormalised p, which is at least 1."""
    x = Kept(make((prefix + sum(tails)) // 16 + 3 * len(tails) + 2, 16, kv, dim, dtype), prefix + dim)
    root = x.open()
    if prefix:
        x.grow([root], [prefix])
    seqs = x.fork(root, len(tails))
    b = x.grow(seqs, list(tails))
    b.plan(1)
    q = rand(x.g, len(seqs), kv * group, 1, dim, dtype=dtype)
    out = b.attend(0, q)
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for i, s in enumerate(seqs):
        k, v = (t[s].double().repeat_interleave(group, 0) for t in (x.k, x.v))
        p = torch.softmax(q[i].double() @ k.transpose(1, 2) / math.sqrt(dim), -1)
        want, mass = p @ v, p @ v.abs()
        rest = (2.0 ** -16 + U[dtype] ** 2) * mass + least * v.abs().sum(1, keepdim=True)
        assert ((want - rest).to(dtype) <= out[i]).all() and (out[i] <= (want + rest).to(dtype)).all(), i
