"""PackedCache where numbers are at the ends of their types, or are none.  Tolerances as in test_gpu_packed_cache.py, but for what a test says itself."""
import math

import pytest
import torch
from test_gpu_packed_cache import INF, NAN, SHAPES, TINY, U, check, fill, formula, gen, held, make, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,dtype", [(128, torch.float16), (64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("group,n", [(1, 1), (4, 1), (4, 2), (7, 1), (4, 20), (4, 70), (4, 300)])
@pytest.mark.parametrize("below,spread", [(11.0, 0.0), (15.0, 0.0), (17.0, 0.3), (18.0, 0.0)])
def test_many_small_probabilities_beside_a_large_one(dim, dtype, group, n, below, spread):
    """A token whose value is zero has nearly all of the attention; the output is what 8192 others, `below` nats less, have left.  (64
    sequences, all the same, so that a unit of work has long stretches of them.)

    Up to eight rows probabilities are as good as 32 bits, so that of the sum of p |v| only what is held in 32 bits is lost.  Of more rows each is
    rounded to 16 bits: by u of itself, or, where an fp16 number has less bits, by half of 2^-24 in units of which the largest has
    2^11 or more: N 2^-36 max |v| in all."""
    g, length, kv, seqs = gen(31), 8193, 8, 64 if n < 100 else 8
    c = make(kv, dim, seqs, length, dtype)
    b = c.batch(c.open(seqs))
    b.extend(length)
    k = rand(g, 1, 1, length, dim, dtype=dtype, scale=spread)
    v = (1 + 0.25 * torch.randn((1, 1, length, dim), generator=g, device="cuda")).to(dtype)
    k[0, 0, 0], v[0, 0, 0] = below / math.sqrt(dim), 0
    b.write(0, k.expand(seqs, kv, -1, -1), v.expand(seqs, kv, -1, -1))
    b.plan(n)
    out, lse = b.attend(0, torch.ones((seqs, kv * group, n, dim), dtype=dtype, device="cuda"), return_lse=True)
    k, v = (x[-1:] for x in held(c, 0, seqs - 1))
    want, mass, want_lse, p, e = formula(torch.ones((group, n, dim), device="cuda"), k, v, n, 1 / math.sqrt(dim))
    few = group * n <= 8
    tol = U[dtype] * want.abs() + ((0 if few else U[dtype]) + 2.0 ** -16 + 2 * e[..., None]) * mass + TINY[dtype]
    if not few and dtype == torch.float16:
        tol = tol + length * 2.0 ** -36 * v.abs().max()
    err = (out[-1, -group:].double() - want).abs()
    assert (err <= tol).all(), ((err / tol).max().item(), (err / want.abs()).max().item())
    assert ((lse[-1, -group:].double() - want_lse).abs() <= e + 2.0 ** -20 * want_lse.abs() + 1e-6).all()


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES[:3])
@pytest.mark.parametrize("length,n,at", [
    (500, 1, "newest"), (512, 1, "newest"), (500, 1, "deep"), (500, 4, "newest"), (509, 2, "middle"), (500, 40, "newest"), (500, 40, "middle"), (500, 9, "deep"),
    (700, 200, "all"), (900, 700, "middle"), (900, 900, "all"), (20000, 1, "newest"), (20000, 40, "all"), (20000, 600, "middle"), (20000, 600, "newest")])
def test_a_value_that_is_none_takes_its_own_dimensions_alone(dim, kv, heads, dtype, length, n, at):
    """The 32 numbers of a value that are none: so are these dimensions of the rows that see it.  The others, log-sum-exps and weights do
    not depend on them, and are bit for bit what they are beside a finite value."""
    g, group = gen(32), heads // kv
    c = make(kv, dim, 2, length + 5, dtype)
    s = c.open(2)[1:]
    b = c.batch(s)
    b.extend(length)
    k, v = (rand(g, 1, kv, length, dim, dtype=dtype) for _ in range(2))
    places = {"newest": [length - 1], "deep": [13], "middle": [length - n // 2 - 1], "all": [length - n, length - n // 2, length - 2, length - 1]}[at]
    places = [(x, i % (dim // 32), (kv - 1) * (1 - i % 2)) for i, x in enumerate(places)]  # token, group, KV head
    for x, y, h in places:
        v[0, h, x, 32 * y:32 * y + 32] = 0
    q = rand(g, 1, heads, n, dim, dtype=dtype)

    def attend():
        b.plan(length)
        b.write(0, k, v)
        b.plan(n)
        out, lse = b.attend(0, q, return_lse=True, weigh=True, decay=0.0)
        return out, lse, c.weights[0, s[0], :, :length].clone()

    fine, fine_lse, fine_weights = attend()
    assert fine.isfinite().all() and fine_lse.isfinite().all() and fine_weights.isfinite().all()
    want = fine.clone()
    for i, (x, y, h) in enumerate(places):
        v[0, h, x, 32 * y + 7] = (INF, NAN, -INF)[i % 3]
        want[0, h * group:(h + 1) * group, max(0, x - (length - n)):, 32 * y:32 * y + 32] = NAN
    out, lse, weights = attend()
    assert torch.equal(lse, fine_lse) and torch.equal(weights, fine_weights)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(-9), want.nan_to_num(-9))


@pytest.mark.parametrize("dim,kv,heads,dtype", [x for x in SHAPES if x[3] == torch.bfloat16])
@pytest.mark.parametrize("length,n", [(150, 2), (150, 12), (250, 60), (900, 700), (9000, 40)])
def test_the_largest_values_do_not_reach_rows_that_do_not_see_them(dim, kv, heads, dtype, length, n):
    g, hidden = gen(33), n // 2
    c = make(kv, dim, 1, length, dtype)
    b = c.batch(c.open())
    k, v = (rand(g, 1, kv, length, dim, dtype=dtype) for _ in range(2))
    q = rand(g, 1, heads, n, dim, dtype=dtype)
    b.extend(length)
    got = []
    for large in (0.0, 2.0 ** 120):
        v[:, :, length - hidden:] = large
        b.plan(length)
        b.write(0, k, v)
        b.plan(n)
        got.append(b.attend(0, q)[:, :, :n - hidden])
    assert torch.equal(*got)


@pytest.mark.parametrize("prefix,n", [(700, 40), (0, 2000), (9000, 300)])
def test_the_largest_values_of_pages_do_not_reach_rows_that_do_not_see_them(prefix, n):
    """The same of the paged cache."""
    from infllm_b200.attention import PagedCache

    g, hidden = gen(35), n // 2
    c = PagedCache(1, 2, 128, 150, page_size=64)
    b = c.batch(c.open())
    b.extend(prefix + n)
    k, v = (rand(g, 1, 2, prefix + n, 128) for _ in range(2))
    q = rand(g, 1, 8, n, 128)
    got = []
    for large in (0.0, 2.0 ** 120):
        v[:, :, prefix + n - hidden:] = large
        b.plan(prefix + n)
        b.write(0, k, v)
        b.plan(n)
        got.append(b.attend(0, q)[:, :, :n - hidden])
    assert torch.equal(*got)


@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("n", [1, 3, 8, 40, 200])
@pytest.mark.parametrize("length,some", [(300, 200), (300, 299), (5000, 4900)])
def test_scores_of_minus_infinity_are_probabilities_of_zero(heads, n, length, some):
    """The first `some` tokens' scores do not fit 32 bits: the others have the attention, in equal parts."""
    g = gen(34)
    c = make(1, 128, 1, length)
    b = c.batch(c.open())
    b.extend(length)
    k = torch.zeros((1, 1, length, 128), dtype=torch.bfloat16, device="cuda")
    k[:, :, :some] = -2.0 ** 100
    k[:, :, 0] = 0  # (every row sees a score that fits)
    v = rand(g, 1, 1, length, 128)
    b.write(0, k, v)
    b.plan(n)
    out, lse = b.attend(0, torch.full((1, heads, n, 128), 2.0 ** 100, dtype=torch.bfloat16, device="cuda"), return_lse=True, weigh=True, decay=0.0)
    assert (k == held(c, 0, 0)[0]).all()
    v, at = held(c, 0, 0)[1][0], torch.arange(length, device="cuda")
    seen = ((at >= some) | (at == 0)) & (at <= torch.arange(length - n, length, device="cuda")[:, None])
    p = seen.double() / seen.sum(-1, keepdim=True)
    tol = U[c.dtype] * (p @ v).abs() + (U[c.dtype] + 2.0 ** -16) * (p @ v.abs())
    assert ((out[0].double() - p @ v).abs() <= tol).all()
    assert ((lse[0].double() - seen.sum(-1).double().log()).abs() <= 1e-5).all()
    assert ((c.weights[0, 0, 0].double() - heads * p.sum(0)).abs() <= 2.0 ** -18 * heads * p.sum(0)).all()


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES[:4] + [(128, 3, 6, torch.bfloat16), (128, 1, 5, torch.float16)])
@pytest.mark.parametrize("lengths,counts", [([1], [1]), ([15, 16, 17], [1, 1, 1]), ([64, 65, 3, 700], [1, 0, 1, 1]), ([5000], [1]), ([2049, 130], [2, 1]), ([60000], [4])])
def test_up_to_eight_rows_round_their_output_alone(dim, kv, heads, dtype, lengths, counts):
    """Their probabilities are as good as 32 bits: 2^-16 of sum_j p_j |v_j| beside the output's own rounding."""
    counts = [min(x, 8 * kv // heads) for x in counts]
    g, most = gen(sum(lengths) + dim), max(counts)
    c = make(kv, dim, len(lengths) + 1, max(lengths) + 3, dtype)
    seqs = c.open(len(lengths) + 1)[1:]
    b = fill(c, g, seqs, lengths)
    b.plan(counts)
    q = rand(g, len(seqs), heads, most, dim, dtype=dtype, scale=1.5)
    out, lse = b.attend(0, q, return_lse=True)
    check(c, b, counts, q, out, lse)
    for i, (s, n) in enumerate(zip(seqs, counts)):
        if n:
            k, v = held(c, 0, s)
            want, mass, _, p, e = formula(q[i, :, most - n:], k, v, n, 1 / math.sqrt(dim))
            err = (out[i, :, most - n:].double() - want).abs()
            tol = U[dtype] * want.abs() + (2.0 ** -16 + 2 * e[..., None]) * mass + TINY[dtype]
            assert (err <= tol).all(), (i, (err / tol).max().item())
            if dtype == torch.bfloat16 and 15 <= k.size(1) <= 1000:  # (probabilities of 16 bits would not do)
                p, v, top = p.cpu(), v.cpu().repeat_interleave(heads // kv, 0), p.amax(-1, keepdim=True).cpu()
                assert (((p / top).to(dtype).double() * top @ v - want.cpu()).abs() > tol.cpu()).any(), i


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES[:3])
def test_a_prompt_and_single_tokens_in_one_call(dim, kv, heads, dtype):
    """All of them go to the kernel of many rows then: each sequence's rows are the formulas', as they are alone."""
    g, lengths, counts = gen(36), [900] + [40 + 97 * i for i in range(20)], [600] + [1] * 20
    c = make(kv, dim, 21, max(lengths), dtype)
    b = fill(c, g, c.open(21), lengths)
    q = rand(g, 21, heads, 600, dim, dtype=dtype, scale=1.5)
    c.weights.fill_(0.5)
    before = c.weights.clone()
    b.plan(counts)
    out, lse = b.attend(0, q, return_lse=True, weigh=1, decay=0.5)
    check(c, b, counts, q, out, lse, weigh=1, before=before, decay=0.5)
    alone = c.batch(b.seqs[1:])
    alone.plan(1)
    out1, lse1 = alone.attend(0, q[1:, :, -1:], return_lse=True)
    check(c, alone, [1] * 20, q[1:, :, -1:], out1, lse1)


def test_calls_of_many_sizes_one_after_the_other():
    """Workspaces are not cleared between calls, whose memory is the allocator's: what one has left does not reach the next."""
    g, calls = gen(37), []
    c = make(2, 128, 6, 3000)
    seqs = c.open(6)
    fill(c, g, seqs, [3000, 1, 700, 129, 2048, 31])
    for s, n, weigh in ((seqs, 1, True), (seqs[:1], 900, True), (seqs[2:5], 100, False), (seqs[:1], 3000, 7), (seqs[4:], 8, True), (seqs[:3:2], 2, False), (seqs[1:2], 1, True)):
        b = c.batch(s)
        b.plan([min(n, c.length(x)) for x in s])
        q = rand(g, len(s), 8, b.tokens, 128)
        calls.append(lambda b=b, q=q, weigh=weigh: (*b.attend(0, q, return_lse=True, weigh=weigh, decay=0.0), c.weights[0, b.seqs].clone()))
    want = []
    for call in calls:
        torch.cuda.empty_cache()
        want.append(call())
    for i in [0, 3, 6, 1, 5, 2, 4, 0, 6, 3, 1, 4, 2, 5, 3, 0] * 2:
        junk = torch.full((1 << 22,), NAN, device="cuda")  # (numbers that are none in what the allocator gives next)
        del junk
        assert all(torch.equal(x.nan_to_num(-9), y.nan_to_num(-9)) for x, y in zip(calls[i]()[:2], want[i][:2])), i
