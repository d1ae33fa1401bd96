"""PackedCache against its definitions in 64 bits.

What is held is compared bit for bit: a group's least number and step, and every code, have one value.  Attention is compared with the
formulas over the numbers that the codes stand for.  Tolerances, per output: u of |o| for the rounding to the 16-bit type (u = 2^-8
for bf16, 2^-11 for fp16), u of sum_j p_j |v_j| for the probabilities, which are 16-bit operands of the product where rows are many,
and for what is held in 32 bits 2^-16 of that sum (a dot product of 128 terms, and sums over thousands of keys in parts).  Of a log-sum-exp
e = 2^-16 of the largest sum_d |q_d k_d| of a row, scaled: a score is off by that.  So a probability exp(s - lse) is off by 2 e of itself,
an output by 2 e of sum_j p_j |v_j| more, and the weights, sums of probabilities in 32 bits, by that and 2^-18.  Probabilities below
2^-126 are none in 32 bits (2^13 keys with values of 2^3: 2^-110), and half of an fp16 output's last place is 2^-25."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -110, torch.float16: 2.0 ** -25}
NAN, INF = float("nan"), float("inf")


def make(kv, dim, n_sequences, max_tokens, dtype=torch.bfloat16, layers=1):
    from infllm_b200.attention import PackedCache

    c = PackedCache(layers, kv, dim, n_sequences, max_tokens, dtype=dtype)
    c.scales.fill_(NAN)  # what no token was written to is not read
    c.codes.fill_(0x55555555)
    c.weights.fill_(NAN)
    c.places.fill_(-7)
    return c


def rand(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pack64(x):
    """codes (.., dim), least and step (.., dim / 32) of rows x (.., dim), from the definition."""
    y = x.double().unflatten(-1, (-1, 32))
    least = y.amin(-1)
    step = ((y.amax(-1) - least) / 15).float().to(x.dtype)
    if x.dtype == torch.float16:  # (the next smaller one where the largest number that the group stands for were infinite)
        over = (least + 15 * step.double()).to(x.dtype).isinf() & step.isfinite()
        step = torch.where(over, (step.view(torch.int16) - 1).view(x.dtype), step)
    step = step.double()
    c = torch.round((y - least[..., None]) / step[..., None])
    c = torch.where(step[..., None] == 0, torch.zeros_like(c), c).clamp(0, 15)
    return c.flatten(-2).long(), least, step


def stand64(c, least, step, dtype):
    c = c.unflatten(-1, (-1, 32)).double()
    return (least[..., None] + step[..., None] * c).to(dtype).double().flatten(-2)


def codes_of(words):
    w = words.long() & 0xffffffff
    return torch.stack([w >> (4 * (i // 2) + 16 * (i % 2)) & 15 for i in range(8)], -1).flatten(-2)


def held(c, layer, s, n=None):
    """What the cache's tensors say of a sequence: keys and values (kv, length, dim), 64 bits."""
    n = c.length(s) if n is None else n
    out = []
    for part in (0, 1):
        sc = c.scales[layer, part, s, :, :n].double()
        out.append(stand64(codes_of(c.codes[layer, part, s, :, :n]), sc[..., 0], sc[..., 1], c.dtype))
    return out


def formula(q, k, v, n, scale):
    """Of the newest n tokens' queries (heads, n, dim): outputs, mass, log-sum-exps, probabilities and the error of a log-sum-exp."""
    group = q.size(0) // k.size(0)
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    x, length = q.double(), k.size(1)
    hidden = torch.ones((n, length), dtype=torch.bool, device="cuda").triu(length - n + 1)
    sc = (x @ k.transpose(1, 2) * scale).masked_fill(hidden, -INF)
    p = torch.softmax(sc, -1)
    big = (x.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(hidden, 0).amax(-1)
    return p @ v, p @ v.abs(), torch.logsumexp(sc, -1), p, 2.0 ** -16 * big


def fill(c, g, seqs, lengths, layer=0, scale=1.0):
    """Tokens into sequences, all of them new."""
    b, most = c.batch(seqs), max(lengths)
    b.extend(lengths)
    k, v = (rand(g, len(seqs), c.n_kv_heads, most, c.head_dim, dtype=c.dtype, scale=s) for s in (scale, 1.0))
    b.write(layer, k, v)
    return b


def check(c, b, counts, q, out, lse, layer=0, scale=None, weigh=0, before=None, decay=1.0):
    from infllm_b200._lib import device_error

    assert device_error() == (0, 0)
    most, u = max(counts), U[c.dtype]
    scale = 1 / math.sqrt(c.head_dim) if scale is None else scale
    assert out.shape == q.shape and out.dtype == c.dtype and lse.shape == q.shape[:3]
    for i, (s, n) in enumerate(zip(b.seqs, counts)):
        assert (out[i, :, :most - n] == 0).all() and (lse[i, :, :most - n] == -INF).all()
        if n == 0:
            continue
        k, v = held(c, layer, s)
        want, mass, want_lse, p, e = formula(q[i, :, most - n:], k, v, n, scale)
        err = (out[i, :, most - n:].double() - want).abs()
        tol = u * want.abs() + (u + 2.0 ** -16 + 2 * e[..., None]) * mass + TINY[c.dtype]
        assert (err <= tol).all(), ("out", i, (err - tol).max().item(), (err / tol).max().item())
        err = (lse[i, :, most - n:].double() - want_lse).abs()
        assert (err <= e + 2.0 ** -20 * want_lse.abs() + 1e-6).all(), ("lse", i, err.max().item())
        if weigh:
            m = min(weigh, n)
            per = p[:, n - m:]
            slack = (p * (2 * e[..., None] + 2.0 ** -18))[:, n - m:]
            got = c.weights[layer, s, :, :k.size(1)].double()
            old = before[layer, s, :, :k.size(1)].double()
            want_w, tol = (x.unflatten(0, (c.n_kv_heads, -1)).sum((1, 2)) for x in (per, slack))
            want_w = want_w + (decay * old if decay else 0)
            tol = tol + 2.0 ** -22 * want_w
            err = (got - want_w).abs()
            assert (err <= tol + 1e-30).all(), ("weights", i, (err / (tol + 1e-30)).max().item())


# ------------------------------------------------------------------------------------------------------------ writes
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,kv,heads", [(128, 8, 32), (64, 1, 7), (128, 3, 3), (64, 2, 2)])
@pytest.mark.parametrize("counts", [[1], [5, 0, 17, 1], [130]])
def test_write_holds_what_the_definition_says(dtype, dim, kv, heads, counts):
    from infllm_b200.attention import RotaryEmbeddingESM

    g, n, most = gen(1), len(counts), max(counts)
    c = make(kv, dim, n + 2, 400, dtype, layers=2)
    seqs = c.open(n + 1)[1:]
    past = [3 + 50 * i for i in range(n)]
    b = c.batch(seqs)
    b.extend(past)
    b.extend(counts)
    was = [t.clone() for t in (c.codes, c.scales, c.weights, c.places)]
    k, v, q = (rand(g, n, most, h, dim, dtype=dtype).permute(0, 2, 1, 3) for h in (kv, kv, heads))
    for t in (k, v, q):  # what is before a sequence's own tokens is not read
        for i, x in enumerate(counts):
            t[i, :, :most - x] = NAN
    k[0, 0, -1, :32] = 1.5          # one number
    v[0, 0, -1, :32] = 0
    v[0, 0, -1, 32] = 1000          # one far from the others
    v[0, -1, -1, :32] = torch.arange(32, device="cuda") * 2.0 ** -20
    rope = RotaryEmbeddingESM(dim, 1e4, 1.0)
    got_q = b.write(1, k, v, q, rope)
    cos, sin = (t[:600].double() for t in rope._tables(600, c.device))

    def turned(x, p0):  # in 32 bits product by product, as the other attention types
        p = torch.arange(p0, p0 + x.size(1), device="cuda")
        a, z = x.float().chunk(2, -1)
        cs, sn = cos[p].float(), sin[p].float()
        return torch.cat((a * cs - z * sn, z * cs + a * sn), -1).to(dtype)

    back_k, back_v = b.values(1)
    for i, (s, x, p) in enumerate(zip(seqs, counts, past)):
        assert (got_q[i, :, :most - x] == 0).all() and (back_k[i, :, :most - x] == 0).all() and (back_v[i, :, :most - x] == 0).all()
        if x == 0:
            continue
        assert torch.equal(got_q[i, :, most - x:], turned(q[i, :, most - x:], p))
        for part, t, back in ((0, turned(k[i, :, most - x:], p), back_k), (1, v[i, :, most - x:], back_v)):
            codes, least, step = pack64(t)
            at = (1, part, s, slice(None), slice(p, p + x))
            assert torch.equal(codes_of(c.codes[at]), codes)
            assert torch.equal(c.scales[at].double(), torch.stack((least, step), -1))
            want = stand64(codes, least, step, dtype)
            assert torch.equal(back[i, :, most - x:].double(), want)
            # (half a step, its rounding over 15 steps, and the value's own)
            width = step.repeat_interleave(32, -1)
            assert ((want - t.double()).abs() <= width * (0.5 + 15 * U[dtype] / 2) + U[dtype] / 2 * t.double().abs() + 1e-6).all()
            was[0][at], was[1][at] = c.codes[at], c.scales[at]
        at = (1, s, slice(None), slice(p, p + x))
        assert (c.weights[at] == 0).all() and (c.places[at] == torch.arange(p, p + x, device="cuda")).all()
        was[2][at], was[3][at] = 0, c.places[at]
    for t, x in zip((c.codes, c.scales, c.weights, c.places), was):  # nothing else is touched
        assert torch.equal(torch.nan_to_num(t.double(), 123.0), torch.nan_to_num(x.double(), 123.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_group_that_is_not_finite_is_none(dtype):
    c = make(1, 128, 1, 16, dtype)
    b = c.batch(c.open())
    b.extend(4)
    k = torch.ones((1, 1, 4, 128), dtype=dtype, device="cuda") * torch.arange(128, device="cuda").to(dtype)
    want = k.clone()
    for i, x in enumerate((NAN, INF, -INF)):
        k[0, 0, i, 37 + i] = x
        want[0, 0, i, 32:64] = NAN
    b.write(0, k, torch.zeros_like(k))
    got = b.values(0)[0]
    assert torch.equal(got.isnan(), want.isnan())
    codes, least, step = pack64(k)
    want = torch.where(want.isnan(), NAN, stand64(codes, least, step, dtype))
    assert torch.equal(got.nan_to_num(-9).double(), want.nan_to_num(-9))


def test_finite_numbers_stay_finite():
    """fp16 groups at the ends of its range, whose steps are rounded up: none of what they stand for is infinite."""
    g = gen(20)
    c = make(1, 128, 1, 600, torch.float16)
    b = c.batch(c.open())
    b.extend(600)
    k = (torch.rand((1, 1, 600, 128), generator=g, device="cuda") * 65504).half()
    k[0, 0, :300, ::32] = 65504
    k[0, 0, :, 1::32] = (torch.rand((600, 4), generator=g, device="cuda") * 131008 - 65504).half()
    k[0, 0, :2, 2::32] = torch.tensor([0.0, -65504.0], device="cuda").half()[:, None]
    b.write(0, k, -k)
    smaller = 0
    for got, x in zip(b.values(0), (k, -k)):
        codes, least, step = pack64(x)
        want = stand64(codes, least, step, torch.float16)
        assert want.isfinite().all() and torch.equal(got.double(), want)
        plain = ((x.double().unflatten(-1, (-1, 32)).amax(-1) - least) / 15).float().half()
        smaller += (plain.double() != step).sum().item()
        assert ((want - x.double()).abs() <= step.repeat_interleave(32, -1) * (0.5 + 15 * U[torch.float16]) + U[torch.float16] * want.abs()).all()
    assert smaller > 100  # (the rule is at work)


@pytest.mark.parametrize("n", [2, 60])
def test_large_values_do_not_reach_rows_that_do_not_see_them(n):
    g = gen(21)
    c = make(1, 128, 1, 300, torch.float16)
    b = c.batch(c.open())
    b.extend(150 + n)
    k, v, q = (rand(g, 1, 1, x, 128, dtype=torch.float16) for x in (150 + n, 150 + n, n))
    v[0, 0, -1, ::2] = 65504
    v[0, 0, -1, 1::2] = 0
    b.write(0, k, v)
    b.plan(n)
    out, lse = b.attend(0, q, return_lse=True)
    assert out.isfinite().all()
    check(c, b, [n], q, out, lse)


@pytest.mark.parametrize("least", [0.0, -7.0, -15.0])
def test_the_widest_steps(least):
    """bf16: groups in steps of 2^121 and of the largest number below 2^122 are held, one of 2^122 and one that is wider (of least -7: its span is not finite) are not."""
    c = make(1, 128, 1, 16)
    b = c.batch(c.open())
    b.extend(1)
    code = torch.arange(32, device="cuda", dtype=torch.float64) % 16
    steps = torch.tensor([2.0 ** 121, 2.0 ** 122 * (1 - 2.0 ** -8), 2.0 ** 122, 2.0 ** 125], device="cuda", dtype=torch.float64)
    k = (steps[:, None] * (code + least)).clamp(-3.3e38, 3.3e38).to(torch.bfloat16).view(1, 1, 1, 128)
    b.write(0, k, torch.zeros_like(k))
    got = b.values(0)[0].view(4, 32)
    assert got[2:].isnan().all() and c.scales[0, 0, 0, 0, 0, 2:, 1].isnan().all()
    codes, low, step = pack64(k)
    want = stand64(codes, low, step, torch.bfloat16).view(4, 32)[:2]
    assert (step.view(4)[:2] < 2.0 ** 122).all() and torch.equal(got[:2].double(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_code_and_the_borders_between_them(dtype):
    """Groups from a to b in steps of (b - a) / 15, and numbers half way between two codes."""
    g = gen(4)
    lo = rand(g, 300, 1, dtype=dtype)
    step = (rand(g, 300, 1, dtype=dtype).abs() + 2.0 ** -9)
    x = (lo.double() + step.double() * torch.arange(32, device="cuda") / 2).to(dtype)
    x[:, 31] = (lo + 15 * step)[:, 0]
    rows = x.repeat(1, 2).view(1, 1, 300, 64)
    c = make(1, 64, 1, 300, dtype)
    b = c.batch(c.open())
    b.extend(300)
    b.write(0, rows, -rows)
    for part, t in ((0, rows), (1, -rows)):
        codes, least, s = pack64(t[0])
        assert torch.equal(codes_of(c.codes[0, part, 0]), codes)
        assert torch.equal(c.scales[0, part, 0].double(), torch.stack((least, s), -1))


# --------------------------------------------------------------------------------------------------------- attention
SHAPES = [(128, 8, 32, torch.bfloat16), (64, 4, 28, torch.float16), (128, 2, 2, torch.float16), (64, 1, 8, torch.bfloat16), (128, 1, 40, torch.bfloat16)]


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES)
@pytest.mark.parametrize("lengths,counts", [
    ([1], [1]), ([15, 16, 17], [1, 1, 1]), ([64, 65, 3, 700], [1, 1, 1, 1]), ([40, 40, 40], [3, 0, 40]), ([5000], [1]), ([2049, 130], [2, 5]),
    ([33, 300, 1000], [33, 18, 1]), ([700], [129]), ([1500, 257], [64, 200])])
def test_attend(dim, kv, heads, dtype, lengths, counts):
    g = gen(sum(lengths) + dim)
    c = make(kv, dim, len(lengths) + 1, max(lengths) + 3, dtype)
    seqs = c.open(len(lengths) + 1)[1:]
    b = fill(c, g, seqs, lengths)
    b.plan(counts)
    most = max(counts)
    q = rand(g, len(seqs), most, heads, dim, dtype=dtype, scale=1.5).permute(0, 2, 1, 3)
    for i, n in enumerate(counts):
        q[i, :, :most - n] = NAN  # not read
    out, lse = b.attend(0, q, return_lse=True)
    check(c, b, counts, q, out, lse)
    assert torch.equal(out, b.attend(0, q))
    out, lse = b.attend(0, q, scale=0.3, return_lse=True)
    check(c, b, counts, q, out, lse, scale=0.3)


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES)
@pytest.mark.parametrize("lengths,counts,weigh,decay", [
    ([1], [1], True, 0.0), ([15, 300, 64], [1, 1, 1], True, 1.0), ([40, 90, 700], [3, 0, 40], True, 0.5), ([3000], [1], 1, 0.0), ([600], [200], 33, 0.9),
    ([1100, 33], [130, 2], 4, 1.0)])
def test_weights(dim, kv, heads, dtype, lengths, counts, weigh, decay):
    g = gen(sum(lengths) + dim)
    c = make(kv, dim, len(lengths) + 1, max(lengths) + 3, dtype)
    seqs = c.open(len(lengths) + 1)[1:]
    b = fill(c, g, seqs, lengths)
    for s, n in zip(seqs, lengths):
        c.weights[0, s, :, :n] = torch.rand((kv, n), generator=g, device="cuda")
    if decay == 0:
        c.weights.fill_(NAN)  # not read
    before = c.weights.clone()
    b.plan(counts)
    most = max(counts)
    q = rand(g, len(seqs), heads, most, dim, dtype=dtype, scale=1.5)
    out, lse = b.attend(0, q, return_lse=True, weigh=weigh, decay=decay)
    check(c, b, counts, q, out, lse, weigh=most if weigh is True else weigh, before=before, decay=decay)
    after = c.weights.clone()
    for s, n, x in zip(seqs, lengths, counts):  # tokens behind the end, sequences without new tokens, other sequences: as they were
        if x:
            before[0, s, :, :n] = after[0, s, :, :n]
    assert torch.equal(before.nan_to_num(-5), after.nan_to_num(-5))
    c.weights.copy_(before)
    if decay == 0:
        b.attend(0, q, weigh=weigh, decay=decay)
        assert torch.equal(c.weights.nan_to_num(-5), after.nan_to_num(-5))  # the same bits again


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES[:4])
@pytest.mark.parametrize("lengths,counts,weigh", [([2600], [2600], True), ([1300, 2100, 5], [900, 1, 0], 700), ([9000], [40], True), ([257, 255], [130, 255], 256)])
def test_weights_of_long_prompts(dim, kv, heads, dtype, lengths, counts, weigh):
    """Prompts whose tiles are taken out of their codes beforehand, units that are cut and added up in parts, and units of one tile of keys."""
    g = gen(sum(lengths) + dim)
    c = make(kv, dim, len(lengths) + 1, max(lengths) + 3, dtype)
    seqs = c.open(len(lengths) + 1)[1:]
    b = fill(c, g, seqs, lengths)
    for s, n in zip(seqs, lengths):
        c.weights[0, s, :, :n] = torch.rand((kv, n), generator=g, device="cuda")
    before, most = c.weights.clone(), max(counts)
    b.plan(counts)
    q = rand(g, len(seqs), most, heads, dim, dtype=dtype, scale=1.5).permute(0, 2, 1, 3)
    out, lse = b.attend(0, q, return_lse=True, weigh=weigh, decay=0.75)
    check(c, b, counts, q, out, lse, weigh=most if weigh is True else weigh, before=before, decay=0.75)
    c.weights.copy_(before)
    out2, lse2 = b.attend(0, q, return_lse=True, weigh=weigh, decay=0.75)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES[:3])
@pytest.mark.parametrize("n", [4, 200, 420])
def test_tokens_that_are_no_numbers_are_none_only_where_they_are_seen(dim, kv, heads, dtype, n):
    g = gen(9)
    c = make(kv, dim, 1, 600, dtype)
    b = c.batch(c.open())
    b.extend(500)
    k, v = (rand(g, 1, kv, 500, dim, dtype=dtype) for _ in range(2))
    k[0, 0, 498, 5] = NAN       # of the third and of the newest token
    v[0, -1, 499, dim - 1] = INF
    b.write(0, k, v)
    b.plan(n)
    q = rand(g, 1, heads, n, dim, dtype=dtype)
    out, lse = b.attend(0, q, return_lse=True)
    group = heads // kv
    assert out[0, :group, n - 2:].isnan().all() and out[0, heads - group:, n - 1].isnan().any(-1).all()
    assert not out[0, :, :n - 2].isnan().any() and (kv == 1 or not out[0, heads - group:, :n - 1].isnan().any())
    c2 = make(kv, dim, 1, 600, dtype)
    b2 = c2.batch(c2.open())
    b2.extend(500)
    k[0, 0, 498, 5], v[0, -1, 499, dim - 1] = 0, 0
    b2.write(0, k, v)
    b2.plan(n)
    fine = b2.attend(0, q)
    assert torch.equal(out[0, :, :n - 2], fine[0, :, :n - 2])


def test_large_scores_and_a_scale_of_zero():
    g = gen(2)
    c = make(2, 128, 1, 300)
    b = fill(c, g, c.open(), [300], scale=30.0)
    for n in (1, 40):
        b.plan(n)
        q = rand(g, 1, 8, n, 128, scale=30.0)
        out, lse = b.attend(0, q, return_lse=True)
        check(c, b, [n], q, out, lse)
        out, lse = b.attend(0, q, scale=0.0, return_lse=True)
        check(c, b, [n], q, out, lse, scale=0.0)


def test_strides_and_layers_and_unaligned_rows():
    g = gen(3)
    c = make(4, 64, 3, 200, layers=3)
    seqs = c.open(3)[1:]
    b = c.batch(seqs)
    b.extend([100, 37])
    big = rand(g, 2, 100, 3, 4, 72)
    k, v = (big[:, :, i, :, :64].permute(0, 2, 1, 3) for i in (0, 1))
    odd = big[:, :, 2, :, 3:67].permute(0, 2, 1, 3)  # rows that are not 16-byte aligned
    b.write(2, k, odd)
    for i, (s, n) in enumerate(zip(seqs, (100, 37))):
        for part, t in ((0, k), (1, odd)):
            codes, least, step = pack64(t[i, :, 100 - n:])
            assert torch.equal(held(c, 2, s)[part], stand64(codes, least, step, torch.bfloat16))
    b.plan([5, 1])
    q = big[:, :5, 0, :, 2:66].permute(0, 2, 1, 3)
    out, lse = b.attend(2, q, return_lse=True)
    check(c, b, [5, 1], q, out, lse, layer=2)
    assert c.scales[:2].isnan().all()


def test_offsets_past_32_bits():
    g = gen(5)
    c = make(8, 128, 40, 131072)
    assert c.codes[0, 0].numel() * 4 > 1 << 31
    seqs = c.open(40)[39:]
    b = c.batch(seqs)
    b.extend(131072 - 40)
    b.extend(40)
    k, v = (rand(g, 1, 8, 40, 128) for _ in range(2))
    b.write(0, k, v)
    # the tokens before are all the same
    for t in (c.codes, c.scales):
        t[0, :, 39, :, :131072 - 40] = t[0, :, 39, :, -1:]
    for n in (1, 40):
        b.plan(n)
        q = rand(g, 1, 8, n, 128)
        out, lse = b.attend(0, q, return_lse=True, weigh=True, decay=0.0)
        check(c, b, [n], q, out, lse, weigh=n, before=c.weights, decay=0.0)
    c.evict(seqs, 300, 100, 100, into=[3])
    assert (c.places[0, 3, :, 200:300] == c.places[0, 39, :, -100:]).all()
    want = stay_of(c.weights[0, 39], 131072, 300, 100, 100)
    for part in (0, 1):
        for h in range(8):
            assert torch.equal(c.codes[0, part, 3, h, :300], c.codes[0, part, 39, h, want[h]])


# ---------------------------------------------------------------------------------------------------------- eviction
def stay_of(weights, n, budget, sink, recent):
    """Tokens that stay of each head, from the rule."""
    out = []
    for w in weights[:, :n].cpu().tolist():
        mid = sorted(range(sink, n - recent), key=lambda j: (-(INF if w[j] != w[j] else w[j]), not w[j] != w[j], j))[:budget - sink - recent]
        out.append(torch.tensor(list(range(sink)) + sorted(mid) + list(range(n - recent, n)) if n > budget else list(range(n)), dtype=torch.long))
    return out


def random_cache(g, kv, dim, slots, most, dtype, layers, ties):
    c = make(kv, dim, slots, most, dtype, layers)
    c.codes.copy_(torch.randint(-1 << 31, 1 << 31, c.codes.shape, generator=g, device="cuda"))
    c.scales.copy_(rand(g, *c.scales.shape, dtype=dtype))
    c.places.copy_(torch.randint(0, 1 << 30, c.places.shape, generator=g, device="cuda"))
    w = torch.randn(c.weights.shape, generator=g, device="cuda").exp()
    if ties == "few values":
        w = torch.randint(0, 3, w.shape, generator=g, device="cuda").float()
    elif ties == "equal":
        w = torch.full_like(w, 0.25)
    elif ties == "odd":
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.1] = NAN
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.1] = INF
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.1] = -1.0
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.1] = -0.0
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.1] = 0.0
    c.weights.copy_(w)
    return c


@pytest.mark.parametrize("dim,kv,dtype,layers", [(128, 2, torch.bfloat16, 1), (64, 3, torch.float16, 2), (128, 8, torch.float16, 11), (64, 8, torch.bfloat16, 40)])
@pytest.mark.parametrize("lengths,budget,sink,recent", [
    ([10, 7, 3], 7, 1, 2), ([900, 300, 299], 300, 4, 100), ([2000], 1, 0, 0), ([700, 650], 640, 0, 0), ([513], 0, 0, 0), ([4097, 1200], 1000, 1000, 0),
    ([1500], 700, 0, 700), ([1500, 20], 700, 350, 350), ([5000, 2500], 2400, 128, 512), ([129], 128, 3, 120)])
@pytest.mark.parametrize("into,ties", [(False, "none"), (True, "none"), (False, "few values"), (True, "equal"), (False, "odd")])
def test_evict(dim, kv, dtype, layers, lengths, budget, sink, recent, into, ties):
    if layers > 2 and sum(lengths) > 6000:
        lengths = lengths[-1:]
    g, m = gen(budget + sum(lengths)), len(lengths)
    c = random_cache(g, kv, dim, 2 * m + 1, max(lengths) + 5, dtype, layers, ties)
    seqs = c.open(2 * m + 1)
    dst, seqs = seqs[:m], seqs[m + 1:]
    c.batch(seqs).extend(lengths)
    c.batch(dst[:1]).extend(2)
    was = [t.clone() for t in (c.codes, c.scales, c.weights, c.places)]
    c.evict(seqs, budget, sink, recent, into=dst if into else None)
    for layer in range(layers):
        for i, (s, n) in enumerate(zip(seqs, lengths)):
            d = dst[i] if into else s
            assert c.length(d) == min(n, budget) and c.position(d) == n and c.length(s) == (n if into else min(n, budget))
            if n <= budget and not into:
                continue
            for h, rows in enumerate(stay_of(was[2][layer, s], n, budget, sink, recent) if layer in (0, layers - 1) else []):
                rows = rows.cuda()
                x = len(rows)
                for t, old in zip((c.codes, c.scales), was):
                    assert torch.equal(t[layer, :, d, h, :x], old[layer, :, s, h, rows])
                for t, old in zip((c.weights, c.places), was[2:]):
                    assert torch.equal(t[layer, d, h, :x].nan_to_num(-9), old[layer, s, h, rows].nan_to_num(-9))
    for t, old, axis in zip((c.codes, c.scales, c.weights, c.places), was, (2, 2, 1, 1)):  # other sequences, and what is behind the sources' ends
        t, old = t.movedim(axis, 0), old.movedim(axis, 0)
        for s in range(2 * m + 1):
            behind = 0 if s not in (dst if into else seqs) else min(lengths[(dst if into else seqs).index(s)], budget) if into else max(lengths)
            a, z = (x[s].movedim(x[s].shape.index(c.max_tokens), 0)[behind:] for x in (t, old))
            assert torch.equal(a.double().nan_to_num(-9), z.double().nan_to_num(-9))


# ------------------------------------------------------------------------------------------------- a run of them together
@pytest.mark.parametrize("n,kv,budget,sink,recent", [(20011, 600, 9001, 3, 100), (9999, 601, 9990, 0, 0), (90001, 2, 45000, 0, 500), (30, 1, 29, 0, 0)])
@pytest.mark.parametrize("values", ["normal", "lowest"])
def test_evict_of_more_weights_than_a_block_has_room_for(n, kv, budget, sink, recent, values):
    g = gen(19)
    c = make(kv, 64, 1, n)
    s = c.open()
    c.batch(s).extend(n)
    w = torch.randn((kv, n), generator=g, device="cuda").exp()
    if values == "lowest":  # one half of them less than any other, and some the least number
        w = torch.where(w < 1, -INF, torch.where(w < 1.5, -3.4028234663852886e38, w.round()))
    c.weights[0, 0].copy_(w)
    c.places[0, 0].copy_(torch.arange(n, dtype=torch.int32, device="cuda").expand(kv, n))
    c.evict(s, budget, sink, recent)
    k = budget - sink - recent
    order = torch.sort(w[:, sink:n - recent], dim=1, descending=True, stable=True).indices[:, :k]  # (of equal ones the earlier)
    want = torch.cat((torch.arange(sink, device="cuda").expand(kv, sink), order.sort(1).values + sink,
                      torch.arange(n - recent, n, device="cuda").expand(kv, recent)), 1)
    assert c.length(s[0]) == budget and torch.equal(c.places[0, 0, :, :budget].long(), want)
    assert torch.equal(c.weights[0, 0, :, :budget], w.gather(1, want))


@pytest.mark.parametrize("dim,kv,heads,dtype", SHAPES[:3])
def test_a_generation_with_evictions(dim, kv, heads, dtype):
    """A prompt, decode steps, drafts that are taken back, evictions in between: every output and weight against the formulas over what the
    cache holds, and what it holds against packed rows that are moved by the rule."""
    from infllm_b200.attention import RotaryEmbeddingESM

    g, rng = gen(11), random.Random(11)
    layers, n = 2, 3
    c = make(kv, dim, n, 260, dtype, layers)
    rope = RotaryEmbeddingESM(dim, 1e4, 1.0)
    b = c.batch(c.open(n))
    mine = [[dict(w=torch.zeros((kv, 0), dtype=torch.float64, device="cuda"), p=torch.zeros((kv, 0), dtype=torch.int32, device="cuda")) for _ in range(n)]
            for _ in range(layers)]
    for step in range(24):
        counts = [150, 90, 121] if step == 0 else [rng.choice([1, 1, 1, 0, 4]) for _ in range(n)]
        if max(counts) == 0:
            counts[0] = 1
        at = [c.position(s) for s in b.seqs]
        b.extend(counts)
        most = max(counts)
        for layer in range(layers):
            q, k, v = (rand(g, n, h, most, dim, dtype=dtype, scale=1.3) for h in (heads, kv, kv))
            q = b.write(layer, k, v, q, rope)
            before = c.weights.clone()
            out, lse = b.attend(layer, q, return_lse=True, weigh=True, decay=0.9)
            check(c, b, counts, q, out, lse, layer=layer, weigh=most, before=before, decay=0.9)
            for i, (s, x) in enumerate(zip(b.seqs, counts)):
                new = torch.arange(at[i], at[i] + x, device="cuda", dtype=torch.int32).expand(kv, -1)
                mine[layer][i]["p"] = torch.cat((mine[layer][i]["p"], new), 1)
                assert torch.equal(c.places[layer, s, :, :c.length(s)], mine[layer][i]["p"])
        if step % 5 == 3:
            b.retract([min(x, 2) for x in counts])
            for layer in range(layers):
                for i, x in enumerate(counts):
                    p = mine[layer][i]["p"]
                    mine[layer][i]["p"] = p[:, :p.size(1) - min(x, 2)]
        if step % 3 == 2 or step == 0:
            w, lens = c.weights.clone(), [c.length(s) for s in b.seqs]
            c.evict(b.seqs, 80, 4, 20)
            for layer in range(layers):
                for i, s in enumerate(b.seqs):
                    rows = stay_of(w[layer, s], lens[i], 80, 4, 20)
                    mine[layer][i]["p"] = torch.stack([mine[layer][i]["p"][h, r.cuda()] for h, r in enumerate(rows)])
                    assert torch.equal(c.places[layer, s, :, :c.length(s)], mine[layer][i]["p"])


def test_the_attention_type():
    from infllm_b200.attention import ATTN_FORWRAD, PackedLayer, RotaryEmbeddingESM

    g, rope = gen(12), RotaryEmbeddingESM(64, 1e4, 1.0)
    c = make(2, 64, 2, 50)
    b = c.batch(c.open(2))
    wq, wk, wv, wo = (rand(g, o, i, scale=i ** -0.5) for o, i in ((256, 96), (128, 96), (128, 96), (96, 256)))
    forward = ATTN_FORWRAD["packed"]()
    for n in (20, 1):
        x = rand(g, 2, n, 96)
        b.extend(n)
        o, past = forward(None, x, x, rope, True, PackedLayer(b, 0, weigh=True), lambda t: t @ wq.T, lambda t: t @ wk.T, lambda t: t @ wv.T, lambda t: t @ wo.T, 64, 4, 2)
        assert o.shape == (2, n, 96) and isinstance(past, PackedLayer)
        other = make(2, 64, 2, 50)
    q = rope._rotate((x @ wq.T).view(2, 1, 4, 64).permute(0, 2, 1, 3), 20, 0)
    want = torch.stack([formula(q[i], *held(c, 0, i), 1, 0.125)[0] for i in (0, 1)]).permute(0, 2, 1, 3).reshape(2, 1, 256) @ wo.double().T
    assert (o.double() - want).abs().max() <= 2.0 ** -6 * want.abs().max()  # (two roundings of 2^-8, 256 terms)
    got = c.weights[0, :, :, :21].sum(-1)
    assert (got - 2 * 21).abs().max() < 1e-3  # every query's probabilities add up to one
    with pytest.raises(TypeError):
        forward(None, x, x, rope, True, None, None, None, None, None, 64, 4, 2)


# ------------------------------------------------------------------------------------- streams, graphs, several calls
def test_calls_of_two_batches_on_two_streams():
    g = gen(13)
    c = make(8, 128, 8, 3000)
    seqs = c.open(8)
    b = fill(c, g, seqs, [3000] * 8)
    parts = [c.batch(seqs[:4]), c.batch(seqs[4:])]
    qs = [rand(g, 4, 32, 1, 128) for _ in parts]
    for p in parts:
        p.plan(1)
    want = [p.attend(0, q, weigh=True, decay=0.0) for p, q in zip(parts, qs)]
    w = c.weights.clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    got = [[], []]
    for _ in range(20):
        for i, (p, q, s) in enumerate(zip(parts, qs, streams)):
            with torch.cuda.stream(s):
                got[i].append(p.attend(0, q, weigh=True, decay=0.0))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
    assert torch.equal(c.weights, w)


@pytest.mark.parametrize("n", [1, 70])
def test_a_captured_step_is_replayed(n):
    from infllm_b200.attention import RotaryEmbeddingESM

    g, rope = gen(14), RotaryEmbeddingESM(128, 1e4, 1.0)
    c = make(2, 128, 3, 900)
    b = c.batch(c.open(2))
    b.extend([700, 300])
    b.write(0, *(rand(g, 2, 2, 700, 128) for _ in range(2)))
    b.extend(n)
    q, k, v = (rand(g, 2, h, n, 128) for h in (8, 2, 2))

    def step():
        return b.attend(0, b.write(0, k, v, q, rope), weigh=True, decay=0.0, return_lse=True), b.values(0)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (out, lse), (hk, hv) = step()
    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    graph.replay()
    got = [x.clone() for x in (out, lse, hk, hv, c.weights, c.codes)]
    (out2, lse2), (hk2, hv2) = step()
    for x, y in zip(got, (out2, lse2, hk2, hv2, c.weights, c.codes)):
        assert torch.equal(x.double().nan_to_num(-3), y.double().nan_to_num(-3))


def test_tables_that_a_captured_write_reads():
    """They are not made inside a capture, and stay when longer ones have taken their place."""
    from infllm_b200.attention import RotaryEmbeddingESM

    g, rope = gen(18), RotaryEmbeddingESM(128, 1e4, 1.0)
    c = make(1, 128, 1, 200)
    b = c.batch(c.open())
    b.extend(20)
    k, v = (rand(g, 1, 1, 20, 128) for _ in range(2))
    with pytest.raises(RuntimeError, match="inside a capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.write(0, k, v, rope=rope)
    assert c.scales.isnan().all() and rope._cos is None
    b.write(0, k, v, rope=rope)
    want = c.codes.clone(), c.scales.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.write(0, k, v, rope=rope)
        b.write(0, k, v, rope=rope)
    assert len(c._captured) == 1
    shape = rope._cos.shape
    rope._tables(5000, c.device)
    over = [torch.full(shape, NAN, device="cuda") for _ in range(20)]  # (memory that was given back would be theirs)
    c.codes.fill_(-1)
    c.scales.fill_(NAN)
    graph.replay()
    assert torch.equal(c.codes[:, :, :, :, :20], want[0][:, :, :, :, :20]) and torch.equal(c.scales[:, :, :, :, :20], want[1][:, :, :, :, :20])
    assert all(x.isnan().all() for x in over)


def test_many_sequences_in_one_call():
    g = gen(15)
    c = make(1, 64, 300, 40, layers=1)
    seqs = c.open(300)
    lengths = [1 + i % 40 for i in range(300)]
    b = fill(c, g, seqs, lengths)
    counts = [min(1 + i % 3, n) for i, n in enumerate(lengths)]
    b.plan(counts)
    q = rand(g, 300, 4, 3, 64)
    before = c.weights.clone()
    out, lse = b.attend(0, q, return_lse=True, weigh=True, decay=0.0)
    check(c, b, counts, q, out, lse, weigh=3, before=before, decay=0.0)
    b.plan(lengths)
    k = b.values(0)[0]
    for i in (0, 39, 127, 128, 299):
        assert torch.equal(k[i, :, 40 - lengths[i]:].double(), held(c, 0, i)[0])
    w = c.weights.clone()
    c.evict(seqs, 11, 1, 3)
    for i in (38, 127, 128, 271, 299):
        rows = stay_of(w[0, i], lengths[i], 11, 1, 3)[0].cuda()
        assert torch.equal(c.weights[0, i, 0, :len(rows)], w[0, i, 0, rows])


def test_a_step_without_tokens():
    c = make(2, 64, 2, 50)
    b = c.batch(c.open(2))
    none = torch.empty((2, 2, 0, 64), dtype=torch.bfloat16, device="cuda")
    for step in (b.extend, b.plan):
        step(0)
        assert b.write(0, none, none) is None
        out, lse = b.attend(0, torch.empty((2, 8, 0, 64), dtype=torch.bfloat16, device="cuda"), return_lse=True, weigh=True)
        assert out.shape == (2, 8, 0, 64) and lse.shape == (2, 8, 0)
        assert b.values(0)[0].shape == (2, 2, 0, 64) and b.values()[1].shape == (1, 2, 2, 0, 64)
    c.evict(b.seqs, 0)
    c.evict([], 5)
    empty = c.batch([])
    empty.extend(3)
    assert c.scales.isnan().all()


def test_refusals_of_tensors():
    c = make(2, 64, 2, 50)
    b = c.batch(c.open())
    b.extend(3)
    t = torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16, device="cuda")
    for call, error in ((lambda: b.write(0, t[:, :1], t), ValueError), (lambda: b.write(0, t, t.half()), TypeError), (lambda: b.write(0, t.cpu(), t), RuntimeError),
                        (lambda: b.attend(0, t[:, :, :2]), ValueError), (lambda: b.attend(0, t.float()), TypeError), (lambda: b.write(0, t, t, rope=3), ValueError),
                        (lambda: b.attend(1, t), ValueError), (lambda: b.attend(1 << 32, t), ValueError), (lambda: b.attend(0, t, weigh=-1), ValueError), (lambda: b.attend(0, t, weigh=-1 << 40), ValueError), (lambda: b.attend(0, t[:, :0]), RuntimeError), (lambda: b.attend(0, t, scale=-1.0), RuntimeError),
                        (lambda: b.values(1), ValueError), (lambda: b.write(-1, t, t), ValueError), (lambda: b.attend(0, t, scale=1e300), RuntimeError), (lambda: b.attend(0, t, weigh=True, decay=-0.5), RuntimeError)):
        with pytest.raises(error):
            call()
    assert c.scales.isnan().all()
