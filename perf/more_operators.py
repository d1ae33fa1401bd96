"""Workloads of the packed key/value cache: keys and values in 4 bits, attention over them, and eviction by attention weight.

The cache holds, of each 32 neighbouring numbers x of a key (rotated to its position) or of a value, in their own 16-bit type T,
the least m = min x and a step s = T((max x - m) / 15), and of each number its code c, the nearest of 0 .. 15 to (x - m) / s
(ties to even; 0 where s is 0).  It stands for T(m + s c).  A word of 32 bits has eight codes: number 2i of the eight at bit 4i,
number 2i + 1 at bit 16 + 4i.  Of every token and KV head it also has the token's position and a weight in 32 bits.

Kinds of work (the "kind" of a case):

attend    attention of the newest `new` tokens of `batch` sequences: one token each is a decode step, more are drafts, questions
          put to a long document, or (batch 1) a chunk of a prompt.  With "ragged" the sequences have different counts of new tokens,
          which stand at the end of the tensors.  With "weigh" the weights of the tokens become what the queries' attention gave
          them, summed over the new tokens and the query heads of a KV head: what an eviction goes by
write     one layer's keys and values of `new` tokens of every sequence into the cache, keys and queries rotated to the tokens'
          positions, and what the cache holds of them read back; the tokens are given back at the end of the pass
evict     of every layer and KV head of `batch` sequences `budget` tokens go to another sequence, in their order: the first `sink`,
          the newest `recent`, and of the others those of the largest weights (of equal ones the earlier); the new sequences are
          read back

Where `own` is false, a pass is elementary torch operations in 32 bits on the same codes.

Sizes are those of the repository's benchmark configurations (32 query heads over 8 or 32 KV heads of 128 dimensions, windows
of 4096 tokens, sinks of 128, chunks of 8192 tokens, contexts up to 131072 tokens) and odd ones of the same kind.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BASE = 1e6  # of the rotary embedding
GROUP = 32  # numbers that share a least one and a step


def _attend(batch, length, new=1, heads=32, kv_heads=8, dim=128, dtype="bf16", weigh=False, ragged=False, **more):
    return dict(kind="attend", batch=batch, length=length, new=new, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                weigh=weigh, ragged=ragged, **more)


def _write(batch, past, new, heads=32, kv_heads=8, dim=128, dtype="bf16", **more):
    return dict(kind="write", batch=batch, past=past, new=new, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, **more)


def _evict(batch, length, budget, sink, recent, layers, kv_heads=8, dim=128, dtype="bf16", **more):
    return dict(kind="evict", batch=batch, length=length, budget=budget, sink=sink, recent=recent, layers=layers,
                kv_heads=kv_heads, dim=dim, dtype=dtype, **more)


def listed():
    return [
        # a decode step of four short sequences: the smallest call of a generation loop
        _attend(4, 1100, name="tokens_4_on_1k"),
        # a decode step of a full server: 32 sequences of up to 32K tokens
        _attend(32, 32768, name="tokens_32_on_32k"),
        # the next token of one long stream, at the longest context of the benchmark configurations
        _attend(1, 131072, name="token_1_on_128k"),
        # 28 query heads over 4 KV heads of 64 dimensions, fp16, lengths of no tile
        _attend(13, 5703, heads=28, kv_heads=4, dim=64, dtype="fp16", name="tokens_13_odd_fp16"),
        # eight questions of up to 48 tokens, each to a document of its own, read at once
        _attend(8, 16384, new=48, ragged=True, name="questions_8_on_16k"),
        # a chunk of a prompt: 2048 tokens behind 28000
        _attend(1, 30048, new=2048, name="chunk_2048_on_28k"),
        # a decode step whose weights decide what leaves a window-sized cache
        _attend(16, 8192, weigh=True, name="weigh_16_on_8k"),
        # a prompt of a window's length is read, and all its queries are counted
        _attend(1, 4096, new=4096, weigh=True, name="weigh_prompt_4k"),
        # a decode step's token of each of 64 sequences
        _write(64, 5000, 1, name="write_64_tokens"),
        # the chunk in which prompts are read, fp16, as many KV heads as query heads
        _write(1, 8192, 8192, kv_heads=32, dtype="fp16", name="write_chunk_8192"),
        # during generation: eight sequences have grown past a window and are cut back to half of it, two layers
        _evict(8, 4224, 2048, 128, 512, 2, name="evict_8_of_4k"),
        # a long prompt has been read: a sixteenth of it stays, in four layers
        _evict(1, 65536, 4096, 128, 1024, 4, name="evict_prompt_64k"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "write", "evict"])
    dim = rng.choice([64, 128, 128])
    kv, group = rng.choice([(1, 8), (2, 2), (4, 7), (8, 1), (8, 4), (8, 4), (32, 1)])
    more = dict(kv_heads=kv, dim=dim, dtype=rng.choice(["bf16", "fp16"]))
    if kind == "attend":
        new = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 2, 2048)])
        c = _attend(_log(rng, 1, 64), _log(rng, 20, 131072), new, heads=kv * group, weigh=rng.random() < 0.4,
                    ragged=rng.random() < 0.3, **more)
        c["length"] = max(c["length"], new)
        # numbers of the cache, and scores, in 32 bits
        while c["batch"] * c["length"] * kv * dim > 1 << 30 or c["batch"] * kv * group * new * c["length"] > 19e8:
            if c["batch"] > 1:
                c["batch"] = (c["batch"] + 1) // 2
            else:
                c["length"] = max(new, c["length"] * 2 // 3)
        return c
    if kind == "write":
        new = rng.choice([1, _log(rng, 1, 8192)])
        return _write(max(1, min(_log(rng, 1, 128), 16384 // new)), _log(rng, 1, 20000), new, heads=kv * group, **more)
    length, batch, layers = _log(rng, 300, 65536), _log(rng, 1, 16), rng.randint(1, 8)
    budget = max(20, int(rng.uniform(0.02, 0.5) * length))
    while layers * batch * kv * dim * (length + 4 * budget) > 1 << 28:
        if layers > 1:
            layers = (layers + 1) // 2
        elif batch > 1:
            batch = (batch + 1) // 2
        else:
            length, budget = (length + 1) // 2, (budget + 1) // 2
    sink = rng.choice([0, min(4, budget), min(128, budget // 2)])
    return _evict(batch, length, budget, sink, rng.choice([0, (budget - sink) // 2, budget - sink]), layers, **more)


def _lens(case):
    """Tokens of each sequence, the newest included: from half of `length` up."""
    n = case["length"]
    if case["batch"] == 1:
        return [n]
    r = random.Random("%d %d" % (case["batch"], n))
    return [r.randint(max(case.get("new", 1), (n + 1) // 2), n) for _ in range(case["batch"])]


def _counts(case):
    """New tokens of each sequence."""
    if not case["ragged"]:
        return [case["new"]] * case["batch"]
    r = random.Random("%d %d" % (case["new"], case["batch"]))
    return [case["new"]] + [r.randint(1, case["new"]) for _ in range(case["batch"] - 1)]


def _pasts(case):
    r = random.Random("%(batch)d %(past)d" % case)
    return [r.randint((case["past"] + 1) // 2, case["past"]) for _ in range(case["batch"])]


def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _shifts():
    return torch.tensor([4 * (i // 2) + 16 * (i % 2) for i in range(8)], dtype=torch.int32, device="cuda")


def _packed(x):
    """Codes (.., dim / 8) int32 and scales (.., dim / 32, 2) of numbers (.., dim)."""
    t = x.float().unflatten(-1, (-1, GROUP))
    least = t.amin(dim=-1, keepdim=True)
    step = ((t.amax(dim=-1, keepdim=True) - least).double() / 15).float().to(x.dtype)
    c = torch.round((t - least) / step.float())
    c = torch.where(step == 0, torch.zeros_like(c), c).clamp(0, 15).to(torch.int32)
    words = (c.flatten(-2).unflatten(-1, (-1, 8)) << _shifts()).sum(dim=-1, dtype=torch.int32)
    return words, torch.cat((least.to(x.dtype), step), dim=-1)


def _values32(words, scales):
    """What codes and scales stand for, in 32 bits."""
    c = ((words.unsqueeze(-1) >> _shifts()) & 15).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    return (scales[..., :1].float() + scales[..., 1:].float() * c).to(scales.dtype).float().flatten(-2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, kv, dim = case["kind"], _DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    b, h, n, layers = case["batch"], case.get("heads"), case.get("new"), case.get("layers", 1)
    held = [p + n for p in _pasts(case)] if kind == "write" else _lens(case)  # tokens at the largest
    slots, most = 2 * b if kind == "evict" else b + 1, max(held)
    # the whole cache, so that what lies behind a sequence's end is what another one left there
    codes = torch.randint(-(1 << 31), 1 << 31, (layers, 2, slots, kv, most, dim // 8), generator=g, device="cuda", dtype=torch.int32)
    scales = torch.empty((layers, 2, slots, kv, most, dim // GROUP, 2), device="cuda", dtype=dtype)
    scales[..., 0] = -2 - _randn(g, dtype, *scales.shape[:-1]).abs()
    scales[..., 1] = (0.2 + 0.1 * _randn(g, torch.float32, *scales.shape[:-1]).abs()).to(dtype)
    # a few tokens have had most of the attention, some none
    weights = torch.exp(2 * _randn(g, torch.float32, layers, slots, kv, most))
    weights *= (torch.rand(weights.shape, generator=g, device="cuda") > 0.1) * (1.0 if kind == "evict" else 1e-4)
    # positions with gaps, where tokens have left before
    places = torch.cumsum(1 + 9 * (torch.rand(weights.shape, generator=g, device="cuda") > 0.9), dim=-1, dtype=torch.int32)
    state = {"case": case}
    if kind == "attend":
        # a direction that all queries of a KV head lean to, and with them the first keys and some others
        lean = _randn(g, torch.float32, kv, 1, dim)
        lean /= lean.norm(dim=-1, keepdim=True)
        for i, length in enumerate(held):
            k, v = _randn(g, torch.float32, 2, kv, length, dim)
            k[:, :4] += 6 * lean
            k[:, 50::97] += 4 * lean
            for part, x in ((0, k), (1, v)):
                codes[0, part, i, :, :length], scales[0, part, i, :, :length] = _packed(x.to(dtype))
        q = _randn(g, torch.float32, b, n, h, dim) + 3 * lean[:, 0].repeat_interleave(h // kv, 0)
        state["q"] = q.to(dtype).permute(0, 2, 1, 3)  # (batch, heads, tokens, dim), as a projection's view
    if kind == "write":
        state["q"] = _randn(g, dtype, b, n, h, dim).permute(0, 2, 1, 3)
        state["k"] = _randn(g, dtype, b, n, kv, dim).permute(0, 2, 1, 3)
        state["v"] = _randn(g, dtype, b, n, kv, dim).permute(0, 2, 1, 3)
    if own:
        from infllm_b200.attention import PackedCache, RotaryEmbeddingESM

        cache = state["cache"] = PackedCache(layers, kv, dim, slots, most, dtype=dtype)
        state["seqs"] = seqs = cache.open(b)
        batch = state["batch"] = cache.batch(seqs)
        batch.extend(_pasts(case) if kind == "write" else held)
        for mine, made in ((cache.codes, codes), (cache.scales, scales), (cache.weights, weights), (cache.places, places)):
            mine.copy_(made)
        if kind == "attend":
            batch.plan(_counts(case) if case["ragged"] else n)
        elif kind == "write":
            state["rope"] = RotaryEmbeddingESM(dim, BASE, 1.0)
        else:
            state["into"] = cache.open(b)
            state["cut"] = cache.batch(state["into"])
        return state
    state |= {"codes": codes, "scales": scales, "weights": weights, "places": places}
    if kind == "write":
        freq = 1.0 / BASE ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim)
        angle = (torch.arange(most, dtype=torch.float32)[:, None] * freq).cuda()
        state["cos"], state["sin"] = angle.cos(), angle.sin()
        state["past"] = torch.tensor(_pasts(case), device="cuda")
    else:
        state["lens"] = torch.tensor(held, device="cuda")
    if kind == "attend":
        state["counts"] = torch.tensor(_counts(case), device="cuda")
    return state


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_attend(s):
    """out = softmax(q k^T / sqrt(dim)) v over the keys up to a query's own place; the weights of the keys are the sums of its columns."""
    case, q, lens = s["case"], s["q"], s["lens"]
    b, h, n, dim = q.shape
    kv, most = case["kv_heads"], s["codes"].shape[4]
    k = _values32(s["codes"][0, 0, :b], s["scales"][0, 0, :b])
    scores = torch.matmul(q.float().reshape(b, kv, h // kv * n, dim), k.transpose(-1, -2)).div_(math.sqrt(dim))
    del k
    at = torch.arange(n, device="cuda")
    place = lens[:, None] - n + at  # (b, n)
    there = at >= n - s["counts"][:, None]
    key = torch.arange(most, device="cuda")
    seen = (key <= place[:, :, None]) & there[:, :, None]  # (b, n, keys)
    scores = scores.view(b, h, n, most).masked_fill_(~seen[:, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total)).view(b, kv, h // kv * n, most)
    # (what lies behind a sequence's end is no number that counts)
    v = _values32(s["codes"][0, 1, :b], s["scales"][0, 1, :b]).masked_fill_((key >= lens[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(p, v).view(b, h, n, dim).to(q.dtype)
    if not case["weigh"]:
        return {"out": out}
    s["weights"][0, :b] = torch.where((key < lens[:, None])[:, None], p.sum(dim=2), s["weights"][0, :b])
    return {"out": out, "weights": s["weights"]}


def _rotate32(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)


def _plain_write(s):
    b, kv, n = s["k"].shape[:3]
    place = s["past"][:, None] + torch.arange(n, device="cuda")  # (b, n)
    cos, sin = s["cos"][place][:, None], s["sin"][place][:, None]
    seq, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(kv, device="cuda")[:, None]
    at = place[:, None]
    for part, x in ((0, _rotate32(s["k"], cos, sin)), (1, s["v"])):
        s["codes"][0, part, seq, head, at], s["scales"][0, part, seq, head, at] = _packed(x)
    s["weights"][0, seq, head, at] = 0.0
    s["places"][0, seq, head, at] = at.int()
    k, v = (_values32(s["codes"][0, i, seq, head, at], s["scales"][0, i, seq, head, at]).to(s["k"].dtype) for i in (0, 1))
    return {"q": _rotate32(s["q"], cos, sin), "k": k, "v": v, "weights": s["weights"], "places": s["places"]}


def _plain_evict(s):
    case = s["case"]
    b, budget = case["batch"], case["budget"]
    w, lens = s["weights"][:, :b], s["lens"][:, None, None]
    key = torch.arange(w.shape[-1], device="cuda")
    rank = torch.where((key < case["sink"]) | (key >= lens - case["recent"]), float("inf"), w)
    rank = torch.where(key >= lens, float("-inf"), rank)
    stay = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    for t in (s["weights"], s["places"]):
        t[:, b:, :, :budget] = torch.gather(t[:, :b], -1, stay)
    wide = stay[:, None, ..., None]
    for t in (s["codes"], s["scales"].flatten(-2)):
        t[:, :, b:, :, :budget] = torch.gather(t[:, :, :b], -2, wide.expand(-1, 2, -1, -1, -1, t.shape[-1]))
    k, v = (_values32(s["codes"][:, i, b:, :, :budget], s["scales"][:, i, b:, :, :budget]).to(s["scales"].dtype) for i in (0, 1))
    return {"k": k, "v": v, "weights": s["weights"], "places": s["places"]}


# ------------------------------------------------------------------------------------------- one pass through an operator
def run(s):
    case = s["case"]
    if not own:
        return {"attend": _plain_attend, "write": _plain_write, "evict": _plain_evict}[case["kind"]](s)
    cache, batch = s["cache"], s["batch"]
    if case["kind"] == "attend":
        if not case["weigh"]:
            return {"out": batch.attend(0, s["q"])}
        return {"out": batch.attend(0, s["q"], weigh=True, decay=0.0), "weights": cache.weights}
    if case["kind"] == "write":
        batch.extend(case["new"])
        q = batch.write(0, s["k"], s["v"], s["q"], s["rope"])
        k, v = batch.values(0)
        batch.retract(case["new"])
        return {"q": q, "k": k, "v": v, "weights": cache.weights, "places": cache.places}
    cache.evict(s["seqs"], case["budget"], case["sink"], case["recent"], into=s["into"])
    cut = s["cut"]
    cut.plan(case["budget"])
    k, v = cut.values()
    return {"k": k, "v": v, "weights": cache.weights, "places": cache.places}


def work(case):
    kv, dim, b = case["kv_heads"], case["dim"], case["batch"]
    row = 2 * (dim // 2 + dim // GROUP * 4)  # bytes of a token's codes and scales, of one KV head: key and value
    if case["kind"] == "attend":
        h, lens, counts = case["heads"], _lens(case), _counts(case)
        pairs = sum(c * n - c * (c - 1) / 2 for c, n in zip(counts, lens))
        rows = sum(counts) * h * dim * 2 + b * case["new"] * h * dim * 2
        return {"bytes": sum(lens) * kv * (row + 4 * case["weigh"]) + rows, "flops": 4.0 * h * dim * pairs}
    if case["kind"] == "write":
        tokens, h = b * case["new"], case["heads"]
        held = kv * (row + 8)
        return {"bytes": tokens * (2 * h * dim * 2 + 2 * kv * dim * 2 + held + kv * row + 2 * kv * dim * 2),
                "flops": tokens * dim * (3.0 * (h + kv) + 6.0 * kv)}
    kept = b * case["budget"] * kv * case["layers"]
    return {"bytes": 4 * sum(_lens(case)) * kv * case["layers"] + kept * (2 * (row + 8) + row + 2 * dim * 2), "flops": 2.0 * kept * 2 * dim}


# --------------------------------------------------------------------------------------------- the definitions in 64 bits
def _numbers(words, scales):
    """What codes and scales stand for, eight codes of a word one by one."""
    out = torch.empty((*words.shape, 8), dtype=torch.float64, device=words.device)
    per = scales.repeat_interleave(GROUP // 8, dim=-2).double()  # a word's least number and step
    for i in range(8):
        c = (words >> (4 * (i // 2) + 16 * (i % 2))).bitwise_and(15).double()
        out[..., i] = (per[..., 0] + per[..., 1] * c).to(scales.dtype).double()
    return out.flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    kind, kv, dim = case["kind"], case["kv_heads"], case["dim"]
    if kind == "attend":
        q, n, group = s["q"], case["new"], case["heads"] // kv
        out, weights = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), s["weights"].double()
        for i, (length, count) in enumerate(zip(_lens(case), _counts(case))):
            hidden = torch.ones((count, length), dtype=torch.bool, device="cuda").triu(length - count + 1)
            for j in range(kv):
                k, v = (_numbers(s["codes"][0, part, i, j, :length], s["scales"][0, part, i, j, :length]) for part in (0, 1))
                x = torch.einsum("gnd,kd->gnk", q[i, j * group:(j + 1) * group, n - count:].double(), k) / math.sqrt(dim)
                p = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1)
                out[i, j * group:(j + 1) * group, n - count:] = p @ v
                if case["weigh"]:
                    weights[0, i, j, :length] = p.sum(dim=(0, 1))
        return {"out": out, "weights": weights} if case["weigh"] else {"out": out}
    if kind == "write":
        half, dtype = dim // 2, s["k"].dtype
        # (angles are products in 32 bits: so the rotary embedding defines them)
        freq = (1.0 / BASE ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim)).cuda()
        got = {x: torch.empty(s[x].shape, dtype=torch.float64, device="cuda") for x in "qkv"}
        weights = s["weights"].double()
        for i, past in enumerate(_pasts(case)):
            place = torch.arange(past, past + case["new"], device="cuda")
            wave = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (place[:, None].float() * freq).double())

            def turn(x):
                z = torch.complex(x[..., :half].double(), x[..., half:].double()) * wave
                return torch.cat((z.real, z.imag), dim=-1)

            got["q"][i] = turn(s["q"][i])
            weights[0, i, :, past:past + case["new"]] = 0
            for name, x in (("k", turn(s["k"][i]).to(dtype).double()), ("v", s["v"][i].double())):
                for at in range(0, dim, GROUP):
                    y = x[..., at:at + GROUP]
                    lo, hi = y.min(dim=-1, keepdim=True).values, y.max(dim=-1, keepdim=True).values
                    step = ((hi - lo) / 15).to(dtype).double()
                    code = torch.round((y - lo) / step.clamp(min=1e-300)).clamp(max=15)
                    got[name][i, ..., at:at + GROUP] = (lo + step * code).to(dtype).double()
        return got | {"weights": weights, "places": None}
    b, budget, sink, lens = case["batch"], case["budget"], case["sink"], _lens(case)
    weights, got = s["weights"].double(), {}
    stay = torch.empty((case["layers"], b, kv, budget), dtype=torch.int64)
    for layer, i, j in np.ndindex(case["layers"], b, kv):
        n = lens[i]
        late = n - case["recent"]
        w = weights[layer, i, j, sink:late].cpu().numpy()
        best = np.lexsort((np.arange(late - sink), -w))[:budget - sink - case["recent"]] + sink
        stay[layer, i, j] = torch.from_numpy(np.sort(np.concatenate((np.arange(sink), best, np.arange(late, n)))))
    stay = stay.cuda()
    layer, seq, head = (torch.arange(x, device="cuda") for x in (case["layers"], b, kv))
    at = (layer[:, None, None, None], seq[:, None, None], head[:, None], stay)
    weights[:, b:, :, :budget] = weights[at]
    for part, name in ((0, "k"), (1, "v")):
        got[name] = _numbers(s["codes"][:, part][at], s["scales"][:, part][at])
    return got | {"weights": weights, "places": None}
