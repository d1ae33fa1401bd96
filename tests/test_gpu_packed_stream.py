"""Long streams over the packed cache (infllm_b200/utils/packed_stream.py): every attention of a generation against the formulas over what the
cache holds, and what stays of a stream."""
import math

import pytest
import torch

from test_gpu_decoder import BASE, SHAPE
from test_gpu_packed_cache import TINY, U, formula, held

pytestmark = pytest.mark.gpu


def decoder(**more):
    from infllm_b200.utils import PackedStreamDecoder

    torch.cuda.set_device(0)
    return PackedStreamDecoder(**SHAPE, seed=3, rope_base=BASE, init_std=0.05, **more)


def prompts(n, length):
    return torch.randint(0, SHAPE["vocab"], (n, length), generator=torch.Generator().manual_seed(5)).cuda()


@pytest.mark.parametrize("n,length,chunk,more", [(1, 1, 64, {}), (2, 300, 128, {}), (3, 500, 130, dict(budget=150, sink=4, recent=40, slack=3)),
                                                 (1, 700, 700, dict(budget=60, sink=0, recent=60, slack=0, decay=0.5))])
def test_every_attention_of_a_generation(monkeypatch, n, length, chunk, more):
    from infllm_b200.attention import PackedBatch

    dec = decoder(max_tokens=800, n_sequences=4, **more)
    attend, seen = PackedBatch.attend, []

    def checked(self, layer, q, **kwargs):
        out = attend(self, layer, q, **kwargs)
        c, tokens, u = self.cache, q.size(2), U[self.cache.dtype]
        for i, s in enumerate(self.seqs):
            want, mass, _, _, e = formula(q[i], *held(c, layer, s), tokens, 1 / math.sqrt(c.head_dim))
            err = (out[i].double() - want).abs()
            assert (err <= u * want.abs() + (u + 2.0 ** -16 + 2 * e[..., None]) * mass + TINY[c.dtype]).all()
        seen.append([c.length(s) for s in self.seqs])
        assert [c.position(s) for s in self.seqs] == [min(chunk * (1 + len(seen[:-1]) // 2), length) + max(0, len(seen[:-1]) // 2 + 1 - -(-length // chunk))] * n
        return out

    monkeypatch.setattr(PackedBatch, "attend", checked)
    out, trail = dec.generate_many(prompts(n, length), max_length=12, chunk_size=chunk)
    assert out.shape == (n, 12) and trail.shape == (n, 12, SHAPE["vocab"]) and torch.equal(out, trail.argmax(-1))
    steps = -(-length // chunk) + 11
    assert len(seen) == 2 * steps
    if "budget" in more:
        most = more["budget"] + max(more["slack"] + 1, chunk)
        assert max(map(max, seen)) <= most and max(seen[-1]) <= more["budget"] + more["slack"] + 1
    else:
        assert seen[-1] == [length + 11] * n
    monkeypatch.undo()
    again, _ = dec.generate_many(prompts(n, length), max_length=12, chunk_size=chunk)
    assert torch.equal(out, again)
    assert dec.cache.open(4) == [0, 1, 2, 3]


def test_refusals_leave_the_cache_as_it_was():
    from infllm_b200 import _lib as L
    from infllm_b200.utils import PackedStreamDecoder

    with pytest.raises(ValueError):
        PackedStreamDecoder(**SHAPE, max_tokens=64, budget=10, sink=5, recent=6)
    with pytest.raises(ValueError):
        PackedStreamDecoder(**SHAPE, max_tokens=64, budget=40, slack=24)
    dec = decoder(max_tokens=100, n_sequences=2, budget=40, slack=20)
    for call, error in ((lambda: dec.generate_many(prompts(3, 10)), L.InfLLMCapacityError), (lambda: dec.generate_many(prompts(1, 200)), L.InfLLMCapacityError),
                        (lambda: dec.generate_many(prompts(1, 0)), ValueError), (lambda: dec.step(prompts(1, 4)), TypeError)):
        with pytest.raises(error):
            call()
    assert dec.cache.open(2) == [0, 1]
    dec.cache.free([0, 1])
    ids, logits = dec.generate(prompts(1, 300), max_length=80, chunk_size=60)
    assert len(ids) == 80 and logits.shape == (80, SHAPE["vocab"]) and logits.isfinite().all()


def test_an_attention_that_gave_up_is_reported():
    """(the record is set from the host)"""
    from infllm_b200 import _lib as L

    dec = decoder(max_tokens=100)
    L.check(L.lib.infllm_device_error_set(1, 770))
    with pytest.raises(L.InfLLMError) as e:
        dec.generate(prompts(1, 20), max_length=2)
    assert e.value.code == L.E_TIMEOUT
    dec.cache.check()
    assert len(dec.generate(prompts(1, 20), max_length=2)[0]) == 2
