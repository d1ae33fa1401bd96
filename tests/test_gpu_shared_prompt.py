"""Many answers to one prompt (infllm_b200/utils/shared_prompt.py) against a textbook fp32 forward over the same weights, each
answer with its prompt as one sequence."""
import pytest
import torch

from test_gpu_decoder import BASE, SHAPE, _plain_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,prompt,n", [(16, 300, 6), (128, 257, 40), (64, 1, 3)])
def test_answers_equal_a_plain_causal_model(page, prompt, n):
    from infllm_b200.utils import SharedPromptDecoder

    torch.cuda.set_device(0)
    dec = SharedPromptDecoder(**SHAPE, n_pages=(prompt + 20 * n) // page + 3 * n + 3, page_size=page, max_tokens=1024, seed=3, rope_base=BASE,
                              init_std=0.05)
    free = dec.cache.free_pages
    ids = torch.randint(0, SHAPE["vocab"], (1, prompt), generator=torch.Generator().manual_seed(5)).cuda()
    out, trail = dec.generate_many(ids, n, max_length=5, chunk_size=128, generator=torch.Generator(device="cuda").manual_seed(1))
    assert out.shape == (n, 5) and trail.shape == (n, 5, SHAPE["vocab"])
    assert len({tuple(x) for x in out.tolist()}) > 1
    for i in range(min(n, 8)):
        want = _plain_forward(dec, torch.cat((ids[0], out[i, :-1])))[-5:]
        # the tolerance of the decoder's own test: bf16 weights' products rounded to bf16 in two layers
        scale = want.abs().max().item()
        assert (trail[i] - want).abs().max().item() <= 3e-2 * scale, i
    assert dec.cache.free_pages == free
    again, _ = dec.generate_many(ids, n, max_length=5, chunk_size=128, generator=torch.Generator(device="cuda").manual_seed(1))
    assert torch.equal(out, again)
    one, _ = dec.generate_many(ids, 2, max_length=3, temperature=0)
    assert torch.equal(one[0], one[1]) and one[0, 0] == trail[0, 0].argmax()


def test_what_does_not_fit_leaves_the_cache_as_it_was():
    from infllm_b200 import _lib as L
    from infllm_b200.utils import SharedPromptDecoder

    dec = SharedPromptDecoder(**SHAPE, n_pages=8, page_size=16, max_sequences=5, max_tokens=256, seed=3)
    ids = torch.zeros((1, 60), dtype=torch.int64, device="cuda")
    for call in (lambda: dec.generate_many(torch.zeros((1, 200), dtype=torch.int64, device="cuda"), 1), lambda: dec.generate_many(ids, 5),
                 lambda: dec.generate_many(ids, 2, max_length=60)):
        with pytest.raises(L.InfLLMCapacityError):
            call()
        assert dec.cache.free_pages == 8
    with pytest.raises(ValueError):
        dec.generate_many(ids[:, :0], 1)
    with pytest.raises(TypeError):  # the attention type alone, without a layer of a batch
        dec.step(ids)
    assert dec.generate_many(ids, 2, max_length=2)[0].shape == (2, 2)


def test_answers_whose_attention_gave_up_are_not_returned(monkeypatch):
    """A wait that ran out in the last steps' kernels is reported before the answers are (set from the host)."""
    from infllm_b200 import _lib as L
    from infllm_b200.utils import SharedPromptDecoder

    dec = SharedPromptDecoder(**SHAPE, n_pages=40, page_size=16, max_sequences=5, max_tokens=256, seed=3)
    ids, step, calls = torch.zeros((1, 60), dtype=torch.int64, device="cuda"), dec.step, []

    def last(x):
        out = step(x)
        calls.append(x)
        if len(calls) == 3:  # the prompt, and two tokens
            L.check(L.lib.infllm_pages_error_set(dec.cache.handle, 1, 722))
        return out

    monkeypatch.setattr(dec, "step", last)
    with pytest.raises(L.InfLLMError, match="wait 722"):
        dec.generate_many(ids, 2, max_length=3)
    assert dec.cache.free_pages == 40
    assert dec.generate_many(ids, 2, max_length=3)[0].shape == (2, 3)


def test_generate_is_one_greedy_answer():
    """The decoder's own generate(): the same tokens and logits as one answer of generate_many."""
    from infllm_b200.utils import SharedPromptDecoder

    dec = SharedPromptDecoder(**SHAPE, n_pages=60, page_size=16, max_tokens=1024, seed=3, rope_base=BASE, init_std=0.05)
    ids = torch.randint(0, SHAPE["vocab"], (1, 300), generator=torch.Generator().manual_seed(5)).cuda()
    out, trail = dec.generate(ids, max_length=5, chunk_size=128)
    assert len(out) == 5 and all(isinstance(x, int) for x in out) and trail.shape == (5, SHAPE["vocab"])
    many, logits = dec.generate_many(ids, 1, max_length=5, chunk_size=128, temperature=0)
    assert many[0].tolist() == out and torch.equal(logits[0], trail)
    assert dec.cache.free_pages == 60


def test_logits_need_not_be_kept():
    """The same answers, without memory of (n, max_length, vocab)."""
    from infllm_b200.utils import SharedPromptDecoder

    shape = dict(SHAPE, vocab=60000)
    dec = SharedPromptDecoder(**shape, n_pages=200, page_size=16, max_tokens=1024, seed=3, rope_base=BASE, init_std=0.05)
    ids = torch.randint(0, shape["vocab"], (1, 40), generator=torch.Generator().manual_seed(5)).cuda()
    most = []
    for keep in (True, False):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        base = torch.cuda.memory_allocated()
        out, trail = dec.generate_many(ids, 30, max_length=40, generator=torch.Generator(device="cuda").manual_seed(1), keep_logits=keep)
        torch.cuda.synchronize()
        most.append(torch.cuda.max_memory_allocated() - base)
        if keep:
            want = out
            assert trail.shape == (30, 40, shape["vocab"])
        else:
            assert trail is None and torch.equal(out, want)
        del trail
    kept = 30 * 40 * shape["vocab"] * 4
    # a step's logits and what the draw makes of them are there in either case
    assert most[0] >= kept and most[1] <= kept // 2
