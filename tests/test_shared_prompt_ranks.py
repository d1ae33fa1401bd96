"""The tokens that the ranks of a decoder go on with are the same ones (infllm_b200/utils/shared_prompt.py), whatever the ranks' random
numbers are.  gloo on the CPU."""
import socket

import pytest
import torch
import torch.multiprocessing as mp


def _rank(rank, world, port, path):
    import torch.distributed as dist

    from infllm_b200.utils import SharedPromptDecoder

    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    try:
        dec = SharedPromptDecoder.__new__(SharedPromptDecoder)
        dec.world, dec.rank, dec.group = world, rank, None
        logits = torch.randn((50, 400), generator=torch.Generator().manual_seed(1))
        g = torch.Generator().manual_seed(100 + rank)
        got = [dec._draw(logits, t, g) for t in (1.0, 0.5, 0)]
        torch.save((got, g.get_state()), f"{path}/{rank}")
        dist.barrier()
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [1, 2])
def test_ranks_go_on_with_the_same_tokens(tmp_path, world):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_rank, args=(world, port, str(tmp_path)), nprocs=world)
    tokens, states = zip(*(torch.load(tmp_path / str(r)) for r in range(world)))
    logits, g = torch.randn((50, 400), generator=torch.Generator().manual_seed(1)), torch.Generator().manual_seed(100)
    want = [torch.multinomial(torch.softmax(logits / t, dim=-1), 1, generator=g)[:, 0] for t in (1.0, 0.5)] + [logits.argmax(dim=-1)]
    for r in range(world):
        assert all(torch.equal(a, b) for a, b in zip(tokens[r], want)), r
    assert torch.equal(states[0], g.get_state())
    if world > 1:  # (the others draw too: their generators go on as before)
        other = torch.Generator().manual_seed(101)
        for t in (1.0, 0.5):
            torch.multinomial(torch.softmax(logits / t, dim=-1), 1, generator=other)
        assert torch.equal(states[1], other.get_state())
