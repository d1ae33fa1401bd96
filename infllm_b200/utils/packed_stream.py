"""Long streams over a cache of bounded size: the minimal decoder (decoder.py) over a cache in 4 bits that drops the tokens that attention
has looked at least.

Prompts are read in chunks; where a sequence has more than `budget` tokens after a chunk, or `slack` more than that while it is continued,
every layer and KV head keeps the first `sink`, the newest `recent` and those of the others that have had most attention.  (The reference
keeps a sink and a window, inf_llm/attention/stream_llm.py:6-111, or moves the others to the host, context_manager.py:196-816.)
"""
import torch

from ..attention import PackedCache, PackedLayer
from .decoder import HeadGroupDecoder


class PackedStreamDecoder(HeadGroupDecoder):
    """A HeadGroupDecoder of attention type "packed" with a cache of its own, for `n_sequences` sequences of up to `max_tokens` tokens:
    as many as stay and a chunk of a prompt have to fit.  budget None: nothing is dropped.  The weights that tokens have had are
    multiplied by `decay` at every step.  The other arguments are HeadGroupDecoder's; ranks choose for their own heads."""

    def __init__(self, n_layers, hidden, n_heads, n_kv_heads, head_dim, ffn, vocab, max_tokens, n_sequences=1, budget=None, sink=0, recent=0,
                 slack=64, decay=1.0, world=1, **kwargs):
        if budget is not None and (min(sink, recent) < 0 or sink + recent > budget):
            raise ValueError(f"{budget} tokens, the first {sink} and the newest {recent} among them")
        if budget is not None and not 0 <= slack < max_tokens - budget:
            raise ValueError(f"{budget} tokens, up to {slack} more and the next one, where {max_tokens} fit")
        super().__init__(n_layers, hidden, n_heads, n_kv_heads, head_dim, ffn, vocab, {}, world=world, attn_type="packed", **kwargs)
        self.cache = PackedCache(n_layers, self.kv_heads, head_dim, n_sequences, max_tokens, self.dtype, self.device)
        self.budget, self.sink, self.recent, self.slack, self.decay = budget, sink, recent, slack, decay

    def _take(self, batch):
        for i, layer in enumerate(self.layers):
            layer["past"] = PackedLayer(batch, i, weigh=self.budget is not None, decay=self.decay)

    def reset(self):
        for layer in self.layers:
            layer["past"] = None

    def _cut(self, seqs, more):
        if self.budget is not None and self.cache.length(seqs[0]) > self.budget + more:
            self.cache.evict(seqs, self.budget, self.sink, self.recent)

    @torch.inference_mode()
    def generate_many(self, input_ids, max_length=64, chunk_size=8192):
        """Greedy continuations of the prompts input_ids (n, L), each of max_length tokens: ids (n, max_length), and the logits that each
        was chosen by (n, max_length, vocab)."""
        if input_ids.size(0) < 1 or input_ids.size(1) < 1:
            raise ValueError("an empty prompt")
        seqs = self.cache.open(input_ids.size(0))
        try:
            batch = self.cache.batch(seqs)
            self._take(batch)
            for st in range(0, input_ids.size(1), chunk_size):
                ids = input_ids[:, st:st + chunk_size]
                batch.extend(ids.size(1))
                logits = self.step(ids)
                self._cut(seqs, 0)
            out, trail = [], []
            for i in range(max_length):
                trail.append(logits.clone())
                nxt = logits.argmax(dim=-1)
                if self.world > 1:  # the first rank's: with another token a rank would add another sequence's rows to the sums
                    import torch.distributed as dist

                    dist.broadcast(nxt, group=self.group, group_src=0)
                out.append(nxt)
                if i < max_length - 1:
                    batch.extend(1)
                    logits = self.step(nxt[:, None])
                    self._cut(seqs, self.slack)
            self.cache.check()
        finally:
            self.reset()
            self.cache.free(seqs)
        return torch.stack(out, dim=1), torch.stack(trail, dim=1)

    def generate(self, input_ids, max_length=64, chunk_size=8192):
        """One continuation of the prompt input_ids (1, L): generated ids, and their logits (max_length, vocab)."""
        out, trail = self.generate_many(input_ids, max_length, chunk_size)
        return out[0].tolist(), trail[0]
