"""Many answers to one prompt: the minimal decoder (decoder.py) over a paged cache.

The prompt is read once, in chunks; its sequence is forked, so that the answers share its pages, and they are decoded
together: every step's attention reads the prompt's keys and values once for all of them.  (The reference decodes one
sequence at a time, inf_llm/utils/greedy_search.py:35-105.)
"""
import torch

from ..attention import PagedCache, PagedLayer
from .decoder import HeadGroupDecoder


class SharedPromptDecoder(HeadGroupDecoder):
    """A HeadGroupDecoder of attention type "paged" with a cache of its own: `n_pages` pages of `page_size` tokens for all
    layers, `max_sequences` sequences of up to `max_tokens` tokens; the other arguments are HeadGroupDecoder's."""

    def __init__(self, n_layers, hidden, n_heads, n_kv_heads, head_dim, ffn, vocab, n_pages, page_size=128, max_sequences=256,
                 max_tokens=131072, world=1, **kwargs):
        super().__init__(n_layers, hidden, n_heads, n_kv_heads, head_dim, ffn, vocab, {}, world=world, attn_type="paged", **kwargs)
        self.cache = PagedCache(n_layers, self.kv_heads, head_dim, n_pages, page_size, max_sequences, max_tokens, self.dtype,
                                self.device)

    def _take(self, batch):
        for i, layer in enumerate(self.layers):
            layer["past"] = PagedLayer(batch, i)

    def reset(self):
        for layer in self.layers:
            layer["past"] = None

    def _draw(self, logits, temperature, generator):
        if temperature == 0:
            nxt = logits.argmax(dim=-1)
        else:
            nxt = torch.multinomial(torch.softmax(logits / temperature, dim=-1), 1, generator=generator)[:, 0]
        if self.world > 1:  # the first rank's: with other tokens than its own a rank would add another sequence's rows to the sums
            import torch.distributed as dist

            nxt = nxt.contiguous()
            dist.broadcast(nxt, group=self.group, group_src=0)
        return nxt

    def read(self, input_ids, chunk_size=8192):
        """A new sequence of the prompt input_ids (1, L): its number in the cache, and the logits of its last position."""
        if input_ids.size(1) < 1:
            raise ValueError("an empty prompt")
        seq = self.cache.open()
        try:
            batch = self.cache.batch(seq)
            self._take(batch)
            for st in range(0, input_ids.size(1), chunk_size):
                ids = input_ids[:, st:st + chunk_size]
                batch.extend(ids.size(1))
                logits = self.step(ids)
        except Exception:
            self.cache.free(seq)
            raise
        finally:
            self.reset()
        return seq[0], logits

    @torch.inference_mode()
    def generate_many(self, input_ids, n, max_length=64, chunk_size=8192, temperature=1.0, generator=None,
                      keep_logits=True):
        """n answers of max_length tokens to the prompt input_ids (1, L), drawn from the softmax of the logits over
        `temperature` with the random numbers of `generator` (a CUDA generator; temperature 0: the largest logit), of several
        ranks with the first one's.
        Returns the answers (n, max_length) and the logits that each token was drawn from (n, max_length, vocab), fp32;
        without keep_logits, None in their place."""
        root, logits = self.read(input_ids, chunk_size)
        seqs = [root]
        try:
            kids = self.cache.fork([root], n)
            seqs = seqs + kids
            batch = self.cache.batch(kids)
            self._take(batch)
            logits = logits.expand(n, -1)
            out, trail = [], []
            for i in range(max_length):
                if keep_logits:
                    trail.append(logits.clone())
                nxt = self._draw(logits, temperature, generator)
                out.append(nxt)
                if i < max_length - 1:
                    batch.extend(1)
                    logits = self.step(nxt[:, None])
            self.cache.check()
        finally:
            self.reset()
            self.cache.free(seqs)
        return torch.stack(out, dim=1), torch.stack(trail, dim=1) if keep_logits else None

    def generate(self, input_ids, max_length=64, chunk_size=8192):
        """One greedy answer to the prompt input_ids (1, L): generated ids, and their logits (max_length, vocab)."""
        out, trail = self.generate_many(input_ids, 1, max_length, chunk_size, temperature=0)
        return out[0].tolist(), trail[0]
