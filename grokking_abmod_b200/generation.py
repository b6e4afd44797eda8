"""Generation and scoring with a Mesh GPT over the 8-bit key/value cache.

``CachedGpt`` holds a trained model's weights on the GPU and, for a batch of
sequences, the cached keys and values of what they have seen.  ``extend``
feeds further tokens - whole prompts or one token each - and returns their
logits, composing the model from the per-op entry points of ``ops``: the
reference regenerates every prefix instead (src/bin/mesh-gpt.rs ``generate``).
"""

import numpy as np

from . import ops
from .gpt import MeshGpt


class CachedGpt:
    """``sequences`` running sequences of ``model``, up to its context each.

    The model's operators set the limits: widths 64, 128, 256, 384 and 512."""

    def __init__(self, model: MeshGpt, sequences: int, page_tokens: int = 16):
        import torch
        c = self.config = model.config
        self.sequences = sequences
        weights = torch.from_numpy(model.parameters()).cuda()
        stack = lambda at, depth: weights[at:at + 2 * c.width * depth].view(depth, c.width, 2)  # noqa: E731
        a, f = c.attention_mesh_depth, c.ffn_mesh_depth
        at = 2 * c.width * a if c.embedding == "mesh" else c.vocab_size * c.width
        self.blocks = []
        for _ in range(c.layers):
            starts = [at + i * 2 * c.width * a for i in range(5)]
            self.blocks.append([stack(s, a) for s in starts[:4]] + [stack(starts[4], f)])
            at = starts[4] + 2 * c.width * f
        self.embeddings = torch.from_numpy(model.token_embeddings()).cuda()
        self.hd = c.width // c.heads
        pages = -(-c.context // page_tokens)
        self.caches = [ops.new_kv_cache(sequences * pages, c.heads, self.hd, page_tokens) for _ in range(c.layers)]
        self.table = torch.arange(sequences * pages, dtype=torch.int32, device="cuda").view(sequences, pages)
        self.lengths = np.zeros(sequences, dtype=np.int64)
        self.status = ops.new_status()
        half = self.hd // 2
        freq = 10000.0 ** (torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(c.context, dtype=torch.float64)[:, None] / freq
        self.cos, self.sin = (t.float().cuda()[:, None] for t in (angle.cos(), angle.sin()))

    def _rotate(self, x, positions):
        """Slice RoPE at the rows' own positions (src/gpt/gpu.rs:175-208)."""
        import torch
        a, b = x.unflatten(1, (self.config.heads, self.hd)).chunk(2, dim=2)
        cos, sin = self.cos[positions], self.sin[positions]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=2)

    def extend(self, tokens):
        """Appends ``tokens[b]`` (a list, possibly empty) to sequence b;
        returns the logits [rows][vocab] of the new rows, in order."""
        import torch
        c = self.config
        news, flat = self._checked(tokens)
        if not flat.size:
            return self.embeddings.new_empty((0, c.vocab_size))
        positions = np.concatenate([np.arange(n, n + m) for n, m in zip(self.lengths, news)])
        held = self.lengths + news
        ints = lambda v: torch.from_numpy(np.asarray(v, dtype=np.int32)).cuda()  # noqa: E731
        lengths, offsets = ints(held), ints(np.concatenate([[0], np.cumsum(news)]))
        positions = torch.from_numpy(positions).cuda()
        most = dict(max_new=int(news.max()), status=self.status)
        conn = 0 if c.connectivity == "neighbor" else 1
        heads = lambda t: t.unflatten(1, (c.heads, self.hd))  # noqa: E731
        x = self.embeddings[torch.from_numpy(flat).cuda()]
        for cache, (wq, wk, wv, wo, wf) in zip(self.caches, self.blocks):
            n = ops.rmsnorm_forward(x)[0]
            q, k, v = (ops.mesh_forward(n, w, conn) for w in (wq, wk, wv))
            q, k = (self._rotate(ops.rmsnorm_forward(t, c.heads)[0], positions) for t in (q, k))
            ops.cache_write(cache, k, heads(v), self.table, lengths, offsets, **most)
            y, _ = ops.cache_attention(q, cache, self.table, lengths, offsets, max_tokens=int(held.max()), **most)
            x = x + ops.mesh_forward(ops.xsa_forward(y.flatten(1), v, c.heads), wo, conn)
            x = x + ops.mesh_forward(ops.rmsnorm_forward(x)[0], wf, conn)
        logits = ops.rmsnorm_forward(x)[0] @ self.embeddings.t()
        self.lengths = held  # not before: what a failed step wrote past the lengths is written again
        return logits

    def _checked(self, tokens, more: int = 0):
        """(number of tokens of each sequence, all of them), if they and
        ``more`` after them fit."""
        c = self.config
        news = np.array([len(t) for t in tokens], dtype=np.int64)
        if len(news) != self.sequences:
            raise ValueError("one list of tokens for each sequence")
        if (self.lengths + news + more > c.context).any():
            raise ValueError("a sequence would outgrow the model's context")
        flat = np.concatenate([np.asarray(t, dtype=np.int64) for t in tokens]) if news.sum() else np.zeros(0, np.int64)
        if ((flat < 0) | (flat >= c.vocab_size)).any():
            raise ValueError("token ID is outside the vocabulary")
        return news, flat

    def _followed(self, tokens, top: int, more: int = 0):
        """Checks, before anything moves, that every sequence brings a token
        for the next one to follow, that ``more`` fit behind, and ``top``."""
        news, _ = self._checked(tokens, more)
        if not news.all():
            raise ValueError("a list of at least one token for each sequence")
        if not 0 <= top <= min(32, self.config.vocab_size):
            raise ValueError("top must be in 0..32 and at most the vocabulary")

    def generate(self, tokens, steps: int, top: int = 1):
        """Extends each sequence by ``tokens[b]`` (one token at least) and
        chooses its most likely token, which extends it for the next of
        ``steps`` choices.  Returns [(TokenLogprobs of the chosen tokens, with
        the ``top`` alternatives) per step]; the chosen tokens are
        ``top_index[:, 0]``.  The last ones are not part of the sequences yet:
        pass them in to go on."""
        import torch
        self._followed(tokens, top, steps - 1)
        out = []
        for _ in range(steps):
            logits = self.extend(tokens)
            ends = torch.from_numpy(np.cumsum([len(t) for t in tokens]) - 1).cuda()
            last = logits[ends]
            chosen = last.argmax(1).int()
            out.append(ops.token_logprobs(last, chosen, max(1, top), status=self.status))
            tokens = [[t] for t in out[-1].top_index[:, 0].tolist()]
        ops.check_status(self.status)
        return out

    def score(self, tokens, answers, top: int = 0):
        """Log-probabilities, entropies and alternatives of ``answers[b]`` as
        the token that follows ``tokens[b]`` (one token at least), by which the
        sequences are extended."""
        import torch
        self._followed(tokens, top)
        given = np.asarray(answers, dtype=np.int64)
        if given.shape != (self.sequences,) or ((given < -1) | (given >= self.config.vocab_size)).any():
            raise ValueError("one answer for each sequence, inside the vocabulary (or -1: none)")
        logits = self.extend(tokens)
        ends = torch.from_numpy(np.cumsum([len(t) for t in tokens]) - 1).cuda()
        given = torch.from_numpy(given.astype(np.int32)).cuda()
        r = ops.token_logprobs(logits[ends], given, top, status=self.status)
        ops.check_status(self.status)
        return r
