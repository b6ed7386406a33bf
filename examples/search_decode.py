"""Beam search, then speculative steps, over one paged KV cache.

A small transformer of random Q8_0 weights (no checkpoint is needed) stands for the model: what matters is the
order of the calls. Each step of the search runs the model on one new token per beam, picks the best
continuations, forks the beams that go on and writes the new rows; the winner then goes on with drafted trees:
the model runs on all drafted tokens at once, the path that it agrees with is written, the rest is dropped.

    python examples/search_decode.py            # on a gfx950 GPU
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import densecore_amd as dc  # noqa: E402

PAGE = dc.KV_BLOCK_SIZE


class Model:
    """Attention layers with residuals and an LM head; every product is the library's."""

    def __init__(self, layers=3, heads=8, kv_heads=2, head_dim=64, vocab=1000, seed=0, device="cuda"):
        self.layers, self.heads, self.kv_heads, self.head_dim, self.vocab = layers, heads, kv_heads, head_dim, vocab
        self.hidden, self.device = heads * head_dim, device
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)

        def weight(n, k):
            w = torch.randn((n, k), generator=gen, device=device) / k ** 0.5
            return dc.quantize_weights(dc.TYPE_Q8_0, w), n, k
        kv = kv_heads * head_dim
        self.embed = torch.randn((vocab, self.hidden), generator=gen, device=device)
        self.blocks = [[weight(n, self.hidden) for n in (self.hidden, kv, kv, self.hidden)] for _ in range(layers)]
        self.head = weight(vocab, self.hidden)

    @staticmethod
    def _product(w, x):
        return dc.mul_mat(dc.TYPE_Q8_0, w[0], w[1], w[2], x)

    @staticmethod
    def _residual(w, x, r):
        return dc.mul_mat_add(dc.TYPE_Q8_0, w[0], w[1], w[2], x, r)

    @staticmethod
    def _normed(x):
        return x / x.square().mean(-1, keepdim=True).add(1e-6).sqrt()

    def forward(self, tokens, cache, tables, lengths, max_past, mask=None):
        """tokens [S, N] after each sequence's cached ones -> logits [S * N, vocab] (temperature 1/3), and the new
        rows k, v [layers, S * N, row_elems]."""
        x = self.embed[tokens.reshape(-1)]
        ks, vs = [], []
        for layer, (wq, wk, wv, wo) in enumerate(self.blocks):
            n = self._normed(x)
            k, v = self._product(wk, n), self._product(wv, n)
            a = cache.tree_attention(layer, tables, lengths, max_past, self._product(wq, n), k, v, self.head_dim ** -0.5,
                                     mask=mask)
            x = self._residual(wo, a, x)
            ks.append(k)
            vs.append(v)
        return 3.0 * self._product(self.head, self._normed(x)), torch.stack(ks), torch.stack(vs)


def grow(tables, lengths, refs, more):
    """Pages for the next `more` positions of each sequence, the lowest free ones (on the device)."""
    for k in range(more):
        pos = lengths + k
        need = ((pos % PAGE == 0) & (torch.gather(tables, 1, (pos // PAGE).long()[:, None])[:, 0] < 0)).long()
        free = torch.sort((refs > 0).int(), stable=True).indices
        page = free[torch.cumsum(need, 0) - need].int()
        at = (pos // PAGE).long()[:, None]
        tables.scatter_(1, at, torch.where(need.bool(), page, torch.gather(tables, 1, at)[:, 0])[:, None])
        refs.index_add_(0, page.long(), need.int())


class Search:
    """The beams' state: block tables, lengths and page counts, all on the device."""

    def __init__(self, model, cache_type, pages=64, width=16):
        self.model, self.width = model, width
        self.cache = dc.PagedKVCache(cache_type, pages, model.layers, model.kv_heads, model.head_dim, device=model.device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=model.device)
        self.tables = torch.full((1, width), -1, dtype=torch.int32, device=model.device)
        self.lengths = torch.zeros(1, dtype=torch.int32, device=model.device)
        self.length = 0  # what the host knows: all sequences are as long

    def _write(self, path, k, v):
        """The rows of the drafted tokens `path` [S, P] behind each sequence."""
        grow(self.tables, self.lengths, self.refs, path.shape[1])
        self.cache.write_path(self.tables, self.lengths, path, None, k, v)
        self.lengths += path.shape[1]
        self.length += path.shape[1]

    def prompt(self, tokens):
        """tokens [1, N]; the last token's logits."""
        logits, k, v = self.model.forward(tokens, self.cache, self.tables, self.lengths, self.length)
        self._write(torch.arange(tokens.shape[1], dtype=torch.int32, device=tokens.device)[None], k, v)
        return logits[-1:]

    def fork(self, parents):
        self.tables, self.lengths, self.refs, missing = self.cache.fork(self.tables, self.lengths, parents, self.refs)
        return missing

    def beams(self, tokens, beams, steps):
        """`steps` tokens behind the prompt: (tokens [beams, steps], scores [1, beams], copies without a page)."""
        logits = self.prompt(tokens)
        scores, parents, picked = dc.beam_select(logits, torch.zeros((1, 1), device=logits.device), beams)
        missing = self.fork(parents[0])
        out = picked[0][:, None]
        zero = torch.zeros((beams, 1), dtype=torch.int32, device=logits.device)
        for _ in range(steps - 1):
            logits, k, v = self.model.forward(out[:, -1:].long(), self.cache, self.tables, self.lengths, self.length)
            self._write(zero, k, v)
            scores, parents, picked = dc.beam_select(logits, scores, beams)
            missing = missing + self.fork(parents[0])
            out = torch.cat([out[parents[0].long()], picked[0][:, None]], 1)
        return out, scores, missing

    def keep(self, beam):
        """One beam goes on, the others' pages become free; the pages in use move to the front."""
        self.fork(torch.tensor([beam], dtype=torch.int32, device=self.refs.device))
        self.tables, self.refs, n_live = self.cache.compact(self.tables, self.lengths, self.refs)
        return n_live

    def speculate(self, last, drafts, parents):
        """One step with a drafted tree: node 0 is the last token, node i > 0 token drafts[i - 1] behind node
        parents[i - 1]. Returns the tokens that greedy decoding takes, one more than accepted drafts."""
        n = len(drafts) + 1
        seen = np.eye(n, dtype=bool)
        for i, p in enumerate(parents, 1):
            seen[i] |= seen[p]
        bits = np.zeros((1, n, (n + 63) // 64), np.uint64)
        for i, j in zip(*np.nonzero(seen)):
            bits[0, i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
        dev = self.refs.device
        tokens = torch.tensor([[last] + list(drafts)], device=dev)
        logits, k, v = self.model.forward(tokens, self.cache, self.tables, self.lengths, self.length,
                                          mask=torch.from_numpy(bits.view(np.int64)).to(dev))
        best = logits.argmax(1).tolist()
        node, path, taken = 0, [0], []
        while True:
            taken.append(best[node])
            follow = [i for i, p in enumerate(parents, 1) if p == node and drafts[i - 1] == best[node]]
            if not follow:
                break
            node = follow[0]
            path.append(node)
        self._write(torch.tensor([path], dtype=torch.int32, device=dev), k, v)
        return taken


def main():
    model = Model()
    search = Search(model, dc.TYPE_F16)
    prompt = torch.arange(40, device="cuda")[None] * 7 % model.vocab
    out, scores, missing = search.beams(prompt, beams=4, steps=24)
    print("beams", [f"{s:.3f}" for s in scores[0].tolist()], "copies without a page:", int(missing))
    print("best ", out[0].tolist())
    print("pages in use after the search:", int(search.keep(0)))
    text, rng = out[0].tolist(), np.random.default_rng(0)
    while len(text) < 40:
        # a draft: some guesses behind the last token, and a chain behind the first of them
        drafts, parents = [int(x) for x in rng.integers(0, model.vocab, 6)], [0, 0, 0, 1, 4, 5]
        text += search.speculate(text[-1], drafts, parents)
    print("then ", text[24:])


if __name__ == "__main__":
    main()
