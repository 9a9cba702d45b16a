"""Endless token-by-token decoding in a bounded cache: the decoding calls as a program uses them.

A small decoder with random weights answers a few requests at once. Every step feeds each request its last token and up
to `draft - 1` guesses of what follows (what followed the same token earlier, as one chain, and the token after that
place's other occurrence as a second branch), and takes the guesses that the decoder itself would have given:

  rotary positions    ekv_rope_append     q and k of all drafted tokens; with one token and no guesses straight into the pages
  attention           ekv_tree_attention  the drafted tree over the cached prefix
  accepted tokens     ekv_append          their rows to the end of the pages
  key weights         ekv_key_weights     what the step's queries gave to each cached key, decaying
  eviction            ekv_evict_by_weight at `limit` cached tokens a request goes back to `keep`: the first, the most
                                          recent and the heaviest, chosen per layer and KV head

    python examples/streaming_decode.py --tokens 600 --draft 8 --limit 384 --keep 256
"""
import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "embodied.cpp_b200"))
import ekv  # noqa: E402

VOCAB, HIDDEN, LAYERS, Q_HEADS, KV_HEADS, DIM = 256, 256, 3, 8, 2, 64
DECAY = 0.98


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def norm(x):
    return x * torch.rsqrt((x.float() ** 2).mean(-1, keepdim=True) + 1e-6).to(x.dtype)


class Decoder:
    """Weights, and one step over `n` tokens of every request; `attend` is the layers' attention."""

    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        def mat(rows, cols):
            return (torch.randn(rows, cols, generator=g) / math.sqrt(rows)).bfloat16().cuda()
        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).bfloat16().cuda()
        self.qkv = [mat(HIDDEN, (Q_HEADS + 2 * KV_HEADS) * DIM) for _ in range(LAYERS)]
        self.out = [mat(Q_HEADS * DIM, HIDDEN) for _ in range(LAYERS)]
        self.head = mat(HIDDEN, VOCAB)

    def __call__(self, tokens, attend):
        x = self.embed[tokens]
        for layer in range(LAYERS):
            q, k, v = (norm(x) @ self.qkv[layer]).view(-1, Q_HEADS + 2 * KV_HEADS, DIM).split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
            x = x + attend(layer, q, k, v).view(len(x), -1) @ self.out[layer]
        return norm(x).float() @ self.head.float()


class Stream:
    """The requests' cache: positions and weights of each cached row beside the pool's pages."""

    def __init__(self, requests, limit, keep, first=4, recent=64, store=ekv.DTYPE_BF16):
        self.n, self.limit, self.keep, self.first, self.recent = requests, limit, keep, first, recent
        room = limit + ekv.MAX_DRAFT
        blocks = -(-room // 16)
        self.pool = ekv.Pool(dtype=store, block_tokens=16, n_blocks=requests * blocks, kv_heads=KV_HEADS, head_dim=DIM,
                             n_layers=LAYERS, max_seqs=requests, max_blocks_per_seq=blocks)
        self.rope = ekv.Rope(rotary_dims=DIM)
        self.seqs = [self.pool.seq_create() for _ in range(requests)]
        self.seq_ids = ints(self.seqs)
        self.cached, self.seen, self.evictions = [0] * requests, [0] * requests, 0
        self.weights = torch.zeros(LAYERS, requests, KV_HEADS, room, device="cuda")
        self.positions = torch.zeros(LAYERS, requests, KV_HEADS, room, dtype=torch.int32, device="cuda")
        self.kept = torch.empty(LAYERS, requests, KV_HEADS, keep, dtype=torch.int32, device="cuda")
        self.slots = torch.arange(room, device="cuda")

    def _grow(self, counts):
        """Room for counts[i] more tokens of each request; the positions of their slots."""
        for i, c in enumerate(counts):
            self.pool.seq_resize(self.seqs[i], self.cached[i] + c)
        self.pool.sync()
        start, seen, end = (torch.tensor(v, device="cuda")[:, None] for v in
                            (self.cached, self.seen, [a + c for a, c in zip(self.cached, counts)]))
        new = (self.slots >= start) & (self.slots < end)
        self.positions = torch.where(new[None, :, None], (self.slots - start + seen).int()[None, :, None], self.positions)

    def _count(self, counts):
        self.cached = [a + c for a, c in zip(self.cached, counts)]
        self.seen = [a + c for a, c in zip(self.seen, counts)]

    def step(self, model, tokens, ancestors=None, accept=None):
        """Logits [requests, n, vocab] of n tokens of each request, as one chain or the tree of `ancestors` (int64
        [requests][n], a bit per visible token; a token's position is its depth). accept(logits) names the tokens that
        stay, by request; all of them without it."""
        n = len(tokens[0])
        depth = [[bin(w).count("1") - 1 for w in r] for r in ancestors] if ancestors else [list(range(n))] * self.n
        pos = ints([s + d for s, r in zip(self.seen, depth) for d in r])
        counts, starts = ints([n] * self.n), ints([n * i for i in range(self.n)])
        single = n == 1
        lens = ints(self.cached)
        if single:
            self._grow([1] * self.n)
        # one token alone is in the pages before it is attended to, so no drafted row is visible; words are 64-bit patterns
        words = [[0]] * self.n if single else ancestors
        up = torch.tensor([[w - (w >> 63 << 64) for w in r] for r in words], device="cuda") if words else None
        prm = [self.pool.tree_params(layer=layer, seq_ids=self.seq_ids, n_draft=n, q_heads=Q_HEADS,
                                     scale=1 / math.sqrt(DIM), ancestors=up) for layer in range(LAYERS)]
        lse, held = torch.empty(self.n, n, Q_HEADS, device="cuda"), []
        ws = torch.empty(self.pool.tree_attention_workspace_size(prm[0]), dtype=torch.uint8, device="cuda")

        def attend(layer, q, k, v):
            qr = torch.empty(self.n * n, Q_HEADS, DIM, dtype=torch.bfloat16, device="cuda")
            out = torch.empty_like(qr)
            if single:
                self.pool.rope_append(self.rope, layer, self.seq_ids, lens, counts, starts, 1, pos, q=q, q_out=qr, k=k, v=v)
                kr = vr = qr  # (not looked at)
            else:
                kr, vr = torch.empty(self.n * n, KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda"), v.contiguous()
                self.pool.rope_append(self.rope, layer, None, None, counts, starts, n, pos, q=q, q_out=qr)
                self.pool.rope_append(self.rope, layer, None, None, counts, starts, n, pos, q=k, q_out=kr)
            self.pool.tree_attention(prm[layer], qr, kr, vr, out, lse, ws)
            self.pool.key_weights(prm[layer], qr, lse, self.weights[layer], DECAY)
            held.append((kr, vr))
            return out

        logits = model(torch.tensor(tokens, device="cuda").flatten(), attend).view(self.n, n, VOCAB)
        if single:
            self._count([1] * self.n)
            if accept:
                accept(logits)
            return logits
        path = accept(logits) if accept else [list(range(n))] * self.n
        taken = [len(p) for p in path]
        self._grow(taken)
        rows = torch.tensor([i * n + j for i, p in enumerate(path) for j in p], device="cuda")
        starts = ints([sum(taken[:i]) for i in range(self.n)])
        for layer, (k, v) in enumerate(held):
            self.pool.append(layer, self.seq_ids, lens, ints(taken), starts, max(taken), k[rows], v[rows])
        self._count(taken)
        return logits

    def evict(self):
        """Once a request is above the limit all go back to `keep` rows per layer and KV head (shorter ones stay)."""
        if max(self.cached) <= self.limit:
            return
        self.pool.evict_by_weight(0, LAYERS, self.seq_ids, self.weights, keep=self.keep, first=self.first,
                                  recent=self.recent, kept=self.kept, weights_out=self.weights,
                                  positions=self.positions, positions_out=self.positions, seen=ints(self.seen))
        self.cached = [min(c, self.keep) for c in self.cached]
        for s, c in zip(self.seqs, self.cached):
            self.pool.seq_resize(s, c)
        self.pool.sync()
        self.weights[..., self.keep:] = 0.0  # of the slots that new tokens will take
        self.evictions += 1


def guesses(text, n):
    """Up to n - 1 tokens that may follow, as (tokens, ancestor words) of a tree under the last token."""
    tokens, words = [text[-1]], [1]
    at = [i for i in range(len(text) - 2, -1, -1) if text[i] == text[-1]][:2]
    for share, i in zip(((n - 1) - (n - 1) // 3, (n - 1) // 3), at):
        word = 1
        for t in text[i + 1:i + 1 + share]:
            word |= 1 << len(tokens)
            tokens.append(t)
            words.append(word)
    while len(tokens) < n:  # (every request drafts as many; these see only themselves and the last token)
        words.append(1 | 1 << len(tokens))
        tokens.append(0)
    return tokens, words


def generate(model, stream, prompts, count, draft):
    """Greedy continuation of `prompts` (of one length) by `count` tokens; the texts, and the steps they took."""
    texts = [list(p) for p in prompts]
    for at in range(0, len(prompts[0]) - 1, ekv.MAX_DRAFT):  # the prompt, in chains; its last token starts the first step
        stream.step(model, [p[at:min(at + ekv.MAX_DRAFT, len(p) - 1)] for p in prompts])
        stream.evict()
    steps = 0
    while min(len(t) for t in texts) < len(prompts[0]) + count:
        drafted = [guesses(t, draft) for t in texts]

        def accept(logits):
            best, paths = logits.argmax(-1).tolist(), []
            for i, (tokens, words) in enumerate(drafted):
                node, path = 0, [0]
                while node is not None:  # down the tree while a guess is what the decoder says
                    texts[i].append(best[i][node])
                    node = next((j for j in range(len(tokens)) if words[j] == words[node] | 1 << j and j > node
                                 and tokens[j] == best[i][node]), None)
                    if node is not None:
                        path.append(node)
                paths.append(path)
            return paths

        stream.step(model, [d[0] for d in drafted], [d[1] for d in drafted] if draft > 1 else None, accept)
        stream.evict()
        steps += 1
    return texts, steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=100)
    ap.add_argument("--tokens", type=int, default=600)
    ap.add_argument("--draft", type=int, default=8, help="tokens per step and request, the last one included (1: no guesses)")
    ap.add_argument("--limit", type=int, default=384)
    ap.add_argument("--keep", type=int, default=256)
    ap.add_argument("--q8", action="store_true", help="8-bit pages")
    a = ap.parse_args()
    if not 1 <= a.draft <= ekv.MAX_DRAFT or a.keep < 68 or a.keep > a.limit:
        ap.error("1 <= draft <= 64, 68 <= keep <= limit")
    model = Decoder()
    stream = Stream(a.requests, a.limit, a.keep, store=ekv.DTYPE_Q8_0 if a.q8 else ekv.DTYPE_BF16)
    prompts = torch.randint(VOCAB, (a.requests, a.prompt), generator=torch.Generator().manual_seed(1)).tolist()
    t0 = time.perf_counter()
    texts, steps = generate(model, stream, prompts, a.tokens, a.draft)
    torch.cuda.synchronize()
    new = sum(len(t) - a.prompt for t in texts)
    print(f"{new} tokens in {steps} steps ({new / steps / a.requests:.2f} a step and request), "
          f"{stream.evictions} evictions, {max(stream.cached)} tokens cached of {max(stream.seen)} seen, "
          f"pool status {stream.pool.status()}, {time.perf_counter() - t0:.2f} s")


if __name__ == "__main__":
    main()
