"""The streaming example on the GPU: what it generates is what its decoder says, and its cache holds what it should.

Tolerance of the first test: the example rounds to bf16 about eight times a layer, each time by 2^-9 of a unit-sized value
(root mean square); over three layers, and the difference of two logits, that is 0.02. The largest of some hundred
differences is taken to be within 7 of these."""
import importlib.util
import os

import pytest
import torch

import ekv

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("streaming_decode", os.path.join(ROOT, "examples", "streaming_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def prompts(ex, n, length):
    return torch.randint(ex.VOCAB, (n, length), generator=torch.Generator().manual_seed(3)).tolist()


def turn(x, pos):
    """x [tokens, heads, dim] turned by its positions, in halves."""
    half = x.shape[-1] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    a = pos.double()[:, None, None] * f
    x = x.double()
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * a.cos() - hi * a.sin(), lo * a.sin() + hi * a.cos()], -1)


def plain_logits(ex, model, text):
    t = torch.tensor(text, device="cuda")
    pos = torch.arange(len(text), device="cuda")
    n, g = len(text), ex.Q_HEADS // ex.KV_HEADS
    unit = lambda x: x * torch.rsqrt((x ** 2).mean(-1, keepdim=True) + 1e-6)
    x = model.embed[t].double()
    for layer in range(ex.LAYERS):
        q, k, v = (unit(x) @ model.qkv[layer].double()).view(n, -1, ex.DIM).split([ex.Q_HEADS, ex.KV_HEADS, ex.KV_HEADS], 1)
        q, k, v = turn(q, pos), turn(k, pos).repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        s = torch.einsum("qhd,khd->hqk", q, k) / ex.DIM ** 0.5
        s = s.masked_fill(pos[None, :, None] < pos[None, None, :], float("-inf")).softmax(-1)
        x = x + torch.einsum("hqk,khd->qhd", s, v).reshape(n, -1) @ model.out[layer].double()
    return unit(x) @ model.head.double()


@pytest.mark.parametrize("draft", [1, 2, 9, 64])
def test_tokens_are_the_decoders(draft):
    ex = example()
    model, length = ex.Decoder(), 70
    stream = ex.Stream(3, 400, 256)
    texts, steps = ex.generate(model, stream, prompts(ex, 3, length), 60, draft)
    assert stream.pool.status() == 0 and stream.evictions == 0 and steps <= 60
    for text in texts:
        logits = plain_logits(ex, model, text)[length - 1:-1]
        got = torch.tensor(text[length:], device="cuda")
        short = logits.max(-1).values - logits.gather(1, got[:, None])[:, 0]
        assert short.max().item() <= 0.14


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("draft", [1, 7])
def test_cache_stays_bounded_and_whole(draft, q8):
    ex = example()
    model, length = ex.Decoder(), 90
    stream = ex.Stream(3, 144, 100, store=ekv.DTYPE_Q8_0 if q8 else ekv.DTYPE_BF16)
    texts, _ = ex.generate(model, stream, prompts(ex, 3, length), 200, draft)
    assert stream.pool.status() == 0 and stream.evictions >= 3
    for i, text in enumerate(texts):
        n, seen = stream.cached[i], stream.seen[i]
        assert n <= 144 and stream.pool.seq_get(stream.seqs[i]).n_tokens == n and seen == len(text) - 1
        for layer in range(ex.LAYERS):
            for h in range(ex.KV_HEADS):
                at = sorted(stream.positions[layer, i, h, :n].tolist())
                assert len(set(at)) == n and at[:4] == [0, 1, 2, 3] and at[-64:] == list(range(seen - 64, seen))
        # the first layer's keys depend on token and position alone
        k, v = (torch.empty(n, ex.KV_HEADS, ex.DIM, device="cuda") for _ in range(2))
        stream.pool.gather(0, stream.seqs[i], 0, n, ekv.GATHER_F32, k, v)
        for h in range(ex.KV_HEADS):
            pos = stream.positions[0, i, h, :n]
            rows = (ex.norm(model.embed[torch.tensor(text, device="cuda")[pos]]) @ model.qkv[0]).view(n, -1, ex.DIM)
            want_k, want_v = turn(rows[:, ex.Q_HEADS + h:ex.Q_HEADS + h + 1], pos)[:, 0], rows[:, -ex.KV_HEADS + h].double()
            for got, want in ((k[:, h], want_k), (v[:, h], want_v)):
                # bf16: 2^-8 of the value, for the product's rounding of another order and the turned value's; Q8_0: half a
                # step of 1/127 of the largest of 32 as well
                top = want.abs().view(n, -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(n, -1)
                size = (want ** 2 + want.roll(ex.DIM // 2, 1) ** 2).sqrt()
                assert ((got.double() - want).abs() <= size * 2 ** -7 + 1e-3 + (top / 250 if q8 else 0)).all()
