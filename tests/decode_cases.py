"""Plain 64-bit forms of the token-by-token decoding operators, and a pool filled with random rows."""
import math

import numpy as np
import torch

import ekv


class Cache:
    """A pool of `lens` tokens per request in shuffled blocks, filled through ekv_append; rows() are the values that the
    pages stand for."""

    def __init__(self, lens, kv_heads, dim, *, store="bf16", block=16, layers=1, seed=0, scale=1.0, spare=3, width=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // block) for n in lens]
        self.lens, self.kv_heads, self.dim, self.layers, self.block = lens, kv_heads, dim, layers, block
        self.pool = ekv.Pool(device=0, dtype=ekv.DTYPE_BF16 if store == "bf16" else ekv.DTYPE_Q8_0, block_tokens=block,
                             n_blocks=sum(need) + spare, kv_heads=kv_heads, head_dim=dim, n_layers=layers,
                             max_seqs=len(lens) + 1, max_blocks_per_seq=max(need + [1, width]))
        perm = torch.randperm(sum(need) + spare, generator=g).tolist()
        self.seqs, at = [], 0
        for n, nb in zip(lens, need):
            s = self.pool.seq_create()
            self.pool.seq_set_blocks(s, perm[at:at + nb], n)
            self.seqs.append(s)
            at += nb
        self.pool.sync()
        self.seq_ids = ints(self.seqs)
        total = sum(lens)
        starts = ints(np.cumsum([0] + lens[:-1]))
        for layer in range(layers):
            k = (torch.randn(max(1, total), kv_heads, dim, generator=g) * scale).bfloat16().cuda()
            v = (torch.randn(max(1, total), kv_heads, dim, generator=g) * scale).bfloat16().cuda()
            if total:
                self.pool.append(layer, self.seq_ids, ints([0] * len(lens)), ints(lens), starts, max(lens), k, v)

    def rows(self, b, layer=0, n=None, fmt=ekv.GATHER_F32):
        """K and V of request b as [n, kv_heads, dim]."""
        n = self.lens[b] if n is None else n
        out = [torch.zeros(n, self.kv_heads, self.dim, device="cuda") for _ in range(2)]
        if n:
            self.pool.gather(layer, self.seqs[b], 0, n, fmt, *out)
        return out

    def raw(self, b, layer=0, n=None):
        """The stored bytes of K and V."""
        n = self.lens[b] if n is None else n
        size = n * self.kv_heads * (self.dim * 2 if self.pool.cfg.dtype == ekv.DTYPE_BF16 else self.dim // 32 * 34)
        out = [torch.zeros(size + 16, dtype=torch.uint8, device="cuda") for _ in range(2)]
        if n:
            self.pool.gather(layer, self.seqs[b], 0, n, ekv.GATHER_NATIVE, *out)
        return [x[:size] for x in out]


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def words(rows):
    """Ancestor words (Python ints below 2^64) as int64 [requests, drafts]."""
    return torch.tensor([[w - (1 << 64) if w >> 63 else w for w in r] for r in rows], dtype=torch.int64, device="cuda")


def tree_words(n, seed, most=4):
    rng = np.random.default_rng(seed)
    up = []
    for i in range(n):
        back = int(rng.integers(1, most + 1))
        up.append((up[i - back] if i >= back else 0) | 1 << i)
    return up


def tree_scores(q, k, scale, cap):
    """[drafts, heads, keys] scores of q [drafts, heads, dim] against k [keys, kv_heads, dim]; also sum |q k|."""
    group = q.shape[1] // k.shape[1]
    kk = k.repeat_interleave(group, 1)
    s = torch.einsum("thd,khd->thk", q, kk) * scale
    size = torch.einsum("thd,khd->thk", q.abs(), kk.abs()) * scale
    return (cap * torch.tanh(s / cap) if cap else s), size


def tree_attention(q, k, v, kd, vd, up, nodes, scale, cap):
    """out, lse, and the row bounds sum p |v| and max sum |q k|, of one request in 64 bits: q [drafts, heads, dim], cached
    k, v [keys, kv_heads, dim], drafted kd, vd; drafted token t sees drafted j where bit j of up[t] is set."""
    q, k, v, kd, vd = (x.double() for x in (q, k, v, kd, vd))
    T, hq, d = q.shape
    group = hq // kd.shape[1]
    out = torch.zeros(T, hq, d, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=q.device)
    most = torch.zeros(T, hq, dtype=torch.float64, device=q.device)
    for t in range(nodes):
        seen = [j for j in range(nodes) if up[t] >> j & 1]
        kk, vv = torch.cat([k, kd[seen]]), torch.cat([v, vd[seen]])
        if kk.shape[0] == 0:
            continue
        s, a = tree_scores(q[t:t + 1], kk, scale, cap)
        p = torch.softmax(s[0], -1)  # [heads, keys]
        vg = vv.repeat_interleave(group, 1)
        out[t] = torch.einsum("hk,khd->hd", p, vg)
        size[t] = torch.einsum("hk,khd->hd", p, vg.abs())
        lse[t] = torch.logsumexp(s[0], -1)
        most[t] = a[0].amax(-1)
    return out, lse, size, most


def rope_table(n, base=10000.0, freq_scale=1.0, ext=0.0, fast=32.0, slow=1.0, ctx=0, factors=None):
    """Radians per position of each pair, in 64 bits."""
    f = np.array([base ** (-2.0 * i / n) / (factors[i] if factors is not None else 1.0) for i in range(n // 2)])
    mix = np.zeros(n // 2)
    if ext:
        dim = lambda turns: n * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(0.0, math.floor(dim(fast))), min(n - 1.0, math.ceil(dim(slow)))
        mix = ext * (1 - np.clip((np.arange(n // 2) - low) / max(0.001, high - low), 0, 1))
    return f * (mix + (1 - mix) * freq_scale)


def rope(x, positions, freq, n, interleaved, magnitude=1.0):
    """x [rows, heads, dim] turned in 64 bits; and the size |a| + |b| of each turned column's pair (0 past them)."""
    x = x.double().clone()
    ang = positions.double()[:, None, None] * torch.as_tensor(freq, dtype=torch.float64, device=x.device)
    c, s = torch.cos(ang) * magnitude, torch.sin(ang) * magnitude
    i, j = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., i].clone(), x[..., j].clone()
    size = torch.zeros_like(x)
    size[..., i] = size[..., j] = (a.abs() + b.abs()) * abs(magnitude)
    x[..., i], x[..., j] = a * c - b * s, a * s + b * c
    return x, size


def evict(weights, n, keep, first, recent, positions=None, seen=None):
    """kept of one (layer, request, KV head): weights, positions are the first n slots'."""
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    age = list(range(n)) if positions is None else positions
    total = n if seen is None else seen

    def key(i):
        if age[i] < first or age[i] >= total - recent:
            return (2, 0.0)
        return (0, 0.0) if math.isnan(weights[i]) else (1, float(weights[i]) + 0.0)

    order = sorted(range(n), key=lambda i: (-key(i)[0], -key(i)[1], i))
    chosen = set(order[:keep])
    tail = iter(i for i in range(keep, n) if i in chosen)
    return [i if i in chosen else next(tail) for i in range(keep)]
