"""The long-context decoding operators over the paged KV pool: cases, their plain forms, and the calls a user makes.

Four operators, in the order a decoding loop runs them on one layer:

  rope     ekv_rope_append        rotary positions on q and k, the rotated k and v written into the pool's pages
  tree     ekv_tree_attention     a tree of drafted tokens attending the cached prefix and their own ancestors
  weights  ekv_key_weights        the attention weight that every cached key got, added up over query rows
  evict    ekv_evict_by_weight    the keys with the least weight leave the cache; survivors of the tail take their rows

`run` computes a case in its plain form (elementary torch operations, 32 bits, one rounding at the end) or, where `own`
is true, through the package. Both hold the cache in the pool's storage format, so the cache itself can be returned:
tiles of `block` rows for each (block, K|V, head); a bf16 tile is [rows / 8][chunks of W bytes][8 rows][W bytes] with the
16-byte units of a row XORed by its row (W = 128 bytes where a row is a multiple of it, else 64 or 32); a Q8_0 tile is
int8 [rows][dim] (units XORed likewise) followed by f16 scales [rows][dim / 32].
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SPREAD = 1.5  # standard deviation of the scaled scores: some keys stand out, as in a trained model


def _ekv():
    path = os.path.join(ROOT, "embodied.cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ekv

    return ekv


# ---------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one decoded token of one request over an action expert's prefix: the smallest call, where latency counts
        dict(name="tree_one_token", op="tree", batch=1, len=816, spread=0, draft=1, q_heads=8, kv_heads=1, dim=256,
             block=16, store="bf16", cap=0.0, shape="chain"),
        # the serving batch of the 8-bit cache, one token each, ragged prefixes
        dict(name="tree_q8_serving", op="tree", batch=64, len=816, spread=116, draft=1, q_heads=8, kv_heads=1, dim=256,
             block=16, store="q8_0", cap=0.0, shape="chain"),
        # plain decoding of a batch over long grouped-query caches
        dict(name="tree_long_decode", op="tree", batch=16, len=16384, spread=3001, draft=1, q_heads=32, kv_heads=8,
             dim=128, block=64, store="bf16", cap=0.0, shape="chain"),
        # a small draft tree with odd sizes, capped scores, an empty cache in the batch and short trees
        dict(name="tree_capped_odd", op="tree", batch=5, len=3001, spread=3001, draft=13, q_heads=12, kv_heads=4,
             dim=64, block=24, store="bf16", cap=30.0, shape="tree"),
        # the widest tree: 64 drafted tokens of grouped-query heads, many rows for each cached key
        dict(name="tree_wide", op="tree", batch=8, len=8192, spread=1000, draft=64, q_heads=32, kv_heads=8, dim=128,
             block=64, store="bf16", cap=0.0, shape="tree"),
        # weights of one decoding step, added to those of the steps before
        dict(name="weights_decode", op="weights", batch=16, len=16384, spread=3001, draft=1, q_heads=32, kv_heads=8,
             dim=128, block=64, store="bf16", cap=0.0, decay=1.0),
        # weights of a window of the last queries, of an 8-bit cache, from scratch
        dict(name="weights_window", op="weights", batch=4, len=4099, spread=1000, draft=33, q_heads=16, kv_heads=4,
             dim=128, block=16, store="q8_0", cap=0.0, decay=0.0),
        # every layer of one streaming request gives up as many rows as a new chunk brought
        dict(name="evict_chunk", op="evict", layers=18, batch=1, len=1100, spread=0, keep=1000, first=4, recent=256,
             kv_heads=1, dim=256, block=16, store="q8_0", aged=True),
        # long prompts cut down to a quarter after their prefill
        dict(name="evict_prompt", op="evict", layers=1, batch=8, len=16384, spread=2047, keep=4096, first=4, recent=512,
             kv_heads=8, dim=128, block=64, store="bf16", aged=False),
        # one new token
        dict(name="rope_one_token", op="rope", batch=1, rows=1, spread=0, past=816, q_heads=8, kv_heads=1, dim=256,
             block=16, layout="half", rotary=256, factor=1.0, yarn=False),
        # an action chunk of a served batch, part of each head rotated in neighbouring pairs
        dict(name="rope_chunks", op="rope", batch=64, rows=50, spread=7, past=816, q_heads=8, kv_heads=1, dim=256,
             block=16, layout="interleaved", rotary=128, factor=1.0, yarn=False),
        # the prefill of long prompts past the trained length
        dict(name="rope_prefill", op="rope", batch=8, rows=4096, spread=1001, past=60000, q_heads=32, kv_heads=8,
             dim=128, block=64, layout="half", rotary=128, factor=8.0, yarn=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "evict", "rope"])
    dim = rng.choice([64, 128, 256])
    block = rng.choice([16, 24, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    if op == "rope":
        batch = _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, 8 * 4096 // batch))
        rows = max(1, min(rows, 8 * 4096 * 40 * 128 // (batch * (group + 2) * kv_heads * dim)))
        return dict(op=op, batch=batch, rows=rows, spread=rng.randrange(rows), past=_log(rng, 1, 100000),
                    q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, block=block,
                    layout=rng.choice(["half", "interleaved"]), rotary=rng.choice([dim, dim // 2, dim // 4 + 2]),
                    factor=rng.choice([1.0, 4.0]), yarn=rng.choice([False, True]))
    batch = _log(rng, 1, 64)
    longest = max(64, 16 * 16384 * 8 * 128 // (batch * kv_heads * dim))
    length = _log(rng, 33, min(60000, longest))
    if op == "evict":
        length = max(64, min(length, 8 * 16384 * 8 * 128 // (batch * kv_heads * dim)))
        keep = max(32, int(length * rng.uniform(0.1, 0.95)))
        return dict(op=op, layers=1, batch=batch, len=length, spread=rng.randrange(length), keep=keep,
                    first=rng.choice([0, 4]), recent=rng.randrange(keep - 4), kv_heads=kv_heads, dim=dim, block=block,
                    store=rng.choice(["bf16", "q8_0"]), aged=rng.choice([False, True]))
    draft = rng.choice([1, 1, _log(rng, 2, 64)])
    # at most the work of the widest listed tree
    length = max(33, min(length, 8 * 64 * 32 * 8192 * 128 // (batch * draft * kv_heads * group * dim)))
    case = dict(op=op, batch=batch, len=length, spread=rng.randrange(length), draft=draft, q_heads=kv_heads * group,
                kv_heads=kv_heads, dim=dim, block=block, store=rng.choice(["bf16", "q8_0"]),
                cap=rng.choice([0.0, 0.0, 50.0]))
    if op == "tree":
        case["shape"] = rng.choice(["chain", "tree"])
    else:
        case["decay"] = rng.choice([0.0, 0.95, 1.0])
    return case


def _lens(c):
    """Cached tokens of each request, in [len - spread, len]; the first has the most, the last the fewest."""
    less = [(b * 7919) % (c["spread"] + 1) for b in range(c["batch"])]
    if c["batch"] > 1:
        less[-1] = c["spread"]
    return [c["len"] - x for x in less]


def _rows(c):
    return [c["rows"] - (b * 7919) % (c["spread"] + 1) for b in range(c["batch"])]


def _nodes(c):
    """Drafted tokens of each request: a chain is full, a tree may be smaller than the call's widest."""
    short = 3 if c.get("shape") == "tree" else 0
    return [max(1, c["draft"] - b % (short + 1)) for b in range(c["batch"])]


def _row_bytes(c):
    return c["dim"] * 2 if c["store"] == "bf16" else c["dim"] // 32 * 34


def work(case):
    c = case
    hk, d = c["kv_heads"], c["dim"]
    if c["op"] == "rope":
        rows = sum(_rows(c))
        heads = 2 * c["q_heads"] + 4 * hk
        return {"bytes": rows * (heads * d * 2 + 16), "flops": rows * (c["q_heads"] + hk) * c["rotary"] * 3}
    lens = _lens(c)
    if c["op"] == "evict":
        slots = c["layers"] * hk * sum(lens)
        kept = c["layers"] * hk * sum(min(n, c["keep"]) for n in lens)
        # the weights are read, the kept slots and weights written; rows move where the tail's survivors take the place of
        # evicted rows: about keep * (1 - keep / len) of them at random weights
        moved = c["layers"] * hk * sum(int(c["keep"] * (1 - c["keep"] / n)) for n in lens if n > c["keep"])
        return {"bytes": slots * (8 if c["aged"] else 4) + kept * 12 + moved * 4 * _row_bytes(c), "flops": slots}
    keys = sum(lens)
    rows = sum(_nodes(c)) * c["q_heads"]
    pairs = sum(n * k for n, k in zip(lens, _nodes(c))) * c["q_heads"]
    if c["op"] == "weights":
        return {"bytes": keys * hk * (_row_bytes(c) + (8 if c["decay"] else 4)) + rows * (2 * d + 4), "flops": 2 * pairs * d}
    drafts = sum(_nodes(c)) * hk * d * 4
    return {"bytes": 2 * keys * hk * _row_bytes(c) + drafts + rows * (4 * d + 4) + 8 * sum(_nodes(c)),
            "flops": 4 * (pairs + sum(n * n for n in _nodes(c)) * c["q_heads"]) * d}


# ---------------------------------------------------------------------------------------------- the cache's storage


def _chunk(dim):
    row = 2 * dim
    return 128 if row % 128 == 0 else 64 if row % 64 == 0 else 32


def _bf16_places(dim):
    """Element offsets, inside 8 rows of a bf16 tile, of (row, column)."""
    w = _chunk(dim)
    r, byte = torch.arange(8, device="cuda")[:, None], 2 * torch.arange(dim, device="cuda")[None, :]
    off = r * w + byte % w
    off = off ^ (((off >> 7) & (w // 16 - 1)) << 4)
    return ((byte // w) * (8 * w) + off) // 2


def _q8_places(dim):
    """Byte offsets, inside 8 rows of a Q8_0 tile's int8 part, of (row, column)."""
    r, d = torch.arange(8, device="cuda")[:, None], torch.arange(dim, device="cuda")[None, :]
    return r * dim + (((d >> 4) ^ (r & (min(dim // 16, 8) - 1))) << 4) + (d & 15)


def _tile_bytes(c):
    return c["block"] * _row_bytes(c)


def _tables(c, lens, g):
    """A shuffled block table: [batch, width] block ids, -1 past a request's blocks; and the number of blocks."""
    need = [-(-n // c["block"]) for n in lens]
    perm = torch.randperm(sum(need) + 1, generator=g)
    width = max(1, max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, sum(need) + 1


class _Memory:
    """The pool's own memory as a tensor; it keeps the pool alive."""

    def __init__(self, pool, n_bytes):
        self.pool = pool
        self.__cuda_array_interface__ = dict(shape=(n_bytes,), typestr="|u1", version=2,
                                             data=(int(pool.info().prefix_base), False))


def _cache(s, c, lens, table, n_blocks, fill, layers=1):
    """The cache: its storage (made here, or the pool's own), its tables and lengths."""
    s["arena"] = fill if fill is not None else torch.zeros(layers * n_blocks * 2 * c["kv_heads"] * _tile_bytes(c),
                                                           dtype=torch.uint8, device="cuda")
    s["table"] = table.clamp(min=0).cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["seq_ids"] = torch.arange(len(lens), dtype=torch.int32, device="cuda")
    if own:
        ekv = _ekv()
        pool = ekv.Pool(device=torch.cuda.current_device(), dtype=ekv.DTYPE_BF16 if c["store"] == "bf16" else ekv.DTYPE_Q8_0,
                        block_tokens=c["block"], n_blocks=n_blocks, kv_heads=c["kv_heads"], head_dim=c["dim"],
                        n_layers=layers, max_seqs=len(lens), max_blocks_per_seq=table.shape[1])
        for b, n in enumerate(lens):
            pool.seq_set_blocks(pool.seq_create(), [x for x in table[b].tolist() if x >= 0], n)
        pool.sync()
        memory = torch.as_tensor(_Memory(pool, s["arena"].numel()), device="cuda")
        if fill is not None:
            memory.copy_(s["arena"])
        s["arena"], s["pool"] = memory, pool


def _random_store(c, n_tiles, g, scale):
    """Tiles of random rows in storage form: the order of random values inside a tile does not matter."""
    n = n_tiles * c["block"] * c["dim"]
    if c["store"] == "bf16":
        return (torch.randn(n, generator=g, device="cuda") * scale).to(torch.bfloat16).view(torch.uint8)
    tiles = torch.empty((n_tiles, _tile_bytes(c)), dtype=torch.uint8, device="cuda")
    whole = c["block"] * c["dim"]
    tiles[:, :whole] = torch.randint(-127, 128, (n_tiles, whole), generator=g, device="cuda", dtype=torch.int8).view(torch.uint8)
    # a quantiser's scales: the largest of 32 values over 127; uniform values of that range have the scale's spread
    steps = (torch.rand(n_tiles, whole // 32, generator=g, device="cuda") * 0.4 + 0.8) * (scale * math.sqrt(3) / 127)
    tiles[:, whole:] = steps.to(torch.float16).view(torch.uint8)
    return tiles.reshape(-1)


def _load(s, c, kv):
    """Rows [batch, kv_heads, tokens, dim] of K (0) or V (1) of the first layer, in 32 bits, through the block table."""
    hk, bt, d, t = c["kv_heads"], c["block"], c["dim"], s["table"]
    tiles = s["arena"].view(-1, 2, hk, _tile_bytes(c))[t, kv]  # [batch, width, heads, bytes]
    if c["store"] == "bf16":
        x = tiles.view(torch.bfloat16).reshape(*tiles.shape[:3], bt // 8, 8 * d)[..., s["places"].reshape(-1)].float()
        x = x.reshape(*tiles.shape[:3], bt, d)
    else:
        q = tiles[..., :bt * d].view(torch.int8).reshape(*tiles.shape[:3], bt // 8, 8 * d)[..., s["places"].reshape(-1)]
        steps = tiles[..., bt * d:].contiguous().view(torch.float16).float().reshape(*tiles.shape[:3], bt, d // 32, 1)
        x = (q.reshape(*tiles.shape[:3], bt, d // 32, 32).float() * steps).reshape(*tiles.shape[:3], bt, d)
    return x.permute(0, 2, 1, 3, 4).reshape(t.shape[0], hk, t.shape[1] * bt, d)


# ---------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    c = dict(case)
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "rope":
        _prepare_rope(s, c, cpu, g)
    elif c["op"] == "evict":
        _prepare_evict(s, c, cpu, g)
    else:
        _prepare_attention(s, c, cpu, g)
    return s


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _prepare_attention(s, c, cpu, g):
    b, t, hq, hk, d = c["batch"], c["draft"], c["q_heads"], c["kv_heads"], c["dim"]
    lens, nodes = _lens(c), _nodes(c)
    table, n_blocks = _tables(c, lens, cpu)
    _cache(s, c, lens, table, n_blocks, _random_store(c, n_blocks * 2 * hk, g, 1.0))
    s["places"] = (_bf16_places if c["store"] == "bf16" else _q8_places)(d)
    s["q"] = _normal(g, b, t, hq, d, scale=SPREAD)
    s["nodes"] = torch.tensor(nodes, dtype=torch.int32, device="cuda")
    s["scale"] = 1.0 / math.sqrt(d)
    if c["op"] == "tree":
        s["k_draft"], s["v_draft"] = _normal(g, b, t, hk, d), _normal(g, b, t, hk, d)
        # a node's ancestors, itself among them: bit j of word i where node i follows node j
        words = []
        for _ in range(b):
            up = []
            for i in range(t):
                back = 1 if c["shape"] == "chain" else 1 + int(torch.randint(0, 4, (1,), generator=cpu))
                up.append((up[i - back] if i >= back else 0) | 1 << i)
            words.append([w - (1 << 64) if w >> 63 else w for w in up])
        s["ancestors"] = torch.tensor(words, dtype=torch.int64, device="cuda")
    else:
        # what an attention call over the same keys says: the logarithm of the sum of about len terms
        noise = torch.rand(b, t, hq, generator=g, device="cuda") * 0.2
        s["lse"] = torch.log(s["lens"].clamp(min=1).float())[:, None, None] + SPREAD ** 2 / 2 + noise
        s["weights"] = torch.rand(b, hk, max(lens) + 3, generator=g, device="cuda") / c["len"]
    if own:
        ekv, pool = _ekv(), s["pool"]
        s["params"] = pool.tree_params(layer=0, seq_ids=s["seq_ids"], n_draft=t, q_heads=hq, scale=s["scale"],
                                       softcap=c["cap"], n_nodes=s["nodes"], ancestors=s.get("ancestors"))
        if c["op"] == "tree":
            n = pool.tree_attention_workspace_size(s["params"])
            s["workspace"] = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
            s["out"] = torch.empty(b, t, hq, d, dtype=torch.bfloat16, device="cuda")
            s["lse"] = torch.empty(b, t, hq, dtype=torch.float32, device="cuda")


def _prepare_evict(s, c, cpu, g):
    b, hk = c["batch"], c["kv_heads"]
    lens = _lens(c)
    table, n_blocks = _tables(c, lens, cpu)
    _cache(s, c, lens, table, n_blocks, _random_store(c, c["layers"] * n_blocks * 2 * hk, g, 1.0), c["layers"])
    s["n_blocks"] = n_blocks
    width = max(lens) + 5
    # weights spread over several orders; a tenth of the keys never got any, so that there are ties
    w = torch.exp(torch.randn(c["layers"], b, hk, width, generator=g, device="cuda") * 1.5)
    s["weights"] = w * (torch.rand(w.shape, generator=g, device="cuda") > 0.1)
    s["positions"] = s["seen"] = None
    if c["aged"]:
        # a cache that gave up keys before: its rows hold every second token or so of those seen, out of order below
        # the rows appended since
        seen = [2 * n + 11 for n in lens]
        pos = torch.rand(c["layers"], b, hk, width, generator=g, device="cuda")
        for i, n in enumerate(lens):
            old = n - n // 8
            order = torch.argsort(pos[:, i, :, :old], dim=-1)
            pos[:, i, :, :old] = order.float() * 2
            pos[:, i, :, old:n] = torch.arange(seen[i] - (n - old), seen[i], device="cuda").float()
        s["positions"] = pos.to(torch.int32)
        s["seen"] = torch.tensor(seen, dtype=torch.int32, device="cuda")
    if own:
        shape = (c["layers"], b, hk, c["keep"])
        s["kept"] = torch.empty(shape, dtype=torch.int32, device="cuda")
        s["weights_out"] = torch.empty(shape, dtype=torch.float32, device="cuda")
        s["positions_out"] = torch.empty(shape, dtype=torch.int32, device="cuda") if c["aged"] else None


def _prepare_rope(s, c, cpu, g):
    c["store"] = "bf16"
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    rows = _rows(c)
    table, n_blocks = _tables(c, [n + 1 for n in rows], cpu)  # rows go to positions 1 .. n of each request's pages
    _cache(s, c, [n + 1 for n in rows], table, n_blocks, None)
    s["places"] = _bf16_places(d)
    qkv = _normal(g, sum(rows), (hq + 2 * hk) * d)  # one projection's output: q, k and v of a row side by side
    s["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
    s["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    s["v"] = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
    s["n_rows"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
    s["src_row"] = (s["n_rows"].cumsum(0) - s["n_rows"]).to(torch.int32)
    s["dst_pos"] = torch.ones_like(s["n_rows"])
    owner = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), s["n_rows"].long(), output_size=sum(rows))
    at = torch.arange(sum(rows), device="cuda") - s["src_row"].long()[owner]
    s["owner"], s["at"] = owner, at + 1
    s["positions"] = (at + c["past"]).to(torch.int32)
    s["turns"] = (_frequencies(c) / (2 * math.pi)).to(torch.float32)
    if own:
        ekv = _ekv()
        s["rope"] = ekv.Rope(device=torch.cuda.current_device(), interleaved=c["layout"] == "interleaved",
                             rotary_dims=c["rotary"], freq_base=10000.0, freq_scale=1.0 / c["factor"],
                             ext_factor=1.0 if c["yarn"] else 0.0, n_ctx_orig=8192)
        s["q_out"] = torch.empty(sum(rows), hq, d, dtype=torch.bfloat16, device="cuda")


def _frequencies(c):
    """Radians per position of each rotated pair, in 64 bits. Scaled contexts: slow pairs are interpolated by the factor,
    fast ones kept, with a ramp between the pairs that turn 32 times and once over the trained length."""
    n = c["rotary"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-2.0 * i / n)
    if not c["yarn"]:
        return freq / c["factor"]
    where = [n * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0)]
    low, high = max(0.0, math.floor(where[0])), min(n - 1.0, math.ceil(where[1]))
    fast = 1 - ((i - low) / max(0.001, high - low)).clamp(0, 1)
    return freq * (fast + (1 - fast) / c["factor"])


def _magnitude(c):
    return 1.0 + 0.1 * math.log(c["factor"]) if c["yarn"] else 1.0


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "tree": _own_tree, "weights": _own_weights, "evict": _own_evict}[op](state)
    return {"rope": _plain_rope, "tree": _plain_tree, "weights": _plain_weights, "evict": _plain_evict}[op](state)


def _own_tree(s):
    s["pool"].tree_attention(s["params"], s["q"], s["k_draft"], s["v_draft"], s["out"], lse=s["lse"], workspace=s["workspace"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_weights(s):
    s["pool"].key_weights(s["params"], s["q"], s["lse"], s["weights"], decay=s["case"]["decay"])
    return {"weights": s["weights"]}


def _own_evict(s):
    c = s["case"]
    s["pool"].evict_by_weight(0, c["layers"], s["seq_ids"], s["weights"], keep=c["keep"], first=c["first"],
                              recent=c["recent"], kept=s["kept"], weights_out=s["weights_out"], positions=s["positions"],
                              positions_out=s["positions_out"], seen=s["seen"])
    r = {"kept": s["kept"], "weights": s["weights_out"], "cache": _seen_as(s)}
    if c["aged"]:
        r["positions"] = s["positions_out"]
    return r


def _own_rope(s):
    c = s["case"]
    s["pool"].rope_append(s["rope"], 0, s["seq_ids"], s["dst_pos"], s["n_rows"], s["src_row"], c["rows"], s["positions"],
                          q=s["q"], q_out=s["q_out"], k=s["k"], v=s["v"])
    return {"q": s["q_out"], "cache": _seen_as(s)}


def _seen_as(s):
    """The cache's own memory: numbers of a bf16 cache, the bytes of an 8-bit one (rows are moved whole)."""
    return s["arena"].view(torch.bfloat16) if s["case"]["store"] == "bf16" else s["arena"]


def _scores(s, k):
    """Scaled, capped scores [batch, kv_heads, group, draft, keys] of the queries against k [batch, kv_heads, keys, dim]."""
    c = s["case"]
    b, t, hq, d = s["q"].shape
    q = s["q"].float().reshape(b, t, c["kv_heads"], hq // c["kv_heads"], d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (hq // c["kv_heads"], t)) * s["scale"]
    return c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x


def _rows_first(x):
    """[batch, kv_heads, group, draft, ...] to [batch, draft, heads, ...]."""
    return x.permute(0, 3, 1, 2, *range(4, x.dim())).flatten(2, 3)


def _plain_tree(s):
    c = s["case"]
    k, v = _load(s, c, 0), _load(s, c, 1)
    cached = torch.arange(k.shape[2], device="cuda")[None, :] < s["lens"][:, None]  # [batch, keys]
    k = torch.cat([k, s["k_draft"].float().transpose(1, 2)], 2)
    v = torch.cat([torch.where(cached[:, None, :, None], v, 0.0), s["v_draft"].float().transpose(1, 2)], 2)
    at = torch.arange(c["draft"], device="cuda")
    drafted = (s["ancestors"][:, :, None] >> at & 1).bool() & (at < s["nodes"][:, None])[:, None, :]  # [batch, draft, draft]
    seen = torch.cat([cached[:, None, :].expand(-1, c["draft"], -1), drafted], 2) & (at < s["nodes"][:, None])[:, :, None]
    x = _scores(s, k).masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, p.shape[2:4]) / torch.where(total == 0, 1.0, total)
    return {"out": _rows_first(out).to(torch.bfloat16), "lse": _rows_first((top + torch.log(total)).squeeze(-1))}


def _plain_weights(s):
    c = s["case"]
    x = _scores(s, _load(s, c, 0)) - s["lse"].unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 3, 1)[..., None]
    row = torch.arange(c["draft"], device="cuda")[None, :] < s["nodes"][:, None]
    got = (torch.exp(x) * row[:, None, None, :, None]).sum((2, 3))  # [batch, kv_heads, keys]
    w = s["weights"]
    n = min(w.shape[-1], got.shape[-1])
    key = torch.arange(n, device="cuda")[None, :] < s["lens"][:, None]
    old = w[..., :n]
    w[..., :n] = torch.where(key[:, None], got[..., :n] + (c["decay"] * old if c["decay"] else 0.0), old)
    return {"weights": w}


def _plain_evict(s):
    c = s["case"]
    w, keep, n = s["weights"], c["keep"], s["lens"].long()[:, None, None]
    slot = torch.arange(w.shape[-1], device="cuda").expand(w.shape)
    age = slot if s["positions"] is None else s["positions"].long()
    total = n if s["seen"] is None else s["seen"].long()[:, None, None]
    safe = (age < c["first"]) | (age >= total - c["recent"])
    rank = torch.where(slot < n, torch.where(safe, math.inf, w), -math.inf)
    best = torch.argsort(rank, dim=-1, descending=True, stable=True)
    chosen = torch.zeros_like(w, dtype=torch.bool).scatter_(-1, best[..., :keep], True) & (slot < n)
    # the i-th free row below `keep` takes the i-th survivor above it
    hole = ~chosen[..., :keep] & (slot[..., :keep] < n)
    tail = chosen & (slot >= keep)
    order = torch.argsort((~tail).to(torch.int8), dim=-1, stable=True)  # the tail's survivors first, in their order
    take = torch.gather(order, -1, (hole.cumsum(-1) - 1).clamp(min=0))
    kept = torch.where(hole, take, slot[..., :keep])
    live = slot[..., :keep] < n
    at = torch.where(live, kept, 0)
    weights = torch.where(live, torch.gather(w, -1, at), 0.0)
    _move_rows(s, hole, kept)
    r = {"kept": torch.where(live, kept, -1).to(torch.int32), "weights": weights, "cache": _seen_as(s)}
    if c["aged"]:
        r["positions"] = torch.where(live, torch.gather(s["positions"], -1, at), -1)
    return r


def _move_rows(s, hole, kept):
    """Rows kept[hole] to the holes, K and V, in storage form."""
    c = s["case"]
    bt, d, hk = c["block"], c["dim"], c["kv_heads"]
    layer, b, h, dst = torch.nonzero(hole, as_tuple=True)
    src = kept[layer, b, h, dst]
    tiles = s["arena"].view(c["layers"] * s["n_blocks"], 2, hk, _tile_bytes(c))
    kv = torch.arange(2, device="cuda")[None, :, None]

    def rows(slot):
        blk = (layer * s["n_blocks"] + s["table"][b, slot // bt])[:, None, None]
        return blk, kv, h[:, None, None], (slot % bt)

    if c["store"] == "bf16":
        places, t = _bf16_places(d), tiles.view(torch.bfloat16)
        at = lambda r: ((r // 8 * 8 * d)[:, None] + places[r % 8])[:, None, :]  # noqa: E731
        (b1, k1, h1, r1), (b0, k0, h0, r0) = rows(src), rows(dst)
        t[b0, k0, h0, at(r0)] = t[b1, k1, h1, at(r1)]
    else:
        places = _q8_places(d)
        steps = torch.arange(d // 16, device="cuda")[None, :]
        at = lambda r: torch.cat([(r // 8 * 8 * d)[:, None] + places[r % 8], bt * d + (r * (d // 16))[:, None] + steps], 1)[:, None, :]  # noqa: E731
        (b1, k1, h1, r1), (b0, k0, h0, r0) = rows(src), rows(dst)
        tiles[b0, k0, h0, at(r0)] = tiles[b1, k1, h1, at(r1)]


def _turn(x, cos, sin, layout, n):
    """The first n columns of x [rows, heads, dim] turned by their angles [rows, 1, n / 2]."""
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if layout == "half" else (x[..., :n:2], x[..., 1:n:2])
    p, q = a * cos - b * sin, a * sin + b * cos
    front = torch.cat([p, q], -1) if layout == "half" else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([front, x[..., n:]], -1)


def _store_rows(s, k, v):
    """Rows k, v [rows, kv_heads, dim] to their pages, in storage form."""
    c = s["case"]
    bt, d, hk = c["block"], c["dim"], c["kv_heads"]
    blk = s["table"][s["owner"], s["at"] // bt]
    r = s["at"] % bt
    tiles = s["arena"].view(torch.bfloat16).view(-1, 2, hk, bt * d)
    at = ((r // 8 * 8 * d)[:, None] + s["places"][r % 8])[:, None, None, :]
    kv, h = torch.arange(2, device="cuda")[None, :, None, None], torch.arange(hk, device="cuda")[None, None, :, None]
    tiles[blk[:, None, None, None], kv, h, at] = torch.stack([k, v], 1)


def _plain_rope(s):
    c = s["case"]
    turns = s["positions"].float()[:, None, None] * s["turns"]
    angle = (turns - torch.round(turns)) * (2 * math.pi)
    cos, sin = torch.cos(angle) * _magnitude(c), torch.sin(angle) * _magnitude(c)
    q = _turn(s["q"].float(), cos, sin, c["layout"], c["rotary"]).to(torch.bfloat16)
    k = _turn(s["k"].float(), cos, sin, c["layout"], c["rotary"]).to(torch.bfloat16)
    _store_rows(s, k, s["v"])
    return {"q": q, "cache": _seen_as(s)}


# ---------------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    """Each operator from its definition, request by request, in 64 bits; whole numbers and moved rows have no other value."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = s["case"]
    if c["op"] == "evict":
        return None
    if c["op"] == "rope":
        return _exact_rope(s, c)
    b, t, hq, d = s["q"].shape
    hk = c["kv_heads"]
    group, lens, nodes = hq // hk, s["lens"].tolist(), s["nodes"].tolist()
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64, device="cuda")
    got = s["weights"].double() if c["op"] == "weights" else None
    for i in range(b):
        one = dict(s, table=s["table"][i:i + 1])
        n, m = lens[i], nodes[i]
        keys = _load(one, c, 0)[0, :, :n].double()
        if c["op"] == "tree":
            values = _load(one, c, 1)[0, :, :n].double()
            words = s["ancestors"][i, :m].tolist()
            hidden = torch.tensor([[not w >> j & 1 for j in range(m)] for w in words], device="cuda")
        for h in range(hk):
            q = s["q"][i, :m, h * group:(h + 1) * group].double().reshape(m * group, d)
            key = keys[h]
            if c["op"] == "tree":
                key = torch.cat([key, s["k_draft"][i, :m, h].double()])
            x = q @ key.T / math.sqrt(d)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["op"] == "weights":
                w = torch.exp(x - s["lse"][i, :m, h * group:(h + 1) * group].double().reshape(-1, 1)).sum(0)
                got[i, h, :n] = w + c["decay"] * got[i, h, :n]
                continue
            x.view(m, group, n + m)[:, :, n:].masked_fill_(hidden[:, None], -math.inf)
            value = torch.cat([values[h], s["v_draft"][i, :m, h].double()])
            lse[i, :m, h * group:(h + 1) * group] = torch.logsumexp(x, -1).reshape(m, group)
            out[i, :m, h * group:(h + 1) * group] = (torch.softmax(x, -1) @ value).reshape(m, group, d)
    return {"weights": got} if c["op"] == "weights" else {"out": out, "lse": lse}


def _exact_rope(s, c):
    n, hk, d, bt = c["rotary"], c["kv_heads"], c["dim"], c["block"]
    angle = s["positions"].double()[:, None, None] * _frequencies(c)
    spin = torch.polar(torch.full_like(angle, _magnitude(c)), angle)  # a pair as a complex number, times e^(i angle)
    turned = []
    for x in (s["q"].double(), s["k"].double()):
        first, second = (slice(0, n // 2), slice(n // 2, n)) if c["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * spin
        x[..., first], x[..., second] = z.real, z.imag
        turned.append(x)
    tiles = torch.zeros(s["arena"].numel() // (2 * bt * d), bt * d, dtype=torch.float64, device="cuda")
    block, r = s["table"][s["owner"], s["at"] // bt], s["at"] % bt
    place = (r // 8 * 8 * d)[:, None] + s["places"][r % 8]
    for kv, x in enumerate((turned[1], s["v"].double())):
        for h in range(hk):
            tiles[((block * 2 + kv) * hk + h)[:, None], place] = x[:, h]
    return {"q": turned[0], "cache": tiles.reshape(-1)}
