"""A language backbone served from the paged KV pool: cases of its operators, their plain forms, and the calls a user makes.

  qk       ekv_norm_rope_append   RMS norms and rotary positions of q and k heads, k and v written into the pool's pages
  window   ekv_window_attention   causal attention of appended tokens with a sliding window and first tokens (sinks) that stay
                                  visible: whole prompts, chunks, and single tokens
  fork     ekv_seq_fork           sequences that share whole blocks with another one and get a copy of its last, partial one
  compact  ekv_compact            the kept rows of sequences move together, in order, in every layer

`run` computes a case in its plain form (elementary torch operations, 32 bits, one rounding at the end) or, where `own` is
true, through the package. Both hold the cache in the pool's storage format, so the cache itself can be returned: tiles of
`block` rows for each (layer, block, K|V, head); a bf16 tile is [rows / 8][chunks of W bytes][8 rows][W bytes] with the
16-byte units of a row XORed by its row (W = 128 bytes where a row is a multiple of it, else 64 or 32); a Q8_0 tile is int8
[rows][dim] (units XORed likewise) followed by f16 scales [rows][dim / 32].
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
        # q and k of one new token: the smallest call, where latency counts
        dict(name="qk_one_token", op="qk", batch=1, rows=1, spread=0, past=816, q_heads=8, kv_heads=1, dim=256, block=16,
             layout="half", rotary=256, after=False, offset=1.0),
        # the prefill of long prompts
        dict(name="qk_prefill", op="qk", batch=8, rows=4096, spread=1001, past=0, q_heads=32, kv_heads=8, dim=128, block=64,
             layout="half", rotary=128, after=False, offset=0.0),
        # one token of one request, long after its prompt
        dict(name="window_one_token", op="window", batch=1, past=16384, rows=1, spread=0, window=1024, sinks=4, q_heads=8,
             kv_heads=1, dim=256, block=16, store="bf16"),
        # the serving batch of an 8-bit cache, one token each
        dict(name="window_q8_serving", op="window", batch=64, past=4999, rows=1, spread=997, window=1024, sinks=4, q_heads=8,
             kv_heads=1, dim=256, block=16, store="q8_0"),
        # decoding of a batch with a wide window
        dict(name="window_long_decode", op="window", batch=16, past=16384, rows=1, spread=3001, window=8192, sinks=4,
             q_heads=32, kv_heads=8, dim=128, block=64, store="bf16"),
        # ragged chunks of odd sizes after caches of any length, an empty one among them
        dict(name="window_chunks_odd", op="window", batch=5, past=3001, rows=77, spread=3001, window=300, sinks=5, q_heads=12,
             kv_heads=4, dim=64, block=24, store="bf16"),
        # the prompts of a served batch in an 8-bit cache, every earlier token visible
        dict(name="window_prompts_q8", op="window", batch=16, past=0, rows=816, spread=116, window=0, sinks=0, q_heads=8,
             kv_heads=1, dim=256, block=16, store="q8_0"),
        # long prompts, a window of a quarter of them: the largest call
        dict(name="window_prefill", op="window", batch=8, past=0, rows=4096, spread=1001, window=1024, sinks=4, q_heads=32,
             kv_heads=8, dim=128, block=64, store="bf16"),
        # four candidates of one prompt
        dict(name="fork_one", op="fork", batch=1, children=4, past=821, spread=0, layers=18, kv_heads=1, dim=256, block=16,
             store="q8_0"),
        # eight candidates of each of 32 prompts, larger pages
        dict(name="fork_batch", op="fork", batch=32, children=8, past=816, spread=101, layers=8, kv_heads=8, dim=128, block=64,
             store="bf16"),
        # old camera frames leave one request's history
        dict(name="compact_history", op="compact", batch=1, past=1100, spread=0, span=256, drop=0.3, layers=18, kv_heads=1,
             dim=256, block=16, store="q8_0"),
        # spans of any length leave long histories
        dict(name="compact_batch", op="compact", batch=8, past=8192, spread=2047, span=97, drop=0.25, layers=4, kv_heads=8,
             dim=128, block=64, store="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk", "window", "window", "window", "fork", "compact"])
    c = dict(op=op, dim=rng.choice([64, 128, 256]), block=rng.choice([16, 24, 32, 64, 128]), kv_heads=rng.choice([1, 2, 4, 8]))
    if op != "qk":  # (its rows are computed: 8-bit pages would hold their integers)
        c["store"] = rng.choice(["bf16", "q8_0"])
    group = rng.choice([1, 2, 3, 4, 8])
    columns = c["kv_heads"] * c["dim"]
    c["batch"] = batch = _log(rng, 1, 64)
    if op == "qk":
        rows = min(_log(rng, 1, 8 * 4096 // batch), 8 * 4096 * 48 * 128 // (batch * (group + 2) * columns))
        rows = max(1, rows)
        c.update(rows=rows, spread=rng.randrange(rows), past=_log(rng, 1, 100000), q_heads=c["kv_heads"] * group,
                 layout=rng.choice(["half", "interleaved"]), rotary=rng.choice([c["dim"], c["dim"] // 2, c["dim"] // 4 + 2]),
                 after=rng.choice([False, True]), offset=rng.choice([0.0, 1.0]))
    elif op == "window":
        rows = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 4096)])
        past = 0 if rows > 1 and rng.random() < 0.5 else _log(rng, 33, 60000)
        window = rng.choice([0, _log(rng, 16, 8192)])
        # at most the work of the longest listed prompts, and their memory
        seen = min(window or past + rows, past + rows)
        rows = max(1, min(rows, 8 * 4096 * 32 * 600 * 128 // (batch * group * c["kv_heads"] * max(128, c["dim"]) * seen)))
        past = min(past, max(0, 16 * 16384 * 8 * 128 // (batch * columns) - rows))
        c.update(past=past, rows=rows, spread=rng.randrange(past + 1) if rows == 1 else rng.randrange(max(past, rows)),
                 window=window, sinks=rng.choice([0, 4, rng.randrange(1, 200)]), q_heads=c["kv_heads"] * group)
    else:
        layers = rng.choice([1, 4, 18])
        past = min(_log(rng, 100, 8192), max(100, 8 * 8192 * 4 * 8 * 128 // (batch * layers * columns)))
        c.update(layers=layers, past=past, spread=rng.randrange(past))
        if op == "fork":
            c.update(children=rng.randrange(1, 9))
        else:
            c.update(span=_log(rng, 1, 300), drop=rng.uniform(0.05, 0.9))
    return c


def _less(c, b):
    """What request b's lengths are short of the longest; the first is the longest, the last the shortest."""
    if c["batch"] > 1 and b == c["batch"] - 1:
        return c["spread"]
    return (b * 7919) % (c["spread"] + 1)


def _past(c):
    """Cached tokens of each request before the call."""
    if c["op"] == "qk":
        return [0] * c["batch"]
    return [max(0, c["past"] - _less(c, b)) for b in range(c["batch"])]


def _rows(c):
    """Tokens that each request brings to the call."""
    if c["op"] in ("fork", "compact"):
        return [0] * c["batch"]
    return [max(1, c["rows"] - _less(c, b)) for b in range(c["batch"])]


def _slots(c, b, n):
    """The slots below n that request b keeps: spans of up to c["span"] tokens stay or go."""
    g = torch.Generator().manual_seed(977 * b + n)
    keep = torch.ones(n, dtype=torch.bool)
    at = 4
    while at < n:
        m = 1 + int(torch.randint(0, c["span"], (1,), generator=g))
        if float(torch.rand(1, generator=g)) < c["drop"]:
            keep[at:at + m] = False
        at += m
    return torch.nonzero(keep).flatten()


def _row_bytes(c):
    return c["dim"] * 2 if c["store"] == "bf16" else c["dim"] // 32 * 34


def _visible(c, past, rows):
    """(row, key) pairs of a request, and the slots that some row of it sees."""
    w, s = c["window"] or past + rows, c["sinks"]
    pairs = 0
    for p in range(past, past + rows):
        low = max(0, p - w + 1)
        pairs += p + 1 - low + min(s, low)
    low = max(0, past - w + 1)
    return pairs, past + rows - low + min(s, low)


def work(case):
    c = case
    hk, d = c["kv_heads"], c["dim"]
    if c["op"] == "qk":
        rows = sum(_rows(c))
        return {"bytes": rows * ((2 * c["q_heads"] + 4 * hk) * d * 2 + 16),
                "flops": rows * (c["q_heads"] + hk) * (4 * d + 3 * c["rotary"])}
    if c["op"] == "window":
        seen = [_visible(c, p, r) for p, r in zip(_past(c), _rows(c))]
        return {"bytes": 2 * hk * _row_bytes(c) * sum(n for _, n in seen) + sum(_rows(c)) * c["q_heads"] * 4 * d,
                "flops": 4 * d * c["q_heads"] * sum(n for n, _ in seen)}
    row = c["layers"] * 2 * hk * _row_bytes(c)  # K and V of a token in every layer
    if c["op"] == "fork":
        tails, tables = (sum(f(p) for p in _past(c)) for f in (lambda p: p % c["block"], lambda p: -(-p // c["block"])))
        return {"bytes": row * tails * (1 + c["children"]) + 4 * tables * (1 + c["children"]), "flops": 0}
    moved = kept = 0
    for b, n in enumerate(_past(c)):
        slots = _slots(c, b, n)
        kept += len(slots)
        moved += int((slots != torch.arange(len(slots))).sum())
    return {"bytes": 2 * row * moved + 4 * kept, "flops": 0}


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


def _random_store(c, n_tiles, g):
    """Tiles of random rows in storage form: the order of random values inside a tile does not matter."""
    n = n_tiles * c["block"] * c["dim"]
    if c["store"] == "bf16":
        return torch.randn(n, generator=g, device="cuda", dtype=torch.bfloat16).view(torch.uint8)
    tiles = torch.empty((n_tiles, _tile_bytes(c)), dtype=torch.uint8, device="cuda")
    whole = c["block"] * c["dim"]
    tiles[:, :whole] = torch.randint(-127, 128, (n_tiles, whole), generator=g, device="cuda", dtype=torch.int8).view(torch.uint8)
    # a quantiser's scales: the largest of 32 values over 127; uniform values of that range have the scale's spread
    steps = (torch.rand(n_tiles, whole // 32, generator=g, device="cuda") * 0.4 + 0.8) * (math.sqrt(3) / 127)
    tiles[:, whole:] = steps.to(torch.float16).view(torch.uint8)
    return tiles.reshape(-1)


class _Memory:
    """Memory of the pool as a tensor; it keeps the pool alive."""

    def __init__(self, pool, pointer, shape, kind):
        self.pool = pool
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, version=2, data=(int(pointer), False))


def _cache(s, c, lens, cpu, g, layers=1, spare=0, sequences=0, fill=True):
    """The cache: shuffled blocks for each request, tables, lengths; its storage made here, or the pool's own."""
    need = [-(-n // c["block"]) for n in lens]
    n_blocks = sum(need) + spare + 1
    perm = torch.randperm(n_blocks, generator=cpu)
    width = max(1, max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    s["free"] = sorted(perm[at:].tolist())  # a pool hands out the lowest first
    s["n_blocks"], s["layers"], s["width"] = n_blocks, layers, width
    s["table"] = table.clamp(min=0).cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["seq_ids"] = torch.arange(len(lens), dtype=torch.int32, device="cuda")
    n_tiles = layers * n_blocks * 2 * c["kv_heads"]
    s["arena"] = (_random_store(c, n_tiles, g) if fill
                  else torch.zeros(n_tiles * _tile_bytes(c), dtype=torch.uint8, device="cuda"))
    s["places"] = (_bf16_places if c["store"] == "bf16" else _q8_places)(c["dim"])
    if own:
        ekv = _ekv()
        pool = ekv.Pool(device=torch.cuda.current_device(), dtype=ekv.DTYPE_BF16 if c["store"] == "bf16" else ekv.DTYPE_Q8_0,
                        block_tokens=c["block"], n_blocks=n_blocks, kv_heads=c["kv_heads"], head_dim=c["dim"],
                        n_layers=layers, max_seqs=len(lens) + sequences, max_blocks_per_seq=width)
        for b, n in enumerate(lens):
            pool.seq_set_blocks(pool.seq_create(), table[b, :need[b]].tolist(), n)
        pool.sync()
        memory = torch.as_tensor(_Memory(pool, pool.info().prefix_base, (s["arena"].numel(),), "|u1"), device="cuda")
        memory.copy_(s["arena"])
        s["arena"], s["pool"] = memory, pool


def _seen_as(s):
    """The cache's own memory: numbers of a bf16 cache, the bytes of an 8-bit one (rows are moved whole)."""
    return s["arena"].view(torch.bfloat16) if s["case"]["store"] == "bf16" else s["arena"]


def _load(s, c, kv, blocks):
    """Rows [batch, kv_heads, tokens, dim] of K (0) or V (1) of the blocks [batch, n], in 32 bits."""
    hk, bt, d = c["kv_heads"], c["block"], c["dim"]
    tiles = s["arena"].view(-1, 2, hk, _tile_bytes(c))[blocks, kv]  # [batch, n, heads, bytes]
    if c["store"] == "bf16":
        x = tiles.view(torch.bfloat16).reshape(*tiles.shape[:3], bt // 8, 8 * d)[..., s["places"].reshape(-1)].float()
        x = x.reshape(*tiles.shape[:3], bt, d)
    else:
        q = tiles[..., :bt * d].view(torch.int8).reshape(*tiles.shape[:3], bt // 8, 8 * d)[..., s["places"].reshape(-1)]
        steps = tiles[..., bt * d:].contiguous().view(torch.float16).float().reshape(*tiles.shape[:3], bt, d // 32, 1)
        x = (q.reshape(*tiles.shape[:3], bt, d // 32, 32).float() * steps).reshape(*tiles.shape[:3], bt, d)
    return x.permute(0, 2, 1, 3, 4).reshape(blocks.shape[0], hk, blocks.shape[1] * bt, d)


# ---------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    c = dict(case)
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    past, rows = _past(c), _rows(c)
    if c["op"] in ("qk", "window"):
        # rows of the call, packed request by request
        s["past"] = past
        s["dst_pos"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        s["n_rows"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        s["src_row"] = (s["n_rows"].cumsum(0) - s["n_rows"]).to(torch.int32)
        s["owner"] = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), s["n_rows"].long(), output_size=sum(rows))
        s["at"] = torch.arange(sum(rows), device="cuda") - s["src_row"].long()[s["owner"]]
    if c["op"] == "qk":
        c["store"] = "bf16"
    {"qk": _prepare_qk, "window": _prepare_window, "fork": _prepare_fork, "compact": _prepare_compact}[c["op"]](
        s, c, past, rows, cpu, g)
    return s


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _prepare_qk(s, c, past, rows, cpu, g):
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    _cache(s, c, rows, cpu, g, fill=False)
    # one projection's output: q, k and v of a row side by side; heads differ in size, as projections' outputs do
    qkv = _normal(g, sum(rows), hq + 2 * hk, d) * torch.exp(torch.randn(hq + 2 * hk, 1, generator=g, device="cuda") * 0.5)
    qkv = qkv.to(torch.bfloat16)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    # learned weights near 1, stored as they are or as their difference from 1
    s["q_weight"], s["k_weight"] = (_normal(g, d, scale=0.2) + (1.0 - c["offset"]) for _ in range(2))
    s["positions"] = (s["at"] + c["past"]).to(torch.int32)
    s["eps"] = 1e-6
    s["turns"] = 10000.0 ** (torch.arange(c["rotary"] // 2, dtype=torch.float64, device="cuda") * -2 / c["rotary"]) / (2 * math.pi)
    if own:
        ekv = _ekv()
        device = torch.cuda.current_device()
        s["rope"] = ekv.Rope(device=device, interleaved=c["layout"] == "interleaved", rotary_dims=c["rotary"], freq_base=10000.0)
        s["norm"] = ekv.HeadNorm(q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"], weight_offset=c["offset"],
                                 after_rotation=c["after"])
        s["q_out"] = torch.empty(sum(rows), hq, d, dtype=torch.bfloat16, device="cuda")


def _prepare_window(s, c, past, rows, cpu, g):
    _cache(s, c, [p + r for p, r in zip(past, rows)], cpu, g)
    s["q"] = _normal(g, sum(rows), c["q_heads"], c["dim"], scale=SPREAD)
    s["scale"] = 1.0 / math.sqrt(c["dim"])
    if own:
        pool = s["pool"]
        s["params"] = pool.window_params(layer=0, seq_ids=s["seq_ids"], dst_pos=s["dst_pos"], n_rows=s["n_rows"],
                                         src_row=s["src_row"], max_rows=max(rows), q_heads=c["q_heads"], scale=s["scale"],
                                         window=c["window"], sinks=c["sinks"])
        n = pool.window_attention_workspace_size(s["params"])
        s["workspace"] = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
        s["out"] = torch.empty_like(s["q"])


def _prepare_fork(s, c, past, rows, cpu, g):
    n = c["batch"] * c["children"]
    _cache(s, c, past, cpu, g, c["layers"], spare=n, sequences=n)
    s["parents"] = [b for b in range(c["batch"]) for _ in range(c["children"])]
    s["tokens"] = [past[b] for b in s["parents"]]
    s["children"] = []
    if own:
        pool, info = s["pool"], s["pool"].info()
        every = c["batch"] + n
        s["tables"] = torch.as_tensor(_Memory(pool, info.block_tables, (every, s["width"]), "<i4"), device="cuda")[c["batch"]:]
        s["lengths"] = torch.as_tensor(_Memory(pool, info.seq_lens, (every,), "<i4"), device="cuda")[c["batch"]:]


def _prepare_compact(s, c, past, rows, cpu, g):
    _cache(s, c, past, cpu, g, c["layers"])
    kept = [_slots(c, b, n) for b, n in enumerate(past)]
    most = max(len(k) for k in kept)
    slots = torch.zeros(c["batch"], most, dtype=torch.int32)
    for b, k in enumerate(kept):
        slots[b, :len(k)] = k
    s["slots"] = slots.cuda()
    s["n_keep"] = torch.tensor([len(k) for k in kept], dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"qk": _own_qk, "window": _own_window, "fork": _own_fork, "compact": _own_compact}[op](state)
    return {"qk": _plain_qk, "window": _plain_window, "fork": _plain_fork, "compact": _plain_compact}[op](state)


def _own_qk(s):
    s["pool"].norm_rope_append(s["rope"], s["norm"], 0, s["seq_ids"], s["dst_pos"], s["n_rows"], s["src_row"], s["case"]["rows"],
                               s["positions"], q=s["q"], q_out=s["q_out"], k=s["k"], v=s["v"])
    return {"q": s["q_out"], "cache": _seen_as(s)}


def _own_window(s):
    s["pool"].window_attention(s["params"], s["q"], s["out"], workspace=s["workspace"])
    return {"out": s["out"]}


def _own_fork(s):
    pool = s["pool"]
    for child in s["children"]:  # those of the last pass are done
        pool.seq_free(child)
    s["children"] = pool.seq_fork(s["parents"], s["tokens"])
    return {"cache": _seen_as(s), "tables": s["tables"], "lengths": s["lengths"]}


def _own_compact(s):
    s["pool"].compact(0, s["case"]["layers"], s["seq_ids"], s["slots"], s["n_keep"])
    return {"cache": _seen_as(s)}


def _turn(x, cos, sin, layout, n):
    """The first n columns of x [rows, heads, dim] turned by their angles [rows, 1, n / 2]."""
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if layout == "half" else (x[..., :n:2], x[..., 1:n:2])
    p, q = a * cos - b * sin, a * sin + b * cos
    front = torch.cat([p, q], -1) if layout == "half" else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([front, x[..., n:]], -1)


def _plain_qk(s):
    c = s["case"]
    turns = s["positions"].double()[:, None, None] * s["turns"]
    angle = ((turns - torch.round(turns)) * (2 * math.pi)).float()
    cos, sin = torch.cos(angle), torch.sin(angle)

    def heads(x, weight):
        x, w = x.float(), weight.float() + c["offset"]
        if c["after"]:
            x = _turn(x, cos, sin, c["layout"], c["rotary"])
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w
        return (x if c["after"] else _turn(x, cos, sin, c["layout"], c["rotary"])).to(torch.bfloat16)

    q, k = heads(s["q"], s["q_weight"]), heads(s["k"], s["k_weight"])
    _store_rows(s, k, s["v"])
    return {"q": q, "cache": _seen_as(s)}


def _store_rows(s, k, v):
    """Rows k, v [rows, kv_heads, dim] to their pages, in storage form."""
    c = s["case"]
    slot = s["dst_pos"].long()[s["owner"]] + s["at"]
    r = slot % c["block"]
    at = ((r // 8 * 8 * c["dim"])[:, None] + s["places"][r % 8])[:, None, None, :]
    blk = s["table"][s["owner"], slot // c["block"]][:, None, None, None]
    kv, h = torch.arange(2, device="cuda")[None, :, None, None], torch.arange(c["kv_heads"], device="cuda")[None, None, :, None]
    tiles = s["arena"].view(torch.bfloat16).view(-1, 2, c["kv_heads"], c["block"] * c["dim"])
    tiles[blk, kv, h, at] = torch.stack([k, v], 1)


def _plain_window(s):
    c = s["case"]
    bt, hk, w, sinks = c["block"], c["kv_heads"], c["window"], c["sinks"]
    group, batch = c["q_heads"] // hk, c["batch"]
    out = torch.empty_like(s["q"])
    most, last = int(c["rows"]), s["table"].shape[1] - 1
    past, src = s["dst_pos"].long(), s["src_row"].long()
    even = len(set(_rows(c))) == 1
    # some rows of every request at a time, so that their scores are a few GB at most
    keys = (w or c["past"] + most) + sinks
    step = max(1, min(most, 400_000_000 // (batch * c["q_heads"] * (keys + 256)), 512))
    for r0 in range(0, most, step):
        n = min(step, most - r0)
        row = torch.arange(r0, r0 + n, device="cuda")
        live = row[None] < s["n_rows"][:, None]  # [batch, rows]
        slot = past[:, None] + row[None]
        # blocks with the first tokens, and those from the first row's window to the last row
        front = -(-sinks // bt)
        low = (past + r0 - w + 1).clamp(min=0) // bt if w else torch.zeros_like(past)
        reach = (n + w) // bt + 2 if w else (max(s["past"]) + r0 + n - 1) // bt + 1
        index = low[:, None] + torch.arange(reach, device="cuda")
        first = torch.arange(front, device="cuda").expand(batch, -1)
        index = torch.cat([first, torch.where(index < front, -1, index)], 1)  # a block once
        blocks = s["table"].gather(1, index.clamp(0, last))
        key = (index[:, :, None] * bt + torch.arange(bt, device="cuda")).flatten(1)  # [batch, keys]
        seen = (key[:, None] >= 0) & (key[:, None] <= slot[:, :, None]) & live[:, :, None]
        if w:
            seen &= (key[:, None] > slot[:, :, None] - w) | (key[:, None] < sinks)
        k, v = _load(s, c, 0, blocks), _load(s, c, 1, blocks)
        at = (src[:, None] + row[None]).clamp(max=s["q"].shape[0] - 1)
        q = s["q"][at].float().unflatten(2, (hk, group)).permute(0, 2, 3, 1, 4)  # [batch, kv_heads, group, rows, dim]
        x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (group, n)) * s["scale"]
        x = x.masked_fill(~seen[:, None, None], -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
        total = p.sum(-1, keepdim=True)
        y = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, n)) / torch.where(total == 0, 1.0, total)
        y = y.permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)  # [batch, rows, heads, dim]
        if even:
            out[at.flatten()] = y.flatten(0, 1)
        else:
            out[at[live]] = y[live]
    return {"out": out}


def _plain_fork(s):
    c = s["case"]
    bt, free = c["block"], iter(s["free"])
    n = len(s["parents"])
    tables = torch.full((n, s["width"]), -1, dtype=torch.int32)
    table = s["table"].cpu()
    tiles = s["arena"].view(s["layers"], s["n_blocks"], 2, c["kv_heads"], _tile_bytes(c))
    whole = bt * c["dim"] * (2 if c["store"] == "bf16" else 1)
    by_tail = {}
    for i, (parent, tokens) in enumerate(zip(s["parents"], s["tokens"])):
        full, tail = tokens // bt, tokens % bt
        tables[i, :full] = table[parent, :full]
        if tail:
            new = next(free)
            tables[i, full] = new
            by_tail.setdefault(-(-tail // 8) * 8, []).append((int(table[parent, full]), new))
    # the last block's rows in use, in whole groups of eight
    for rows, pairs in by_tail.items():
        src, dst = torch.tensor(pairs, device="cuda").T
        used = rows * (whole // bt)
        tiles[:, dst, :, :, :used] = tiles[:, src, :, :, :used]
        if c["store"] == "q8_0":
            end = whole + rows * (c["dim"] // 16)
            tiles[:, dst, :, :, whole:end] = tiles[:, src, :, :, whole:end]
    return {"cache": _seen_as(s), "tables": tables.cuda(), "lengths": torch.tensor(s["tokens"], dtype=torch.int32, device="cuda")}


def _plain_compact(s):
    c = s["case"]
    bt, d = c["block"], c["dim"]
    i = torch.arange(s["slots"].shape[1], device="cuda")[None]
    b, dst = torch.nonzero((i < s["n_keep"][:, None]) & (s["slots"] != i), as_tuple=True)
    src = s["slots"].long()[b, dst]
    tiles = s["arena"].view(s["layers"], s["n_blocks"], 2, c["kv_heads"], _tile_bytes(c))

    def places(slot):
        r = slot % bt
        at = (r // 8 * 8 * d)[:, None] + s["places"][r % 8]
        if c["store"] == "q8_0":
            at = torch.cat([at, bt * d + (r * (d // 16))[:, None] + torch.arange(d // 16, device="cuda")], 1)
        return s["table"][b, slot // bt][:, None], at

    # every row is read before any is written
    t = tiles.view(torch.bfloat16) if c["store"] == "bf16" else tiles
    from_block, from_at = places(src)
    to_block, to_at = places(dst)
    for layer in range(s["layers"]):
        for kv in range(2):
            for h in range(c["kv_heads"]):
                t[layer, to_block, kv, h, to_at] = t[layer, from_block, kv, h, from_at]
    return {"cache": _seen_as(s)}


# ---------------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    """The computed operators from their definitions, request by request, in 64 bits; moved rows have no other value."""
    global own
    if case["op"] in ("fork", "compact"):
        return None
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return (_exact_qk if case["op"] == "qk" else _exact_window)(s, s["case"])


def _exact_qk(s, c):
    n, hk, d, bt = c["rotary"], c["kv_heads"], c["dim"], c["block"]
    angle = s["positions"].double()[:, None, None] * (s["turns"] * (2 * math.pi))
    spin = torch.polar(torch.ones_like(angle), angle)  # a pair as a complex number, times e^(i angle)
    done = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x, w = x.double(), w.double() + c["offset"]
        for step in ("turn", "norm") if c["after"] else ("norm", "turn"):
            if step == "norm":
                x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / d + s["eps"]) * w
            else:
                x = x.clone()
                one, two = (slice(0, n // 2), slice(n // 2, n)) if c["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
                z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * spin
                x[..., one], x[..., two] = z.real, z.imag
        done.append(x)
    tiles = torch.zeros(s["arena"].numel() // (2 * bt * d), bt * d, dtype=torch.float64, device="cuda")
    block, r = s["table"][s["owner"], s["at"] // bt], s["at"] % bt
    place = (r // 8 * 8 * d)[:, None] + s["places"][r % 8]
    for kv, x in enumerate((done[1], s["v"].double())):
        for h in range(hk):
            tiles[((block * 2 + kv) * hk + h)[:, None], place] = x[:, h]
    return {"q": done[0], "cache": tiles.reshape(-1)}


def _exact_window(s, c):
    pairs = sum(_visible(c, p, r)[0] for p, r in zip(_past(c), _rows(c))) * c["q_heads"]
    if pairs * c["dim"] > 1 << 39:
        return None
    hk, group = c["kv_heads"], c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    start = s["src_row"].tolist()
    for b, (past, rows) in enumerate(zip(_past(c), _rows(c))):
        n = past + rows
        blocks = s["table"][b:b + 1, :-(-n // c["block"])]
        keys, values = (_load(s, c, kv, blocks)[0, :, :n].double() for kv in range(2))
        k = torch.arange(n, device="cuda")
        for r0 in range(0, rows, 256):
            p = torch.arange(past + r0, past + min(rows, r0 + 256), device="cuda")[:, None]
            back = p - k
            hidden = back < 0
            if c["window"]:
                hidden |= (back >= c["window"]) & (k >= c["sinks"])
            q = s["q"][start[b] + r0:start[b] + r0 + len(p)].double()
            for h in range(c["q_heads"]):
                x = (q[:, h] @ keys[h // group].T) / math.sqrt(c["dim"])
                x.masked_fill_(hidden, -math.inf)
                out[start[b] + r0:start[b] + r0 + len(p), h] = torch.softmax(x, -1) @ values[h // group]
    return {"out": out}
