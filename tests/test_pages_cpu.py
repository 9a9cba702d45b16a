"""Sequences that share blocks: the host's bookkeeping against a model with a holder count per block (random operations on a
host-only pool), and the argument checks of the calls that fork, own, drop and compact, and of the rotary append with norms."""
import ctypes as C
import math

import numpy as np
import pytest

import ekv

P = 0x10000  # a pointer that is never followed
L = ekv.lib


def pool(**kw):
    cfg = dict(device=-1, dtype=ekv.DTYPE_BF16, block_tokens=16, n_blocks=40, kv_heads=2, head_dim=64, n_layers=2, max_seqs=6,
               max_blocks_per_seq=12)
    cfg.update(kw)
    return ekv.Pool(**cfg)


class Model:
    """Blocks and sequences by their rules: lowest free first, a block is free when nobody holds it."""

    def __init__(self, n_blocks, bt, max_seqs, width):
        self.bt, self.width, self.n_blocks, self.max_seqs = bt, width, n_blocks, max_seqs
        self.seqs = {}

    def holders(self, b):
        return sum(s["blocks"].count(b) for s in self.seqs.values())

    def free(self):
        held = {b for s in self.seqs.values() for b in s["blocks"]}
        return [b for b in range(self.n_blocks) if b not in held]

    def ids(self):
        return [i for i in range(self.max_seqs) if i not in self.seqs]

    def fork(self, parents, tokens):
        tails = sum(t % self.bt != 0 for t in tokens)
        if len(self.ids()) < len(parents) or len(self.free()) < tails:
            return None
        out = []
        for p, t in zip(parents, tokens):
            blocks = self.seqs[p]["blocks"][:t // self.bt]
            if t % self.bt:
                blocks = blocks + [self.free()[0]]
            i = self.ids()[0]
            self.seqs[i] = {"n": t, "blocks": blocks}
            out.append(i)
        return out

    def own(self, s, pos, n):
        q = self.seqs[s]["blocks"]
        if n == 0:
            return True
        at = [i for i in range(pos // self.bt, (pos + n - 1) // self.bt + 1) if self.holders(q[i]) > 1]
        if len(self.free()) < len(at):
            return False
        new = self.free()[:len(at)]
        for i, b in zip(at, new):
            q[i] = b
        return True


@pytest.mark.parametrize("seed", range(6))
def test_shared_blocks_against_the_model(seed):
    rng = np.random.default_rng(seed)
    bt = int(rng.choice([8, 16, 24]))
    p, m = pool(block_tokens=bt, n_blocks=30, max_seqs=7, max_blocks_per_seq=9), Model(30, bt, 7, 9)
    for _ in range(400):
        op = rng.choice(["create", "resize", "fork", "own", "drop", "free", "front"])
        live = list(m.seqs)
        if op == "create":
            if m.ids():
                s = p.seq_create()
                assert s == m.ids()[0]
                m.seqs[s] = {"n": 0, "blocks": []}
            continue
        if not live:
            continue
        s = int(rng.choice(live))
        q = m.seqs[s]
        if op == "resize":
            n = int(rng.integers(0, 9 * bt + 1))
            need = -(-n // bt)
            if need - len(q["blocks"]) > len(m.free()):
                with pytest.raises(ekv.EkvError) as e:
                    p.seq_resize(s, n)
                assert e.value.code == ekv.ERR_POOL_EXHAUSTED
            else:
                p.seq_resize(s, n)
                q["blocks"] = q["blocks"][:need] + m.free()[:max(0, need - len(q["blocks"]))]
                q["n"] = n
        elif op == "fork":
            parents = [int(x) for x in rng.choice(live, size=int(rng.integers(1, 4)))]
            tokens = [int(rng.integers(0, m.seqs[x]["n"] + 1)) for x in parents]
            want = m.fork(parents, tokens)
            if want is None:
                with pytest.raises(ekv.EkvError) as e:
                    p.seq_fork(parents, tokens)
                assert e.value.code == ekv.ERR_POOL_EXHAUSTED
            else:
                assert p.seq_fork(parents, tokens) == want
        elif op == "own":
            reach = len(q["blocks"]) * bt
            pos = int(rng.integers(0, reach + 1))
            n = int(rng.integers(0, reach - pos + 1))
            if m.own(s, pos, n):
                p.seq_own(s, pos, n)
            else:
                with pytest.raises(ekv.EkvError) as e:
                    p.seq_own(s, pos, n)
                assert e.value.code == ekv.ERR_POOL_EXHAUSTED
        elif op == "drop":
            first = int(rng.integers(0, len(q["blocks"]) + 1))
            k = int(rng.integers(0, len(q["blocks"]) - first + 1))
            p.seq_drop_blocks(s, first, k)
            q["n"] -= min(q["n"], (first + k) * bt) - min(q["n"], first * bt)
            q["blocks"] = q["blocks"][:first] + q["blocks"][first + k:]
        elif op == "front":
            k = int(rng.integers(0, len(q["blocks"]) + 1))
            p.seq_evict_front(s, k)
            q["blocks"], q["n"] = q["blocks"][k:], max(0, q["n"] - k * bt)
        else:
            p.seq_free(s)
            del m.seqs[s]
        assert p.info().free_blocks == len(m.free())
        for i, q in m.seqs.items():
            got = p.seq_get(i)
            assert (got.n_tokens, got.blocks) == (q["n"], q["blocks"])


def test_set_blocks_beside_shared_blocks():
    p = pool()
    a = p.seq_create()
    p.seq_set_blocks(a, [5, 6, 7], 40)
    b, = p.seq_fork([a], [32])
    with pytest.raises(ekv.EkvError):  # shared with another sequence only
        p.seq_set_blocks(p.seq_create(), [5], 16)
    p.seq_set_blocks(b, [6, 5], 20)  # its own, in another order
    p.seq_free(a)
    assert p.info().free_blocks == 38
    p.seq_free(b)
    assert p.info().free_blocks == 40


def test_dropped_blocks_and_predicted_tokens():
    p = pool()
    s = p.seq_create()
    p.seq_append_tokens(s, 70)
    p.seq_append_tokens(s, 20, pred=True)
    for first, n in ((4, 1), (3, 2), (5, 1)):
        assert L.ekv_seq_drop_blocks(p.h, s, first, n) == ekv.ERR_UNSUPPORTED
    p.seq_drop_blocks(s, 1, 2)
    assert p.seq_get_pred(s) == (38, 58) and p.seq_get(s).n_tokens == 58
    for first, n in ((-1, 1), (0, -1), (5, 0), (0, 5), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1)):
        assert L.ekv_seq_drop_blocks(p.h, s, first, n) == ekv.ERR_RANGE
    assert L.ekv_seq_drop_blocks(p.h, s + 1, 0, 0) == ekv.ERR_NO_SEQ
    assert L.ekv_seq_drop_blocks(None, s, 0, 0) == ekv.ERR_NO_SEQ


def test_fork_and_own_refusals():
    p = pool()
    s = p.seq_create()
    p.seq_resize(s, 50)
    one = C.c_int32 * 1
    def fork(n=1, parent=s, tokens=50, parents=True, lengths=True, children=True):
        out = one(-7)
        rc = L.ekv_seq_fork(p.h, n, one(parent) if parents else None, one(tokens) if lengths else None, out if children else None, None)
        return rc, out[0]
    assert fork(n=-1)[0] == ekv.ERR_INVALID_ARG
    for kw in (dict(parents=False), dict(lengths=False), dict(children=False)):
        assert fork(**kw)[0] == ekv.ERR_INVALID_ARG, kw
    assert fork(parent=s + 1) == (ekv.ERR_NO_SEQ, -7) and fork(parent=-1)[0] == ekv.ERR_NO_SEQ
    assert fork(tokens=51) == (ekv.ERR_RANGE, -7) and fork(tokens=-1)[0] == ekv.ERR_RANGE
    assert L.ekv_seq_fork(None, 0, None, None, None, None) == ekv.ERR_INVALID_ARG
    assert L.ekv_seq_fork(p.h, 0, None, None, None, None) == ekv.OK
    assert p.info().live_seqs == 1 and p.info().free_blocks == 36
    for args in ((-1, 1), (0, -1), (0, 65), (64, 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert L.ekv_seq_own(p.h, s, *args, None) == ekv.ERR_RANGE, args
    assert L.ekv_seq_own(p.h, s + 1, 0, 0, None) == ekv.ERR_NO_SEQ
    with pytest.raises(ValueError):
        p.seq_fork([s, s], [1])


def test_compact_refusals():
    p = pool()

    def call(**kw):
        c = ekv.CompactParams(0, 2, 3, 0, P, P, P, 40)
        for k, v in kw.items():
            setattr(c, k, v)
        return L.ekv_compact(p.h, C.byref(c), None)

    assert call() == ekv.ERR_UNSUPPORTED  # no device
    assert call(n_batch=0) == ekv.OK and call(slot_stride=0) == ekv.OK
    for kw in (dict(layer0=-1), dict(layer0=1), dict(n_layers=0), dict(n_layers=3), dict(n_batch=-1), dict(slot_stride=-1), dict(seq_ids=None),
               dict(n_keep=None), dict(slots=None), dict(slots=P + 2), dict(n_keep=P + 1), dict(seq_ids=P + 3), dict(layer0=2 ** 31 - 1)):
        assert call(**kw) == ekv.ERR_INVALID_ARG, kw
    assert L.ekv_compact(None, C.byref(ekv.CompactParams()), None) == ekv.ERR_INVALID_ARG
    assert L.ekv_compact(p.h, None, None) == ekv.ERR_INVALID_ARG


def test_norm_rope_append_refusals():
    p, rope = pool(), ekv.Rope(device=-1, rotary_dims=64)

    def call(norm=None, pl=None, layer=0, n=3, seq=P, dst=P, rows=P, src=P, most=5, pos=P, hq=4, q=P, qs=0, qo=P, k=P, v=P, kvs=0):
        nm = ekv.HeadNormConfig(P, P, ekv.DTYPE_BF16, 0, 0.0, 1e-6)
        for key, val in (norm or {}).items():
            setattr(nm, key, val)
        return L.ekv_norm_rope_append((pl or p).h, rope.h, C.byref(nm), layer, n, seq, dst, rows, src, most, pos, hq, q, qs, qo, k, v, kvs, None)

    assert call() == ekv.ERR_UNSUPPORTED  # no device
    assert call(n=0) == ekv.OK and call(most=0) == ekv.OK
    assert call(norm=dict(q_weight=None, k_weight=None)) == ekv.ERR_UNSUPPORTED
    for kw in (dict(layer=2), dict(n=-1), dict(n=65536), dict(most=-1), dict(seq=None), dict(dst=None), dict(rows=None), dict(src=None),
               dict(pos=None), dict(hq=0), dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(q=None, qo=None, k=None, v=None),
               dict(qs=255), dict(qs=260), dict(kvs=127), dict(kvs=132), dict(q=P + 8, qo=P), dict(k=P + 2), dict(qs=512, qo=P),
               dict(norm=dict(eps=-1.0)), dict(norm=dict(eps=math.nan)), dict(norm=dict(eps=math.inf)), dict(norm=dict(weight_offset=math.nan)),
               dict(norm=dict(q_weight=P + 8)), dict(norm=dict(k_weight=P + 4))):
        assert call(**kw) == ekv.ERR_INVALID_ARG, kw
    assert call(norm=dict(weight_dtype=ekv.DTYPE_F16)) == ekv.ERR_UNSUPPORTED
    assert call(pl=pool(head_dim=48)) == ekv.ERR_INVALID_ARG  # more rotated columns than a head has
    assert L.ekv_norm_rope_append(p.h, rope.h, None, 0, 1, P, P, P, P, 1, P, 4, P, 0, P, P, P, 0, None) == ekv.ERR_INVALID_ARG


class NoStream:
    cuda_stream = 0


@pytest.mark.parametrize("how", ["rope", "norm"])
def test_rotary_appends_refuse_other_index_arrays(how):
    """Arrays of another integer type, with gaps, or too short for the requests or rows would be read wrongly, or past their ends."""
    torch = pytest.importorskip("torch")
    p, rope, norm = pool(), ekv.Rope(device=-1, rotary_dims=64), ekv.HeadNorm()
    kv_heads = p.cfg.kv_heads
    q = torch.zeros(9, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(9, kv_heads, 64, dtype=torch.bfloat16)
    good = dict(seq_ids=torch.zeros(3, dtype=torch.int32), dst_pos=torch.zeros(4, dtype=torch.int32), n_rows=torch.zeros(3, dtype=torch.int32),
                src_row=torch.zeros(3, dtype=torch.int32), positions=torch.zeros(9, dtype=torch.int32))

    def call(rows, **kw):
        a = {**good, **kw}
        args = (0, a["seq_ids"], a["dst_pos"], a["n_rows"], a["src_row"], 3, a["positions"])
        if how == "rope":
            p.rope_append(rope, *args, **rows, stream=NoStream)
        else:
            p.norm_rope_append(rope, norm, *args, **rows, stream=NoStream)

    for rows in (dict(q=q, q_out=q), dict(k=k, v=k), dict(q=q, q_out=q, k=k, v=k)):
        for kw in ({}, {name: t.to(torch.uint32) for name, t in good.items()}, dict(positions=torch.zeros(30, dtype=torch.int32)),
                   dict(seq_ids=ekv.DevArray(0x10000, 3), dst_pos=ekv.DevArray(0x10000, 3))):
            with pytest.raises(ekv.EkvError) as e:
                call(rows, **kw)
            assert e.value.code == ekv.ERR_UNSUPPORTED  # no device: the arrays have passed
        append = "k" in rows
        for name in good:
            if name in ("seq_ids", "dst_pos") and not append:
                with pytest.raises(ekv.EkvError) as e:  # not looked at
                    call(rows, **{name: None})
                assert e.value.code == ekv.ERR_UNSUPPORTED
                continue
            n = good[name].numel()
            bad = [torch.zeros(n, dtype=torch.int64), torch.zeros(n), torch.zeros(2 * n, dtype=torch.int32)[::2]]
            if name in ("seq_ids", "dst_pos"):
                bad += [torch.zeros(2, dtype=torch.int32), ekv.DevArray(0x10000, 2)]
            if name == "src_row":
                bad.append(torch.zeros(2, dtype=torch.int32))
            if name == "n_rows":
                bad.append(torch.zeros(5, dtype=torch.int32))  # more requests than the other arrays have
            if name == "positions" and how == "norm":
                bad += [torch.zeros(8, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)]
            for t in bad:
                with pytest.raises(ValueError):
                    call(rows, **{name: t})
        if append:
            with pytest.raises(ekv.EkvError) as e:
                call(rows, seq_ids=None)
            assert e.value.code == ekv.ERR_INVALID_ARG
