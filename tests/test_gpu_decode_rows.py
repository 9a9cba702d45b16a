"""Draft-tree attention around the row counts where its form changes, and the join of many rows' parts. Tolerances are those
of test_gpu_decode.py, whose checks are used."""
import pytest
import torch

import decode_cases as dc
from test_gpu_decode import check_tree, rand, run_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("q8_0", 64), ("q8_0", 128), ("q8_0", 256)])
@pytest.mark.parametrize("T,hq,block", [(16, 1, 8), (17, 1, 24), (8, 4, 128), (11, 3, 40), (64, 1, 16), (13, 5, 24), (32, 4, 64),
                                        (43, 3, 8), (64, 4, 24), (61, 5, 128)])
@pytest.mark.parametrize("cap", [0.0, 12.0])
def test_tree_row_counts(store, dim, T, hq, block, cap):
    lens = [1300, 0, 65, 64, 700]
    c = dc.Cache(lens, 1, dim, store=store, block=block, seed=T)
    q, kd, vd = rand(21, 5, T, hq, dim, scale=2.0), rand(22, 5, T, 1, dim), rand(23, 5, T, 1, dim)
    nodes = [T, T // 2, 1, T - 1, 0]
    up = [dc.tree_words(T, 90 + b) for b in range(5)]
    out, lse, _ = run_tree(c, q, kd, vd, nodes=nodes, up=dc.words(up), cap=cap)
    check_tree(c, q, kd, vd, out, lse, nodes=nodes, up=up, cap=cap)


@pytest.mark.parametrize("store,dim", [("bf16", 48), ("bf16", 64), ("bf16", 128), ("bf16", 256), ("q8_0", 128)])
@pytest.mark.parametrize("T,hq,hk", [(3, 27, 9), (37, 21, 7)])
def test_tree_join_of_many_rows(store, dim, T, hq, hk):
    """Enough rows for the join to take several a warp, row counts that its groups do not divide, f32 outputs."""
    lens = [611, 1200, 0, 64, 900, 333] * 8
    c = dc.Cache(lens, hk, dim, store=store, block=32, seed=5)
    B = len(lens)
    q, kd, vd = rand(31, B, T, hq, dim), rand(32, B, T, hk, dim), rand(33, B, T, hk, dim)
    nodes = [max(0, T - b % 4) for b in range(B)]
    out, lse, _ = run_tree(c, q, kd, vd, nodes=nodes, dtype=torch.float32)
    check_tree(c, q, kd, vd, out, lse, nodes=nodes)


def test_tree_scales_that_are_not_finite_stay_hidden():
    """Rows of an 8-bit cache past the prefix in use hold infinite scales; no row sees them."""
    c = dc.Cache([200, 90], 1, 128, store="q8_0", block=16, seed=2)
    big = torch.full((40, 1, 128), float("inf"), dtype=torch.bfloat16, device="cuda")
    c.pool.append(0, c.seq_ids, dc.ints([160, 50]), dc.ints([40, 40]), dc.ints([0, 0]), 40, big, big)
    q, kd, vd = rand(41, 2, 20, 2, 128), rand(42, 2, 20, 1, 128), rand(43, 2, 20, 1, 128)
    for use in ([160, 50], [131, 1]):
        out, lse, _ = run_tree(c, q, kd, vd, prefix_len=use)
        check_tree(c, q, kd, vd, out, lse, prefix_len=use)


@pytest.mark.parametrize("rotary", [2, 18, 34, 66, 126, 64])
def test_rope_in_place_is_the_same(rotary):
    """Turning q where it lies gives the bits of turning it elsewhere, in the odd split form too."""
    import ekv
    c = dc.Cache([40, 9], 2, 128, seed=1)
    rope = ekv.Rope(rotary_dims=rotary)
    q = rand(51, 49, 6, 128)
    pos = dc.ints(list(range(100, 149)))
    args = (None, None, dc.ints([40, 9]), dc.ints([0, 40]), 40, pos)
    out = torch.empty_like(q)
    c.pool.rope_append(rope, 0, *args, q=q, q_out=out)
    c.pool.rope_append(rope, 0, *args, q=q, q_out=q)
    assert torch.equal(q.view(torch.int16), out.view(torch.int16)) and c.pool.status() == 0
