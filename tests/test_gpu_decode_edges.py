"""Decoding operators where inputs are not finite, and what rounding may not cost. Shapes, checks and tolerances not derived
here are those of test_gpu_decode.py."""
import pytest
import torch

import decode_cases as dc
from test_gpu_decode import check_tree, rand, run_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("T,hq", [(1, 1), (1, 8), (2, 8), (3, 6), (9, 8), (32, 8)])
@pytest.mark.parametrize("cap", [0.0, 6.0])
def test_tree_weighted_mean_of_equal_values(dim, T, hq, cap):
    """Where every key holds the same 8-bit row, the output is that row whatever the probabilities. Tolerance: a
    probability as two bf16 parts is off by 2^-17, its product with the value's scale (or the value as two parts) by another
    2^-17, the sums of up to 200 terms by 200 * 2^-24; the rest of 2^-14 is room."""
    lens = [1, 2, 17, 200]
    c = dc.Cache(lens, 1, dim, store="q8_0", seed=3)
    row = rand(71, 1, 1, dim)
    k = rand(72, 200, 1, dim)
    for b, n in enumerate(lens):
        c.pool.append(0, dc.ints([c.seqs[b]]), dc.ints([0]), dc.ints([n]), dc.ints([0]), n, k[:n].contiguous(), row.expand(n, 1, dim).contiguous())
    q, kd, vd = rand(73, 4, T, hq, dim), rand(74, 4, T, 1, dim), rand(75, 4, T, 1, dim)
    up = [[0] * T for _ in range(4)]
    out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), cap=cap, dtype=torch.float32)
    want = c.rows(0)[1][0, 0].double()
    assert ((out.double() - want).abs() <= 2 ** -14 * want.abs()).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("T,hq", [(1, 4), (2, 8), (9, 4), (32, 4)])
def test_tree_values_beyond_their_scale(dim, T, hq):
    """8-bit values whose f16 scale overflowed are infinite (and NaN where the 8 bits are 0): so are the outputs."""
    c = dc.Cache([40, 300], 1, dim, store="q8_0", seed=4)
    big = torch.ones(1, 1, dim, dtype=torch.bfloat16, device="cuda")
    big[0, 0, 5], big[0, 0, 32:64] = 1e8, -1e8
    c.pool.append(0, c.seq_ids, dc.ints([7, 290]), dc.ints([1, 1]), dc.ints([0, 0]), 1, torch.ones_like(big), big)
    q, kd, vd = rand(81, 2, T, hq, dim), rand(82, 2, T, 1, dim), rand(83, 2, T, 1, dim)
    out, lse, _ = run_tree(c, q, kd, vd)
    assert torch.isinf(out[..., 32:64]).all() and torch.isnan(out[..., 6]).all()
    check_tree(c, q, kd, vd, out, lse)
