"""Q8_0 pools keep what is appended at every head_dim, also where a row is not a power of two of 16-byte units."""
import pytest
import torch

import ekv
import oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_q8_append_gather_every_head_dim(dim):
    rows, heads = 37, 2
    pool = ekv.Pool(dtype=ekv.DTYPE_Q8_0, block_tokens=16, n_blocks=4, kv_heads=heads, head_dim=dim, max_seqs=1,
                    max_blocks_per_seq=4)
    s = pool.seq_create()
    pool.seq_resize(s, rows)
    pool.sync()
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randn(rows, heads, dim, generator=g).bfloat16() for _ in range(2))
    one = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    pool.append(0, one(s), one(0), one(rows), one(0), rows, k.cuda(), v.cuda())
    out = [torch.zeros(rows, heads, dim, device="cuda") for _ in range(2)]
    pool.gather(0, s, 0, rows, ekv.GATHER_F32, *out)
    torch.cuda.synchronize()
    assert pool.status() == 0
    for x, y in zip((k, v), out):
        want = oracle.dequantize_q8_0(oracle.quantize_q8_0(x.float().numpy().reshape(rows * heads, dim)))
        assert torch.equal(y.cpu().reshape(rows * heads, dim), torch.from_numpy(want.copy()).reshape(rows * heads, dim))
