"""Packed attention with eight heads a tile (groups with a factor of eight and no more), at the lengths of test_attn_packed_gpu.py."""
import pytest
import torch

import test_attn_packed_gpu as packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", packed.TYPES)
@pytest.mark.parametrize("heads,kv", [(8, 1), (24, 1), (16, 2)])
@pytest.mark.parametrize("lens", packed.LENS)
def test_packed_eight_heads_a_tile(ops, cuda, dtype, lens, heads, kv):
    q, k, v = packed._rows(*lens, heads, kv, dtype, cuda, seed=heads + len(lens[0]))
    ws = ops.Workspace()
    args = (q, k, v, packed._cu(lens[0], cuda), packed._cu(lens[1], cuda), ws)
    got = ops.attn_packed(*args)
    ws.check()
    packed._check(got, q, k, v, *lens)
    assert torch.equal(ops.attn_packed(*args), got)
    ws.check()
