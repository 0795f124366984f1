"""The e4m3 kernels where their pipelines run: tiles that many CTAs share, and
CTAs with many steps and several tiles, against 64-bit formulas with the error
bounds derived in tests/fp8_reference.py."""
from __future__ import annotations

import pytest
import torch

from dsv4_carve_b200 import moe
from tests import fp8_reference as R

pytestmark = pytest.mark.gpu


def _layer(cuda, E, H, I, seed):
    return (*R.e4m3_weight((E, 2 * I, H), 100 + seed, cuda), *R.e4m3_weight((E, H, I), 200 + seed, cuda))


def _route(T, E, topk, seed, cuda):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)]).to(torch.int32)
    return ids.to(cuda), torch.softmax(torch.randn((T, topk), generator=g), dim=1).to(cuda)


@pytest.mark.parametrize("T", [1, 4, 6])
def test_moe_tiles_shared_by_many_ctas(cuda, T):
    """16 and more output tiles of 32 blocks over all CTAs: each tile is the sum of
    several CTAs' parts, and the same bits every time."""
    layer = _layer(cuda, 16, 4096, 256, T)
    state = moe.Fp8MoeState(*layer)
    ids, rw = _route(T, 16, 8, T, cuda)
    x = R.activations(T, 4096, T, torch.bfloat16, cuda)
    y = moe.apply_moe(x, ids, rw, state, None, 10.0, out_dtype=torch.float32)
    want, allowed = R.moe(x, *layer, ids, rw, 10.0)
    assert R.worst(y, want, allowed) <= 1.0
    flush = torch.empty(64 << 20, device=cuda)
    for i in range(40):
        if i % 4 == 0:
            flush.fill_(i)
        assert torch.equal(moe.apply_moe(x, ids, rw, state, None, 10.0, out_dtype=torch.float32), y)
