"""The e4m3 kernels where their pipelines run: tiles that many CTAs share, and
CTAs with many steps and several tiles, against 64-bit formulas with the error
bounds derived in tests/fp8_reference.py."""
from __future__ import annotations

import pytest
import torch

from dsv4_carve_b200 import moe
from dsv4_carve_b200 import vllm_exl3_c as ext
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


# ------------------------------------------------------------------ many steps a CTA
def _weight(shape, seed, cuda):
    """R.e4m3_weight made on the GPU, for large ones."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    q = torch.empty(shape, dtype=R.F8, device=cuda)
    for part in q.view(-1, shape[-1]).split(4096):
        part.copy_((torch.randn(part.shape, generator=g, device=cuda) * 109.0).clamp_(-448, 448))
    s = 0.5 + torch.rand((*shape[:-2], R.groups(shape[-2]), R.groups(shape[-1])), generator=g, device=cuda)
    return q, s * (0.02 / 109.0)


def _sms(cuda):
    return torch.cuda.get_device_properties(cuda).multi_processor_count


E40, H40, I40 = 40, 1024, 1024


@pytest.fixture(scope="module")
def layer40(cuda):
    return (*_weight((E40, 2 * I40, H40), 1, cuda), *_weight((E40, H40, I40), 2, cuda))


def _spread_route(T, topk, seed, cuda):
    """Every expert in turn, in a random order a round, so that as many as fit are active."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.cat([torch.randperm(E40, generator=g) for _ in range(-(-T * topk // E40))])[: T * topk]
    return flat.view(T, topk).to(torch.int32).to(cuda), torch.softmax(torch.randn((T, topk), generator=g), dim=1).to(cuda)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("T,topk", [(4, 10), (5, 8), (16, 8), (16, 16), (17, 15), (32, 8), (33, 7), (64, 4)])
def test_moe_many_steps_a_cta(cuda, layer40, T, topk, pow2):
    """Kernel 1's CTAs go through two whole tiles and more, both rings are refilled
    and TMEM's and the factors' buffers reused, for each number of columns."""
    ids, rw = _spread_route(T, topk, T, cuda)
    nt = 16 if T <= 16 else 32 if T <= 32 else 64
    groups = sum(-(-int(n) // nt) for n in ids.flatten().bincount() if n)
    steps = groups * (I40 // 128) * (H40 // 128) // _sms(cuda)          # of either kernel
    assert steps >= 2 * (H40 // 128) and steps >= 12                     # whole tiles; more than a ring's blocks
    x = R.activations(T, H40, T, torch.bfloat16, cuda)
    state = moe.Fp8MoeState(*layer40, pow2_scale=pow2)
    y = moe.apply_moe(x, ids, rw, state, None, 10.0, out_dtype=torch.float32)
    want, allowed = R.moe(x, *layer40, ids, rw, 10.0, pow2)
    assert R.worst(y, want, allowed) <= 1.0
    for _ in range(5):
        assert torch.equal(moe.apply_moe(x, ids, rw, state, None, 10.0, out_dtype=torch.float32), y)


@pytest.mark.parametrize("T", [4, 24, 64])
def test_moe_crowded_experts(cuda, layer40, T):
    """A few experts with most tokens beside many with one, slots of other ranks, an expert listed twice."""
    ids, rw = _spread_route(T, 4, 9, cuda)
    ids[::2, 0] = 7
    ids[1::3, 1] = 7
    ids[::5, 2] = -1
    ids[2] = 11
    y = moe.apply_moe(R.activations(T, H40, 3, torch.float16, cuda), ids, rw, moe.Fp8MoeState(*layer40), None, 10.0,
                      out_dtype=torch.float32)
    want, allowed = R.moe(R.activations(T, H40, 3, torch.float16, cuda), *layer40, ids, rw, 10.0)
    assert R.worst(y, want, allowed) <= 1.0


@pytest.mark.parametrize("E,H,I,T,topk", [(16, 4096, 2048, 4, 4), (1, 16384, 8192, 2, 1), (2, 16384, 128, 6, 2), (2, 128, 8192, 40, 2)])
def test_moe_configured_and_largest_sizes(cuda, E, H, I, T, topk):
    layer = (*_weight((E, 2 * I, H), 3, cuda), *_weight((E, H, I), 4, cuda))
    ids, rw = _route(T, E, topk, T, cuda)
    x = R.activations(T, H, T, torch.bfloat16, cuda)
    y = moe.apply_moe(x, ids, rw, moe.Fp8MoeState(*layer), None, 10.0, out_dtype=torch.float32)
    want, allowed = R.moe(x, *layer, ids, rw, 10.0)
    assert R.worst(y, want, allowed) <= 1.0


@pytest.fixture(scope="module")
def square(cuda):
    return _weight((8192, 8192), 5, cuda)


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 32, 47, 64, 100, 128])
def test_linear_few_rows_many_steps(cuda, square, rows):
    """64 tiles of 64 groups: a CTA has more steps than its ring has stages."""
    split = 8
    while split > 1 and 64 * split > 2 * _sms(cuda):                     # CTAs that may split k, at most
        split //= 2
    assert 64 // split > 12                                              # 12: no ring has more stages
    x = R.activations(rows, 8192, rows, torch.bfloat16, cuda)
    y = ext.fp8_linear(x, *square, out_dtype=torch.float32)
    want, allowed = R.linear(R.rows_dequant(x), R.weight(*square))
    assert R.worst(y, want, allowed) <= 1.0
    for _ in range(5):
        assert torch.equal(ext.fp8_linear(x, *square, out_dtype=torch.float32), y)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("k", [100, 640, 2000])
@pytest.mark.parametrize("n", [4096, 4099, 2304, 2301])
def test_linear_many_rows_several_tiles_a_pair(cuda, n, k, out):
    """More tiles than pairs of CTAs, 256 and 128 wide, so that the ring, the sums'
    buffers and the output's go on from one tile to the next; rows of y on 16-byte
    boundaries, which leave by TMA, and off them."""
    rows = 2310
    assert -(-rows // 256) * -(-n // 256) > _sms(cuda) // 2
    w, ws = _weight((n, -(-k // 16) * 16), n + k, cuda)
    w = w[:, :k]
    x = R.activations(rows, k, k, torch.bfloat16, cuda)
    b = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(out).to(cuda)
    y = ext.fp8_linear(x, w, ws, bias=b, out_dtype=out)
    want, allowed = R.linear(R.rows_dequant(x), R.weight(w, ws), b, out)
    assert R.worst(y, want, allowed) <= 1.0
    for _ in range(3):
        assert torch.equal(ext.fp8_linear(x, w, ws, bias=b, out_dtype=out), y)
    assert ext.fp8_status(cuda) == 0


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n", [(129, 1335), (200, 1), (300, 131), (513, 257)])
def test_linear_rows_of_y_off_16_bytes(cuda, rows, n, out):
    w, ws = R.e4m3_weight((n, 400), 6, cuda)
    x = R.activations(rows, 400, 7, torch.float16, cuda)
    want, allowed = R.linear(R.rows_dequant(x), R.weight(w, ws), None, out)
    assert R.worst(ext.fp8_linear(x, w, ws, out_dtype=out), want, allowed) <= 1.0
