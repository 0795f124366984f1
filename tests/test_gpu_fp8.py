"""The e4m3 operators on the GPU: quantiser (bit for bit), block-scaled linear
and the routed-MoE layer over e4m3 experts, against 64-bit formulas with the
error bounds derived in tests/fp8_reference.py."""
from __future__ import annotations

import pytest
import torch

from dsv4_carve_b200 import moe
from dsv4_carve_b200 import vllm_exl3_c as ext
from dsv4_carve_b200.linear import LinearFP8
from tests import fp8_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _same(q, want):
    got = q.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# ------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 257), (130, 520), (128, 1000), (65, 4096), (9, 1036), (300, 4008)])
def test_quantize_bits(cuda, rows, cols, block_rows, dtype, pow2):
    x = R.activations(rows, cols, rows + cols, dtype, cuda)
    q, s = ext.fp8_quantize(x, block_rows=block_rows, pow2_scale=pow2)
    wq, ws = R.quantize(x, block_rows, pow2)
    assert torch.equal(s.double(), ws)
    _same(q, wq)


@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_midpoints_and_borders(cuda, pow2):
    """Values at and next to the midpoints of two e4m3 values, for scales that
    are and are not fp32 divisors of them, and amax at and next to 448 * 2^e."""
    mids = torch.tensor([(m + 0.5) / 8 * 2.0 ** -6 for m in range(8)] +
                        [(1 + (m + 0.5) / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-2], dtype=torch.float64)
    rows = []
    for amax in (448.0, 448.0 * 0.7, 448.0 * 1.0000001, 447.99997, 448.00003, 1.0, 3.0, 1e-30, 2e30, 7e-36, 1e-37, 3.3e38,
                 1.3e-15, 2.7e33):
        s = float(R.scale_of(torch.tensor([amax], dtype=torch.float64).float().double(), pow2))
        v = (mids * s).float()
        v = torch.cat([v, torch.nextafter(v, torch.zeros_like(v)), torch.nextafter(v, torch.full_like(v, 1e38)), -v])
        v = v[v.abs() <= amax]
        v = torch.cat([v, torch.zeros((-v.numel()) % 127)]).view(-1, 127)
        rows.append(torch.cat([torch.full((v.shape[0], 1), amax), v], dim=1))
    x = torch.cat(rows).to(cuda)
    q, s = ext.fp8_quantize(x, pow2_scale=pow2)
    wq, ws = R.quantize(x, 1, pow2)
    assert torch.equal(s.double(), ws)
    _same(q, wq)


def test_quantize_zeros_tiny_and_non_finite(cuda):
    x = torch.zeros((6, 256), device=cuda)
    x[1, 3] = 1e-42
    x[2, 5] = float("nan")
    x[3, 130] = float("inf")
    x[4, 7] = -3.0e38
    q, s = ext.fp8_quantize(x)
    wq, ws = R.quantize(x)
    assert torch.equal(torch.nan_to_num(s.double(), nan=-1.0), torch.nan_to_num(ws, nan=-1.0))
    assert torch.isnan(s[2, 0]) and torch.isfinite(s[2, 1]) and torch.isinf(s[3, 1])
    _same(q, wq)
    assert float(s[0, 0]) == 2.0 ** -126 and not q[0].double().any()


def test_quantize_strides_offsets_and_shapes(cuda):
    base = R.activations(9, 700, 3, torch.bfloat16, cuda)
    for x in (base[:, 5:261], base[1:, 8:392], base[::2, :256], base[:, ::2], base[:, 1:2]):
        q, s = ext.fp8_quantize(x)
        wq, ws = R.quantize(x.contiguous())
        assert torch.equal(s.double(), ws)
        _same(q, wq)
    q, s = ext.fp8_quantize(base.view(3, 3, 700))
    assert q.shape == (3, 3, 700) and s.shape == (3, 3, 6)
    q, s = ext.fp8_quantize(base[:0])
    assert q.shape == (0, 700) and s.shape == (0, 6)
    q1, s1 = ext.fp8_quantize(base[0, :256].expand(4, 256))
    assert torch.equal(q1[0].view(torch.uint8), q1[3].view(torch.uint8)) and torch.equal(s1[0], s1[3])


# ------------------------------------------------------------------ linear
def _linear(cuda, rows, n, k, dtype, out, pow2=False, bias=False, seed=0):
    w, ws = R.e4m3_weight((n, k), seed + n, cuda)
    x = R.activations(rows, k, seed + rows, dtype, cuda)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(out).to(cuda) if bias else None
    y = LinearFP8(w, ws, bias=b, pow2_scale=pow2).forward(x, {}, out_dtype=out)
    want, allowed = R.linear(R.rows_dequant(x, pow2), R.weight(w, ws), b, out)
    assert y.shape == (rows, n) and y.dtype == out
    return R.worst(y, want, allowed)


@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 32, 33, 64, 65, 130, 200, 257, 300, 513])
@pytest.mark.parametrize("n,k", [(128, 128), (576, 1040), (1336, 2048), (100, 4096), (1, 144)])
def test_linear_rows_and_ragged(cuda, rows, n, k):
    assert _linear(cuda, rows, n, k, torch.bfloat16, torch.float32) <= 1.0


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 140])
def test_linear_types(cuda, rows, dtype, out):
    assert _linear(cuda, rows, 384, 640, dtype, out, pow2=True, bias=True) <= 1.0


@pytest.mark.parametrize("rows,n,k", [(1, 4096, 4096), (8, 1536, 4096), (100, 4096, 1536), (512, 4096, 4096),
                                      (4, 256, 16384), (700, 2048, 4096)])
def test_linear_configured_sizes(cuda, rows, n, k):
    assert _linear(cuda, rows, n, k, torch.bfloat16, torch.bfloat16) <= 1.0


@pytest.mark.parametrize("k", [1, 16, 100, 127, 129, 1000])
@pytest.mark.parametrize("rows", [2, 150])
def test_linear_any_k(cuda, rows, k):
    """k that is no multiple of 16: LinearFP8 lays the weight's rows out on 16-byte boundaries."""
    assert _linear(cuda, rows, 200, k, torch.float16, torch.float32) <= 1.0


@pytest.mark.parametrize("rows", [1, 6, 20, 129, 400])
def test_linear_prequantised(cuda, rows):
    """An e4m3 x with its scales gives what quantising inside the call gives."""
    w, ws = R.e4m3_weight((512, 1040), 5, cuda)
    x = R.activations(rows, 1040, 6, torch.bfloat16, cuda)
    q, s = ext.fp8_quantize(x)
    a = ext.fp8_linear(q, w, ws, x_scale=s, out_dtype=torch.float32)
    b = ext.fp8_linear(x, w, ws, out_dtype=torch.float32)
    assert torch.equal(a, b)
    assert ext.fp8_linear(q, w, ws, x_scale=s).dtype == torch.bfloat16


def test_linear_weight_from_quantiser(cuda):
    w = (torch.randn(300, 512, generator=torch.Generator().manual_seed(1)) * 0.05).to(cuda)
    lin = LinearFP8.from_weight(w.bfloat16(), out_dtype=torch.float32)
    x = R.activations(4, 512, 2, torch.bfloat16, cuda)
    want, allowed = R.linear(R.rows_dequant(x), R.weight(lin.weight, lin.weight_scale))
    assert R.worst(lin.forward(x), want, allowed) <= 1.0
    # against the unquantised product: e4m3 operands are off by at most 2^-4 each, relative to normal
    # values, so a product by 2^-3 + 2^-8; over 512 terms the row's relative error is far below that
    full = x.double() @ w.double().t()
    assert float((lin.forward(x).double() - full).norm() / full.norm()) < 2.0 ** -3


@pytest.mark.parametrize("rows", [3, 200])
def test_linear_strided_x_and_weight(cuda, rows):
    """Row views at odd offsets, leading batch dimensions, a weight inside a wider one."""
    w, ws = R.e4m3_weight((256, 640), 7, cuda)
    wide = torch.zeros((256, 1024), dtype=torch.uint8, device=cuda).view(R.F8)
    wide[:, 128:768] = w
    big = R.activations(rows, 900, 8, torch.bfloat16, cuda)
    for off in (0, 3, 4, 8):
        x = big[:, off:off + 640]
        want, allowed = R.linear(R.rows_dequant(x.contiguous()), R.weight(w, ws))
        assert R.worst(ext.fp8_linear(x, w, ws, out_dtype=torch.float32), want, allowed) <= 1.0
        assert R.worst(ext.fp8_linear(x, wide[:, 128:768], ws, out_dtype=torch.float32), want, allowed) <= 1.0
    x = big[:, :640].contiguous()
    y = ext.fp8_linear(x.view(1, rows, 640), w, ws)
    assert y.shape == (1, rows, 256) and torch.equal(y[0], ext.fp8_linear(x, w, ws))
    assert ext.fp8_linear(x[:0], w, ws).shape == (0, 256)
    assert torch.equal(ext.fp8_linear(x[0], w, ws), ext.fp8_linear(x[:1], w, ws)[0])


@pytest.mark.parametrize("rows", [4, 260])
def test_linear_non_finite_rows_stay_apart(cuda, rows):
    w, ws = R.e4m3_weight((256, 512), 9, cuda)
    x = R.activations(rows, 512, 10, torch.bfloat16, cuda)
    clean = ext.fp8_linear(x, w, ws)
    bad = x.clone()
    bad[1, 77] = float("nan")
    bad[rows - 1, 300] = float("inf")
    y = ext.fp8_linear(bad, w, ws)
    keep = [r for r in range(rows) if r not in (1, rows - 1)]
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[1]).all() and torch.isnan(y[rows - 1]).all()


@pytest.mark.parametrize("rows", [2, 50, 300])
def test_linear_deterministic_and_status(cuda, rows):
    w, ws = R.e4m3_weight((1536, 4096), 11, cuda)
    x = R.activations(rows, 4096, 12, torch.bfloat16, cuda)
    a = ext.fp8_linear(x, w, ws, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(ext.fp8_linear(x, w, ws, out_dtype=torch.float32), a)
    assert ext.fp8_status(cuda) == 0


# ------------------------------------------------------------------ MoE
def _layer(cuda, E, H, I, seed=0):
    w13, s13 = R.e4m3_weight((E, 2 * I, H), 100 + seed, cuda)
    w2, s2 = R.e4m3_weight((E, H, I), 200 + seed, cuda)
    return w13, s13, w2, s2


def _route(T, E, topk, seed, cuda, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)]).to(dtype)
    return ids.to(cuda), torch.softmax(torch.randn((T, topk), generator=g), dim=1).to(cuda)


def _moe(cuda, layer, x, ids, rw, limit=10.0, out_dtype=torch.float32, pow2=False, expert_map=None, local=None):
    state = moe.Fp8MoeState(*layer, pow2_scale=pow2)
    y = moe.apply_moe(x, ids, rw, state, expert_map, limit, out_dtype=out_dtype)
    want, allowed = R.moe(x, *layer, ids if local is None else local, rw, limit, pow2, out_dtype)
    return R.worst(y, want, allowed)


@pytest.mark.parametrize("T,E,topk,H,I", [
    (1, 4, 1, 128, 128), (1, 8, 8, 512, 256), (3, 16, 4, 1024, 384), (4, 32, 8, 640, 512), (16, 4, 2, 256, 128),
    (17, 8, 2, 384, 256), (32, 16, 8, 512, 128), (33, 4, 4, 256, 256), (64, 3, 3, 384, 128), (2, 300, 6, 256, 128)])
def test_moe_shapes(cuda, T, E, topk, H, I):
    layer = _layer(cuda, E, H, I)
    ids, rw = _route(T, E, topk, T + E, cuda)
    assert _moe(cuda, layer, R.activations(T, H, T, torch.bfloat16, cuda), ids, rw) <= 1.0


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_moe_types(cuda, dtype, out):
    layer = _layer(cuda, 6, 384, 256, 1)
    ids, rw = _route(5, 6, 3, 1, cuda, torch.int64)
    assert _moe(cuda, layer, R.activations(5, 384, 2, dtype, cuda), ids, rw.to(dtype), out_dtype=out, pow2=True) <= 1.0


def test_moe_routes(cuda):
    """Invalid ids, a row without a valid slot, an expert listed twice, one expert for all, the clamp."""
    layer = _layer(cuda, 8, 512, 256, 2)
    x = R.activations(6, 512, 3, torch.bfloat16, cuda)
    ids, rw = _route(6, 8, 4, 3, cuda)
    ids[0] = torch.tensor([-1, 8, -5, 1000], dtype=torch.int32)
    ids[1] = torch.tensor([3, 3, -1, 3], dtype=torch.int32)
    rw[0] = float("nan")
    rw[1, 2] = float("inf")
    state = moe.Fp8MoeState(*layer)
    y = moe.apply_moe(x, ids, rw, state, None, 10.0, out_dtype=torch.float32)
    assert not y[0].any()
    want, allowed = R.moe(x, *layer, ids, rw, 10.0)
    assert R.worst(y, want, allowed) <= 1.0
    one = torch.full((6, 4), 5, dtype=torch.int32, device=cuda)
    assert _moe(cuda, layer, x, one, torch.rand((6, 4), device=cuda)) <= 1.0
    assert _moe(cuda, layer, x * 4, _route(6, 8, 4, 3, cuda)[0], torch.rand((6, 4), device=cuda), limit=0.5) <= 1.0
    none = torch.full((6, 4), -1, dtype=torch.int32, device=cuda)
    assert not moe.apply_moe(x, none, rw, state, None, 10.0).any()


def test_moe_one_expert_many_slots(cuda):
    """More pairs of one expert than a group holds: the expert's weights run more than once."""
    layer = _layer(cuda, 2, 256, 128, 3)
    for T, topk in ((16, 16), (12, 5), (32, 8)):
        ids = torch.ones((T, topk), dtype=torch.int32, device=cuda)
        ids[0, 0] = 0
        rw = torch.rand((T, topk), device=cuda)
        assert _moe(cuda, layer, R.activations(T, 256, T, torch.float16, cuda), ids, rw) <= 1.0


def test_moe_expert_map(cuda):
    layer = _layer(cuda, 4, 256, 256, 4)
    emap = torch.tensor([-1, 2, 0, -1, 3, 1, 9], dtype=torch.int64, device=cuda)     # 9: past the local experts
    ids = torch.tensor([[0, 1, 2], [6, 4, 5], [3, 0, 7], [2, 2, -1]], dtype=torch.int64, device=cuda)
    local = [[int(emap[i]) if 0 <= i < 7 else -1 for i in row] for row in ids.tolist()]
    rw = torch.rand((4, 3), device=cuda)
    x = R.activations(4, 256, 5, torch.bfloat16, cuda)
    assert _moe(cuda, layer, x, ids, rw, expert_map=emap, local=torch.tensor(local)) <= 1.0


def test_moe_non_finite_tokens_stay_apart(cuda):
    layer = _layer(cuda, 4, 256, 256, 5)
    ids, rw = _route(5, 4, 2, 7, cuda)
    x = R.activations(5, 256, 8, torch.bfloat16, cuda)
    state = moe.Fp8MoeState(*layer)
    clean = moe.apply_moe(x, ids, rw, state, None, 10.0)
    bad = x.clone()
    bad[2, 9] = float("nan")
    y = moe.apply_moe(bad, ids, rw, state, None, 10.0)
    keep = [0, 1, 3, 4]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[2]).all()


@pytest.mark.parametrize("T", [1, 5, 20])
def test_moe_prequantised(cuda, T):
    """An e4m3 x with its scales gives what quantising inside the call gives."""
    layer = _layer(cuda, 8, 512, 256, 12)
    ids, rw = _route(T, 8, 3, T, cuda)
    x = R.activations(T, 512, T, torch.bfloat16, cuda)
    scratch = torch.zeros(ext.fp8_moe_scratch_bytes(T, 3, 512, 256), dtype=torch.uint8, device=cuda)
    q, s = ext.fp8_quantize(x)
    a = ext.fp8_moe_decode(q, torch.empty_like(x), *layer, ids, rw, 10.0, scratch, x_scale=s)
    b = ext.fp8_moe_decode(x, torch.empty_like(x), *layer, ids, rw, 10.0, scratch)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 4])
def test_moe_few_tokens_quantised_inside(cuda, T, dtype):
    """Up to four tokens are quantised by the experts' kernel: the bits of a call on
    an e4m3 x, from a start off 16 bytes too, on either side of its width limit."""
    for H, I, E in ((128, 128, 3), (640, 384, 8), (4096, 128, 4), (4224, 128, 4)):
        layer = _layer(cuda, E, H, I, 13)
        ids, rw = _route(T, E, 3, T, cuda)
        flat = R.activations(1, T * H + 1, T, dtype, cuda).view(-1)
        for x in (flat[:-1].view(T, H), flat[1:].view(T, H)):
            for pow2 in (False, True):
                scratch = torch.zeros(ext.fp8_moe_scratch_bytes(T, 3, H, I), dtype=torch.uint8, device=cuda)
                q, s = ext.fp8_quantize(x, pow2_scale=pow2)
                a = ext.fp8_moe_decode(q, torch.empty_like(x), *layer, ids, rw, 10.0, scratch, x_scale=s, pow2_scale=pow2)
                b = ext.fp8_moe_decode(x, torch.empty_like(x), *layer, ids, rw, 10.0, scratch, pow2_scale=pow2)
                assert torch.equal(a, b)


def test_moe_many_rows_in_pieces(cuda):
    layer = _layer(cuda, 4, 256, 128, 6)
    ids, rw = _route(150, 4, 2, 9, cuda)
    assert _moe(cuda, layer, R.activations(150, 256, 9, torch.bfloat16, cuda), ids, rw) <= 1.0


def test_moe_repeats_scratch_and_status(cuda):
    """The same bits every time, on a scratch that larger, smaller and other
    geometries use in turn and that starts as NaN behind its control words."""
    ctrl = 131072
    need = max(ext.fp8_moe_scratch_bytes(32, 8, 512, 256), ext.fp8_moe_scratch_bytes(4, 2, 256, 512))
    scratch = torch.full((need,), 255, dtype=torch.uint8, device=cuda)
    scratch[:ctrl] = 0
    a, b = _layer(cuda, 8, 512, 256, 7), _layer(cuda, 4, 256, 512, 8)
    cases = []
    for layer, T, topk, E, H in ((a, 32, 8, 8, 512), (b, 4, 2, 4, 256), (a, 1, 4, 8, 512)):
        ids, rw = _route(T, E, topk, T, cuda)
        cases.append((layer, R.activations(T, H, T, torch.bfloat16, cuda), ids, rw))
    first = []
    for round_ in range(4):
        for i, (layer, x, ids, rw) in enumerate(cases):
            y = ext.fp8_moe_decode(x, torch.empty_like(x), *layer, ids, rw, 10.0, scratch, check_status=True)
            if round_ == 0:
                first.append(y)
            assert torch.equal(y, first[i])
    assert ext.lna2_moe_status(scratch) == 0


# ------------------------------------------------------------------ together, streams, graphs
def test_a_block_as_a_decoder_runs_it(cuda):
    """Projection, routed experts, shared expert and their sum for a few tokens, then for a longer prompt."""
    H, I, E = 512, 256, 8
    proj = LinearFP8(*R.e4m3_weight((H, H), 20, cuda), out_dtype=torch.bfloat16)
    up = LinearFP8(*R.e4m3_weight((2 * I, H), 21, cuda), out_dtype=torch.float32)
    down = LinearFP8(*R.e4m3_weight((H, I), 22, cuda), out_dtype=torch.bfloat16)
    layer = _layer(cuda, E, H, I, 9)
    state = moe.Fp8MoeState(*layer)
    for T in (3, 100):
        x = R.activations(T, H, T, torch.bfloat16, cuda)
        ids, rw = _route(T, E, 2, T, cuda)
        h = proj.forward(x)
        g, u = up.forward(h).chunk(2, dim=1)
        mid = (torch.nn.functional.silu(g) * u).bfloat16()
        y = moe.apply_moe(h, ids, rw, state, None, 10.0) + down.forward(mid)
        want_h, ah = R.linear(R.rows_dequant(x), R.weight(proj.weight, proj.weight_scale), None, torch.bfloat16)
        assert R.worst(h, want_h, ah) <= 1.0
        wm, am = R.moe(h, *layer, ids, rw, 10.0, False, torch.bfloat16)
        wd, ad = R.linear(R.rows_dequant(mid), R.weight(down.weight, down.weight_scale), None, torch.bfloat16)
        assert R.worst(y, wm + wd, am + ad + 2.0 ** -8 * (wm + wd).abs() + 2.0 ** -7 * (am + ad)) <= 1.0


def test_two_streams_at_once(cuda):
    w, ws = R.e4m3_weight((1024, 2048), 30, cuda)
    layer = _layer(cuda, 8, 512, 256, 10)
    state = moe.Fp8MoeState(*layer)
    ids, rw = _route(8, 8, 4, 5, cuda)
    xl, xm = R.activations(300, 2048, 31, torch.bfloat16, cuda), R.activations(8, 512, 32, torch.bfloat16, cuda)
    want_l, want_m = ext.fp8_linear(xl, w, ws), moe.apply_moe(xm, ids, rw, state, None, 10.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ext.fp8_linear(xl, w, ws), moe.apply_moe(xm, ids, rw, state, None, 10.0)))
    torch.cuda.synchronize()
    assert all(torch.equal(l, want_l) and torch.equal(m, want_m) for l, m in got)


def test_captured_and_replayed_side_by_side(cuda):
    """Two graphs captured one after another, replayed at once on two streams with inputs changed in between."""
    w, ws = R.e4m3_weight((512, 1024), 40, cuda)
    layer = _layer(cuda, 8, 1024, 256, 11)
    state = moe.Fp8MoeState(*layer)
    ids, rw = _route(200 // 50, 8, 4, 6, cuda)
    graphs = []
    for i in range(2):
        x, big = R.activations(4, 1024, 41 + i, torch.bfloat16, cuda), R.activations(200, 1024, 51 + i, torch.bfloat16, cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = (moe.apply_moe(x, ids, rw, state, None, 10.0), ext.fp8_linear(x, w, ws), ext.fp8_linear(big, w, ws),
                    *ext.fp8_quantize(big))
        graphs.append((graph, x, big, outs))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for round_ in range(3):
        for _, x, big, _ in graphs:
            x.mul_(-0.5)
            big.add_(1.0)
        torch.cuda.synchronize()
        for s, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for _, x, big, (m, a, b, q, s) in graphs:
            assert torch.equal(m, moe.apply_moe(x, ids, rw, state, None, 10.0))
            assert torch.equal(a, ext.fp8_linear(x, w, ws)) and torch.equal(b, ext.fp8_linear(big, w, ws))
            q2, s2 = ext.fp8_quantize(big)
            assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


# ------------------------------------------------------------------ refusals
def test_refusals(cuda):
    w, ws = R.e4m3_weight((256, 512), 1, cuda)
    x = torch.zeros((2, 512), dtype=torch.bfloat16, device=cuda)
    layer = _layer(cuda, 2, 256, 128)
    xm = torch.zeros((2, 256), dtype=torch.bfloat16, device=cuda)
    ids, rw = _route(2, 2, 1, 1, cuda)
    scratch = torch.zeros(ext.fp8_moe_scratch_bytes(2, 1, 256, 128), dtype=torch.uint8, device=cuda)
    mo = lambda **k: ext.fp8_moe_decode(**{**dict(x=xm, out=torch.empty_like(xm), gate_up=layer[0], gate_up_scale=layer[1],  # noqa: E731
                                                  down=layer[2], down_scale=layer[3], expert_ids=ids, routing_weights=rw,
                                                  swiglu_limit=10.0, scratch=scratch), **k})
    mo()
    bad = [
        (lambda: ext.fp8_quantize(x.cpu()), "CUDA"),
        (lambda: ext.fp8_quantize(x.int()), "fp16, bf16 or fp32"),
        (lambda: ext.fp8_quantize(x, block_rows=64), "block_rows"),
        (lambda: ext.fp8_quantize(x[0], block_rows=128), "2-D"),
        (lambda: ext.fp8_linear(x[:, :256], w, ws), "does not match"),
        (lambda: ext.fp8_linear(x.double(), w, ws), "x must be"),
        (lambda: ext.fp8_linear(x.to(R.F8), w, ws), "x_scale"),
        (lambda: ext.fp8_linear(x, w, ws, x_scale=ws), "e4m3 x only"),
        (lambda: ext.fp8_linear(x, w, ws[:1]), "weight_scale"),
        (lambda: ext.fp8_linear(x, w, ws.half()), "weight_scale"),
        (lambda: ext.fp8_linear(x[:, :500], w[:, :500].contiguous(), ws), "16-byte"),
        (lambda: ext.fp8_linear(x, w.view(torch.uint8), ws), "float8_e4m3fn"),
        (lambda: ext.fp8_linear(x, w, ws, bias=torch.zeros(5, device=cuda)), "bias"),
        (lambda: ext.fp8_linear(x, w, ws, out_dtype=torch.float64), "out_dtype"),
        (lambda: ext.fp8_linear(x.cpu(), w, ws), "different devices"),
        (lambda: mo(x=xm[:, :128]), "contiguous"),
        (lambda: mo(x=xm.cpu()), "device"),
        (lambda: mo(x=xm.to(R.F8)), "x_scale"),
        (lambda: mo(x_scale=rw), "x_scale"),
        (lambda: mo(expert_ids=ids.short()), "expert_ids"),
        (lambda: mo(routing_weights=rw.double()), "routing_weights"),
        (lambda: mo(swiglu_limit=0.0), "limit"),
        (lambda: mo(swiglu_limit=float("nan")), "limit"),
        (lambda: mo(scratch=scratch[:1024]), "scratch"),
        (lambda: mo(down_scale=layer[3].half()), "scales"),
        (lambda: mo(gate_up=layer[0][:, :128]), "contiguous|must be"),
        (lambda: mo(expert_map=torch.zeros(3, dtype=torch.int32, device=cuda)), "expert_map"),
        (lambda: mo(expert_ids=ids.expand(2, 17).contiguous(), routing_weights=rw.expand(2, 17).contiguous()), "served"),
    ]
    for call, match in bad:
        with pytest.raises(RuntimeError, match=match):
            call()
    assert moe.apply_moe(xm[:0], ids[:0], rw[:0], moe.Fp8MoeState(*layer)) is None
