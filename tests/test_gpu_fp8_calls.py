"""Calls of the e4m3 operators that a serving program makes: from several host
threads, on slices, with signed zeros."""
from __future__ import annotations

import threading

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


def test_moe_two_host_threads_on_one_stream(cuda):
    """Layers of different sizes from two threads whose current stream is the same."""
    work = []
    for i, (T, H, I) in enumerate(((8, 512, 256), (3, 256, 512))):
        state = moe.Fp8MoeState(*_layer(cuda, 8, H, I, i))
        ids, rw = _route(T, 8, 4, i, cuda)
        x = R.activations(T, H, i, torch.bfloat16, cuda)
        work.append((x, ids, rw, state, moe.apply_moe(x, ids, rw, state, None, 10.0)))
    torch.cuda.synchronize()
    wrong = [None, None]

    def run(i):
        x, ids, rw, state, want = work[i]
        wrong[i] = sum(((moe.apply_moe(x, ids, rw, state, None, 10.0) != want).any() for _ in range(400)),
                       torch.zeros((), dtype=torch.int64, device=cuda))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert [int(w) for w in wrong] == [0, 0]


def test_status_covers_replayed_moe_layers(cuda):
    """One word for the device, read and cleared outside captures; eager and replayed calls leave it at 0."""
    state = moe.Fp8MoeState(*_layer(cuda, 8, 512, 256, 3))
    ids, rw = _route(4, 8, 2, 3, cuda)
    x = R.activations(4, 512, 3, torch.bfloat16, cuda)
    want = moe.apply_moe(x, ids, rw, state, None, 10.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe.apply_moe(x, ids, rw, state, None, 10.0)
    for _ in range(3):
        graph.replay()
        assert ext.fp8_status(cuda) == 0
    assert torch.equal(y, want)
    assert ext.fp8_status(cuda, clear=True) == 0 and ext.fp8_status() == 0


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [128, 136, 131])
def test_quantize_keeps_the_sign_of_zero(cuda, cols, dtype, pow2):
    """The bytes, not the values: -0.0 gives 0x80 in each kind of group, beside
    ordinary values, alone, and where the scale is tiny or huge; so do negative
    values that round to zero."""
    x = R.activations(7, cols, 3, torch.float32, cuda)
    x[:, ::3] = -0.0
    x[:, 1::5] = 0.0
    x[1] = -0.0
    x[2, 2], x[2, 4] = -1e-7, 1e-7
    if dtype == torch.float32:
        x[3] *= 1e-30
        x[4] *= 1e32
        x[5, 2] = -1e-44
    x = x.to(dtype)
    for rows in (1, 128):
        q, _ = ext.fp8_quantize(x, block_rows=rows, pow2_scale=pow2)
        wq, _ = R.quantize(x, rows, pow2)
        sign = torch.signbit(x)
        assert torch.equal(q.double(), wq)
        assert torch.equal((q.view(torch.uint8) & 128) != 0, sign)
        assert bool(((q.view(torch.uint8) == 128) == (sign & (wq == 0))).all())


@pytest.mark.parametrize("rows", [1, 5, 20, 129, 300])
def test_linear_e4m3_rows_at_any_offset(cuda, rows):
    """e4m3 x whose rows start off 16 bytes or lie apart, eager and captured: the bits of an aligned one."""
    w, ws = R.e4m3_weight((384, 528), 5, cuda)
    q, s = ext.fp8_quantize(R.activations(rows, 528, 6, torch.bfloat16, cuda))
    want = ext.fp8_linear(q, w, ws, x_scale=s, out_dtype=torch.float32)
    for off, width in ((0, 529), (3, 560), (4, 576), (16, 592), (1, 529)):
        wide = torch.zeros((rows, width), dtype=torch.uint8, device=cuda)
        wide[:, off:off + 528] = q.view(torch.uint8)
        x = wide.view(R.F8)[:, off:off + 528]
        assert torch.equal(ext.fp8_linear(x, w, ws, x_scale=s, out_dtype=torch.float32), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ext.fp8_linear(x, w, ws, x_scale=s, out_dtype=torch.float32)
        y.zero_()
        for _ in range(2):
            graph.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_from_another_stream(cuda, captured):
    """Rows, ids and weights that a side stream makes while the calls' stream is at
    other work, joined by an event directly ahead of each call."""
    H = 1024
    w, ws = R.e4m3_weight((512, H), 50, cuda)
    state = moe.Fp8MoeState(*_layer(cuda, 8, H, 256, 51))
    side = torch.cuda.Stream()
    src = torch.zeros((300, H), device=cuda)
    lst = torch.zeros((32, 4), dtype=torch.int32, device=cuda)
    waste = torch.ones((2048, 2048), device=cuda)
    calls = {"quantize": lambda x, i: ext.fp8_quantize(x)[0].view(torch.uint8),
             "linear 4": lambda x, i: ext.fp8_linear(x[:4], w, ws), "linear 40": lambda x, i: ext.fp8_linear(x[:40], w, ws),
             "linear 300": lambda x, i: ext.fp8_linear(x, w, ws),
             "moe 2": lambda x, i: moe.apply_moe(x[:2], i[:2], torch.ones((2, 4), device=cuda), state, None, 10.0),
             "moe 32": lambda x, i: moe.apply_moe(x[:32], i, torch.ones((32, 4), device=cuda), state, None, 10.0)}

    def step(call):
        main = torch.cuda.current_stream()
        call(src, lst)                                       # the kernels that came before, whose end may be overlapped
        side.wait_stream(main)
        with torch.cuda.stream(side):
            m = waste
            for _ in range(4):
                m = m @ waste * 2.0 ** -11                   # 1.0 again, late
            x = src * m[0, 0]
            ids = lst + (m[1, 1] - 1.0).to(torch.int32)
        call(src, lst)
        main.wait_stream(side)
        return call(x, ids), x, ids, m

    for name, call in calls.items():
        if captured:
            step(call)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                kept = step(call)
        for seed in range(3):
            src.copy_(R.activations(300, H, seed, torch.bfloat16, cuda))
            lst.copy_(_route(32, 8, 4, seed, cuda)[0])
            if captured:
                graph.replay()
            else:
                kept = step(call)
            torch.cuda.synchronize()
            assert torch.equal(kept[1], src) and torch.equal(kept[2], lst)
            assert torch.equal(kept[0], call(src, lst)), name
            torch.cuda.synchronize()


def test_offsets_past_32_bits(cuda):
    """x, y, its e4m3 copy and the weight with more than 2^31 elements: their last rows."""
    rows, tail = 530000, 300
    w, ws = R.e4m3_weight((136, 4096), 60, cuda)
    x = torch.empty((rows, 4096), dtype=torch.bfloat16, device=cuda).normal_(generator=torch.Generator(device=cuda).manual_seed(1))
    assert x.numel() > 2 ** 31
    wq, wscale = R.quantize(x[-tail:])
    q, s = ext.fp8_quantize(x)
    assert torch.equal(q[-tail:].double(), wq) and torch.equal(s[-tail:].double(), wscale)
    del q, s
    q, s = ext.fp8_quantize(x, block_rows=128)
    last = rows // 128 * 128
    wq, wscale = R.quantize(x[last - 128:], 128)
    assert torch.equal(q[last - 128:].double(), wq) and torch.equal(s[-wscale.shape[0]:].double(), wscale)
    del q, s
    want, allowed = R.linear(R.rows_dequant(x[-tail:]), R.weight(w, ws))
    assert R.worst(ext.fp8_linear(x, w, ws, out_dtype=torch.float32)[-tail:], want, allowed) <= 1.0
    x = x[:, :128].contiguous()
    for n in (4096, 4097):
        w, ws = R.e4m3_weight((n, 128), n, cuda)
        want, allowed = R.linear(R.rows_dequant(x[-tail:]), R.weight(w, ws), None, torch.bfloat16)
        y = ext.fp8_linear(x, w, ws)
        assert y.numel() > 2 ** 31 and R.worst(y[-tail:], want, allowed) <= 1.0
        del y
    n = 128 * 4150
    w = torch.randint(0, 126, (n, 4096), dtype=torch.uint8, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)).view(R.F8)
    ws = torch.rand((4150, 32), device=cuda)
    for m in (3, 20, 140):
        xm = R.activations(m, 4096, m, torch.bfloat16, cuda)
        want, allowed = R.linear(R.rows_dequant(xm), R.weight(w[-256:], ws[-2:]))
        assert R.worst(ext.fp8_linear(xm, w, ws, out_dtype=torch.float32)[:, -256:], want, allowed) <= 1.0
