"""The e4m3 operators' host side, without a GPU: argument checks of the C ABI
and of the Python layer, size queries, the loader, and the tests' own 64-bit
reference against torch's e4m3 conversion."""
from __future__ import annotations

import ctypes as C

import pytest
import torch
from safetensors.torch import save_file

from dsv4_carve_b200 import _lib, loader
from dsv4_carve_b200 import vllm_exl3_c as ext
from dsv4_carve_b200.linear import LinearFP8
from tests import fp8_reference as R


def _err(code: int, fragment: str):
    assert code in (_lib.EXL3_ERR_ARG, _lib.EXL3_ERR_UNSUPPORTED), code
    assert fragment in _lib.last_error()


@pytest.fixture
def buf():
    raw = (C.c_uint8 * 256)()
    base = C.addressof(raw)
    yield (base + 15) // 16 * 16
    del raw


def test_quantize_argument_checks(buf):
    lib, p = _lib.load(), buf

    def call(x=p, dt=1, rows=4, cols=256, ldx=256, q=p, ldq=256, s=p, br=1):
        return lib.exl3_fp8_quantize(x, dt, rows, cols, ldx, q, ldq, s, br, 0, None)

    _err(call(x=None), "null pointer")
    _err(call(q=None), "null pointer")
    _err(call(s=None), "null pointer")
    _err(call(dt=3), "dtype")
    _err(call(rows=-1), "rows")
    _err(call(cols=0), "cols")
    _err(call(br=64), "block_rows")
    _err(call(ldx=255), "leading dimensions")
    _err(call(ldq=8), "leading dimensions")
    _err(call(x=p + 1), "aligned")
    assert call(rows=0, x=None, q=None, s=None) == 0


def test_linear_argument_checks(buf):
    lib, p = _lib.load(), buf

    def call(x=p, xd=1, ldx=256, xs=None, rows=2, k=256, n=128, w=p, ldw=256, ws=p, b=None, bd=0, y=p, yd=1, ldy=128,
             scratch=None, nbytes=0):
        return lib.exl3_fp8_linear(x, xd, ldx, xs, rows, k, n, w, ldw, ws, b, bd, y, yd, ldy, 0, scratch, nbytes, None)

    for name in ("x", "w", "ws", "y"):
        _err(call(**{name: None}), "null pointer")
    _err(call(xd=4), "dtypes")
    _err(call(yd=3), "dtypes")
    _err(call(b=p, bd=3), "dtypes")
    _err(call(k=0), "k and n")
    _err(call(n=0), "k and n")
    _err(call(rows=-1), "rows")
    _err(call(rows=1 << 31), "2^30")
    _err(call(ldx=255), "leading dimensions")
    _err(call(ldw=128), "leading dimensions")
    _err(call(ldy=127), "leading dimensions")
    _err(call(ldw=264), "16-byte")
    _err(call(w=p + 8), "16-byte")
    _err(call(xs=p), "x_scale")
    _err(call(xd=3), "x_scale")
    assert call(rows=0, x=None, w=None, ws=None, y=None) == 0
    sizes = [lib.exl3_fp8_linear_scratch_bytes(r, 1000, 256, d) for r in (0, 1, 8, 17, 4096) for d in (1, 3)]
    assert all(v >= 0 for v in sizes) and sizes[-2] >= 4096 * 1000 and sizes[2] == 0 and sizes[0] == 0
    assert lib.exl3_fp8_linear_scratch_bytes(-1, 1000, 256, 1) == -1
    assert lib.exl3_fp8_linear_scratch_bytes(4, 1000, 256, 4) == -1


def test_moe_argument_checks(buf):
    lib, p = _lib.load(), buf

    def call(x=p, xd=1, xs=None, out=p, od=1, m=4, H=512, I=256, gu=p, gus=p, dn=p, dns=p, E=8, ids=p, idt=0, rw=p, wdt=2,
             emap=None, ng=0, topk=4, limit=10.0, scratch=p, nbytes=1 << 40, null_route=False):
        route = _lib.MoeRoute(ids, idt, rw, wdt, emap, ng)
        return lib.exl3_fp8_moe_decode(x, xd, xs, out, od, m, H, I, gu, gus, dn, dns, E,
                                       None if null_route else C.addressof(route), topk, limit, 0, scratch, nbytes, None)

    for name in ("x", "out", "gu", "gus", "dn", "dns", "ids", "rw", "scratch"):
        _err(call(**{name: None}), "null pointer")
    _err(call(null_route=True), "null pointer")
    _err(call(m=0), "row count")
    _err(call(m=65), "row count")
    _err(call(topk=17), "topk")
    _err(call(m=64, topk=5), "topk")
    _err(call(H=500), "hidden")
    _err(call(H=16512), "hidden")
    _err(call(I=100), "intermediate")
    _err(call(I=8320), "intermediate")
    _err(call(E=0), "expert count")
    _err(call(E=40000), "expert count")
    _err(call(xd=4), "dtypes")
    _err(call(od=3), "dtypes")
    _err(call(wdt=3), "dtypes")
    _err(call(idt=2), "dtypes")
    _err(call(xd=3), "x_scale")
    _err(call(xs=p), "x_scale")
    _err(call(emap=p, ng=0), "expert map")
    _err(call(limit=0.0), "limit")
    _err(call(limit=float("nan")), "limit")
    _err(call(gu=p + 8), "16-byte")
    _err(call(scratch=p + 4), "16-byte")
    _err(call(nbytes=1024), "scratch too small")
    a, b = lib.exl3_fp8_moe_scratch_bytes(4, 8, 4096, 2048), lib.exl3_fp8_moe_scratch_bytes(32, 8, 4096, 2048)
    assert _lib.FP8_MOE_CTRL_BYTES < a < b
    for bad in ((0, 8, 4096, 2048), (65, 1, 4096, 2048), (64, 8, 4096, 2048), (4, 8, 100, 2048), (4, 8, 4096, 100)):
        assert lib.exl3_fp8_moe_scratch_bytes(*bad) == -1
    assert lib.exl3_fp8_moe_max_rows() == 64


def test_python_layer_refuses_cpu_tensors():
    w, s = R.e4m3_weight((128, 256), 1, "cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.fp8_quantize(torch.zeros(2, 128))
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.fp8_linear(torch.zeros(2, 256), w, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        LinearFP8(w, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.fp8_moe_decode(torch.zeros(1, 256), torch.zeros(1, 256), w[None], s[None], w[None], s[None],
                           torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, 1), 10.0, torch.zeros(4))


# ------------------------------------------------------------------ the tests' reference
def test_reference_rounds_like_torch():
    g = torch.Generator().manual_seed(3)
    v = torch.randn(200000, generator=g, dtype=torch.float64) * torch.logspace(-5, 2.6, 200000, dtype=torch.float64)
    v = v.clamp(-448, 448).float().double()
    assert torch.equal(R.round_e4m3(v), v.float().to(R.F8).double())
    codes = torch.arange(127, dtype=torch.uint8).view(R.F8).double()
    assert torch.equal(R.round_e4m3(codes), codes)
    mid = (codes[1:] + codes[:-1]) / 2
    assert torch.equal(R.round_e4m3(mid), mid.float().to(R.F8).double())


def test_reference_scales():
    a = torch.tensor([448.0, 448.0001, 447.99, 0.0, 1e-40, 1.75, 3.5e38], dtype=torch.float64).float().double()
    s = R.scale_of(a, False)
    assert s[0] == 1.0 and s[3] == 2.0 ** -126 and s[4] == 2.0 ** -126 and s[5] == 2.0 ** -8
    p = R.scale_of(a, True)
    assert p[0] == 1.0 and p[1] == 2.0 and p[2] == 1.0 and p[3] == 2.0 ** -126 and p[5] == 2.0 ** -8
    fin = torch.isfinite(a)
    assert torch.all(a[fin] <= 448 * p[fin]) and torch.all((a[fin] > 224 * p[fin]) | (p[fin] == 2.0 ** -126))


# ------------------------------------------------------------------ loader
def _pack(tmp_path, scale_name="scale", scale_dtype=torch.float32, E=2, H=256, I=512):
    tensors = {}
    for e in range(E):
        for j, (name, shape) in enumerate((("w1", (I, H)), ("w3", (I, H)), ("w2", (H, I)))):
            q, s = R.e4m3_weight(shape, 10 * e + j, "cpu")
            if scale_dtype == torch.float8_e8m0fnu:
                s = torch.exp2(torch.round(torch.log2(s)))
            tensors[f"layers.0.ffn.experts.{e}.{name}.weight"] = q
            tensors[f"layers.0.ffn.experts.{e}.{name}.{scale_name}"] = s.to(scale_dtype)
    q, s = R.e4m3_weight((300, 400), 77, "cpu")
    tensors["layers.0.attn.wo.weight"], tensors[f"layers.0.attn.wo.{scale_name}"] = q, s.to(scale_dtype)
    tensors["layers.0.attn.wo.bias"] = torch.arange(300).float()
    save_file(tensors, str(tmp_path / "model.safetensors"))
    return loader.Checkpoint(tmp_path), tensors


@pytest.mark.parametrize("name,dtype", [("scale", torch.float8_e8m0fnu), ("weight_scale_inv", torch.float32),
                                        ("weight_scale", torch.bfloat16)])
def test_loader_reads_e4m3_modules(tmp_path, name, dtype):
    ck, t = _pack(tmp_path, name, dtype)
    assert loader.has_fp8(ck, "layers.0.attn.wo") and not loader.has_fp8(ck, "layers.0.attn.wq")
    w, s, pow2 = loader.load_fp8_weight(ck, "layers.0.attn.wo")
    assert torch.equal(w.view(torch.uint8), t["layers.0.attn.wo.weight"].view(torch.uint8))
    assert s.dtype == torch.float32 and s.shape == (3, 4) and torch.equal(s, t[f"layers.0.attn.wo.{name}"].float())
    assert pow2 == (dtype == torch.float8_e8m0fnu)


def test_loader_shards_whole_blocks(tmp_path):
    ck, t = _pack(tmp_path)
    parts = [loader.shard_fp8_expert(p, *loader.load_fp8_weight(ck, f"layers.0.ffn.experts.0.{n}")[:2], r, 2)
             for p, n in (("gate", "w1"), ("down", "w2")) for r in (0, 1)]
    g = torch.cat([R.weight(*parts[0]), R.weight(*parts[1])])
    d = torch.cat([R.weight(*parts[2]), R.weight(*parts[3])], dim=1)
    assert torch.equal(g, R.weight(t["layers.0.ffn.experts.0.w1.weight"], t["layers.0.ffn.experts.0.w1.scale"]))
    assert torch.equal(d, R.weight(t["layers.0.ffn.experts.0.w2.weight"], t["layers.0.ffn.experts.0.w2.scale"]))
    with pytest.raises(ValueError, match="128-blocks"):
        loader.shard_fp8_expert("gate", *loader.load_fp8_weight(ck, "layers.0.ffn.experts.0.w1")[:2], 0, 8)


def test_loader_refuses_bad_scales(tmp_path):
    q, s = R.e4m3_weight((256, 256), 1, "cpu")
    save_file({"a.weight": q, "a.scale": s[:1].clone(), "b.weight": q.float(), "b.scale": s, "c.weight": q.clone()},
              str(tmp_path / "m.safetensors"))
    ck = loader.Checkpoint(tmp_path)
    with pytest.raises(ValueError, match="128 x 128"):
        loader.load_fp8_weight(ck, "a")
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        loader.load_fp8_weight(ck, "b")
    with pytest.raises(KeyError, match="no block scales"):
        loader.load_fp8_weight(ck, "c")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float8_e8m0fnu])
def test_loaded_layer_runs(cuda, tmp_path, dtype):
    """A pack's e4m3 linear and experts, loaded and run; two shards' sum is the layer."""
    from dsv4_carve_b200 import moe

    ck, t = _pack(tmp_path, "scale", dtype)
    pow2 = dtype == torch.float8_e8m0fnu
    lin = loader.load_linear(ck, "layers.0.attn.wo", cuda)
    assert isinstance(lin, LinearFP8) and lin.pow2_scale == pow2
    x = R.activations(3, 400, 1, torch.bfloat16, cuda)
    want, allowed = R.linear(R.rows_dequant(x, pow2), R.weight(lin.weight, lin.weight_scale), lin.bias)
    assert R.worst(lin.forward(x, {}, out_dtype=torch.float32), want, allowed) <= 1.0
    x = R.activations(3, 256, 2, torch.bfloat16, cuda)
    ids, rw = torch.tensor([[0, 1], [1, -1], [0, 0]], dtype=torch.int32, device=cuda), torch.rand((3, 2), device=cuda)
    total = torch.zeros((3, 256), dtype=torch.float64, device=cuda)
    bound = torch.zeros_like(total)
    for world in (1, 2):
        for r in range(world):
            st = loader.load_fp8_moe_layer(ck, 0, 2, r, world, cuda)
            assert st.pow2_scale == pow2 and st.inter == 512 // world
            y = moe.apply_moe(x, ids, rw, st, None, 10.0, out_dtype=torch.float32)
            want, allowed = R.moe(x, st.gate_up, st.gate_up_scale, st.down, st.down_scale, ids, rw, 10.0, pow2)
            assert R.worst(y, want, allowed) <= 1.0
            total += y.double() * (1 if world == 1 else -1)
            bound += allowed
    # the two shards quantise the same 128-column groups of the inner activations as the whole layer does
    assert bool((total.abs() <= bound).all())
