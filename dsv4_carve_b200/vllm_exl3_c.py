"""Drop-in for the reference's native extension module ``vllm_exl3_c``.

Same entry-point names, positional argument order, argument meaning and
error behaviour (RuntimeError with the reference's messages) as the
pybind11 module the vllm-exl3 plugin imports through its ``NATIVE_SO`` hook
(recipe-lna/lna2/bindings.cpp:178-224, recipe-lna/lna2/lna_moe_ticket.cu:489-581).
Every call goes to the sm_100a kernels of libexl3b200.so on the tensors'
CUDA device and the current stream; there is no CPU path (the reference's CPU
fallback of dequant_trellis / exl3_gemv is its CPU baseline, not product).

Generalisations over the reference, all optional keyword arguments:
  * lna2_moe_decode(..., intermediate=256, k_table=None, codebook=1, precise=False):
    any hidden / intermediate that are multiples of 128, top-k 1..16,
    per-expert bit widths through an int32 [experts] table (K = largest);
  * precise: round each decoded weight to fp16 before the MMA (the dense
    entries default to True, the MoE to False; see include/exl3_b200.h);
  * dequant_trellis / exl3_gemv / exl3_gemm(..., codebook=None): the
    reference maps mcg=True to MCG and mcg=False to MUL1 (bindings.cpp:49);
    ``codebook=0`` selects 3INST explicitly.

Besides the EXL3 entries, ``fp8_quantize``, ``fp8_linear`` and
``fp8_moe_decode`` serve the modules that a pack leaves in the checkpoint's
e4m3 with one fp32 scale for each 128 x 128 block.
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import _lib

__all__ = [
    "dequant_trellis", "exl3_gemv", "exl3_gemm", "exl3_mgemm", "lna2_moe_decode", "lna2_moe_scratch_bytes",
    "lna2_moe_max_rows", "lna2_moe_prepare", "lna2_moe_info", "lna2_moe_status", "lna2_moe_status_word",
    "lna2_moe_decode_routed", "lna2_moe_prefill", "lna2_moe_prefill_scratch_bytes", "exl3_linear_scratch_bytes",
    "fp8_quantize", "fp8_linear", "fp8_status", "fp8_moe_decode", "fp8_moe_scratch_bytes", "fp8_moe_max_rows",
]

_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The raw handle without a Stream object around it (0.1 us instead of 2.2 us, of a call's
# 10), and the current device without the module's own initialisation check.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _on_device:
    """Make `device` current for the C-ABI call when it is not already."""

    def __init__(self, device: torch.device):
        self.index = device.index if device.index is not None else torch.cuda.current_device()
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.index:
            self.prev = cur
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


def _codebook(mcg: bool, codebook) -> int:
    if codebook is None:
        return _lib.CB_MCG if mcg else _lib.CB_MUL1
    _check(int(codebook) in (0, 1, 2), "codebook must be 0 (3INST), 1 (MCG) or 2 (MUL1)")
    return int(codebook)


# --------------------------------------------------------------------- dequant
def dequant_trellis(trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, K: int, mcg: bool,
                    *, codebook: int | None = None, inner_only: bool = False) -> torch.Tensor:
    """Decode an EXL3 trellis tensor into an fp16 weight matrix [in, out].

    recipe-lna/lna2/bindings.cpp:118-133.  ``inner_only`` returns W' (no
    Hadamards or sign vectors)."""
    bits = int(K)
    _check(1 <= bits <= 8, "K must be in 1..8")
    _check(trellis.dim() == 3 and trellis.dtype == torch.int16,
           "trellis must be int16 [rows/16, cols/16, 16*K]")
    _check(trellis.size(2) == 16 * bits, "trellis last dimension must be 16*K")
    _check(trellis.size(0) > 0 and trellis.size(1) > 0, "trellis dimensions must be positive")
    _check(suh.dtype == torch.float16 and svh.dtype == torch.float16, "suh and svh must be float16")
    _check(suh.numel() >= trellis.size(0) * 16 and svh.numel() >= trellis.size(1) * 16,
           "suh/svh are too short")
    _check(trellis.is_cuda, "dequant_trellis: the B200 build decodes on CUDA tensors only")
    if not inner_only:
        _check(trellis.size(0) % 8 == 0 and trellis.size(1) % 8 == 0,
               "trellis dimensions must reconstruct whole 128-element Hadamard blocks")
    t = trellis.contiguous()
    su = suh.to(t.device).contiguous()
    sv = svh.to(t.device).contiguous()
    out = torch.empty((t.size(0) * 16, t.size(1) * 16), dtype=torch.float16, device=t.device)
    with _on_device(t.device):
        _lib.call("exl3_dequant", t.data_ptr(), t.size(0), t.size(1), bits, _codebook(mcg, codebook),
                  su.data_ptr(), sv.data_ptr(), out.data_ptr(), 0 if inner_only else 1, _stream(t.device))
    return out


# --------------------------------------------------------------------- dense
_LIN_SCRATCH: dict[tuple[int, int], torch.Tensor] = {}


def exl3_linear_scratch_bytes(rows: int, k: int, n: int, K: int) -> int:
    return int(_lib.load().exl3_linear_scratch_bytes(rows, k, n, K))


def _linear_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Shared per-(device, stream) linear scratch, zeroed on creation; the
    kernel restores its control words, so it is reused without a memset."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    key = (idx, _stream(device))
    buf = _LIN_SCRATCH.get(key)
    if buf is None or buf.numel() < nbytes:
        _check(not torch.cuda.is_current_stream_capturing(),
               "exl3 linear scratch was not prewarmed for this device/stream (graph capture)")
        buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _LIN_SCRATCH[key] = buf
    return buf


def linear_forward(x2: torch.Tensor, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor,
                   K: int, codebook: int, out_dtype: torch.dtype, precise: bool = True) -> torch.Tensor:
    """y[m, n] = x2[m, k] . W on the current stream (k, n multiples of 128).

    precise=True rounds every decoded weight to fp16 as the reference does;
    False feeds the codebook's half pair to the tensor core unrounded."""
    m, k = x2.shape
    n = trellis.size(1) * 16
    _check(x2.dtype in _DT and out_dtype in _DT, "exl3 linear: dtypes must be fp16, bf16 or fp32")
    y = torch.empty((m, n), dtype=out_dtype, device=x2.device)
    nbytes = exl3_linear_scratch_bytes(m, k, n, K)
    scratch = _linear_scratch(x2.device, nbytes)
    with _on_device(x2.device):
        _lib.call("exl3_linear", x2.data_ptr(), _DT[x2.dtype], m, k, n, trellis.data_ptr(), K, codebook,
                  suh.data_ptr(), svh.data_ptr(), y.data_ptr(), _DT[out_dtype], scratch.data_ptr(),
                  scratch.numel(), int(bool(precise)), _stream(x2.device))
    return y


def linear_group_forward(x2: torch.Tensor, mats: list, K: int, codebook: int, out_dtype: torch.dtype,
                         precise: bool = True) -> list:
    """[x2 . W_j for each (trellis_j, suh_j, svh_j) in mats] in one launch:
    one input, up to 8 matrices of the same k, bit width and codebook
    (exllamav3_ext.exl3_mgemm with a broadcast input,
    recipe-lna/exllamav3/exl3_gemm.cu.lna:659-679)."""
    import ctypes

    m, k = x2.shape
    nm = len(mats)
    _check(1 <= nm <= 8, "exl3 linear group: 1 to 8 matrices")
    _check(x2.dtype in _DT and out_dtype in _DT, "exl3 linear: dtypes must be fp16, bf16 or fp32")
    for t, su, sv in mats:
        _linear_checks(x2, t, su, sv, K)
    ns = [int(t.size(1)) * 16 for t, _, _ in mats]
    ys = [torch.empty((m, n), dtype=out_dtype, device=x2.device) for n in ns]
    arr_n = (ctypes.c_int64 * nm)(*ns)
    ptrs = lambda ts: (ctypes.c_void_p * nm)(*[t.data_ptr() for t in ts])   # noqa: E731
    lib = _lib.load()
    nbytes = int(lib.exl3_linear_group_scratch_bytes(m, k, nm, arr_n, K))
    _check(nbytes > 0, "exl3 linear group: unsupported shape")
    scratch = _linear_scratch(x2.device, nbytes)
    with _on_device(x2.device):
        _lib.check(lib.exl3_linear_group(x2.data_ptr(), _DT[x2.dtype], m, k, nm, arr_n,
                                         ptrs([t for t, _, _ in mats]), K, codebook, ptrs([su for _, su, _ in mats]),
                                         ptrs([sv for _, _, sv in mats]), ptrs(ys), _DT[out_dtype],
                                         scratch.data_ptr(), scratch.numel(), int(bool(precise)), _stream(x2.device)))
    return ys


def exl3_mgemm(x: torch.Tensor, trellis: list, suh: list, svh: list, K: int, mcg: bool, *,
               codebook: int | None = None, out_dtype: torch.dtype = torch.float32) -> list:
    """Grouped EXL3 GEMM over matrices sharing the input x [..., k]: returns
    one [m, n_j] output per matrix (fp32 by default, as the plugin's dense
    groups use it, recipe-lna/vllm_exl3_exl3.py.lna:546-613)."""
    bits = int(K)
    _check(len(trellis) == len(suh) == len(svh), "exl3_mgemm: trellis, suh and svh lists differ in length")
    x2 = x.contiguous().view(x.numel() // x.size(-1), x.size(-1))
    mats = [(t.contiguous(), su.contiguous(), sv.contiguous()) for t, su, sv in zip(trellis, suh, svh)]
    return linear_group_forward(x2, mats, bits, _codebook(mcg, codebook), out_dtype)


def _linear_checks(x, trellis, suh, svh, bits):
    _check(x.dim() >= 2, "x must have shape [..., in_features]")
    _check(x.size(-1) == trellis.size(0) * 16, "x feature dimension does not match trellis")
    _check(trellis.dim() == 3 and trellis.dtype == torch.int16 and trellis.size(2) == 16 * bits,
           "trellis must be int16 [rows/16, cols/16, 16*K]")
    _check(suh.dtype == torch.float16 and svh.dtype == torch.float16, "suh and svh must be float16")
    _check(x.is_cuda and trellis.is_cuda and suh.is_cuda and svh.is_cuda,
           "exl3 linear: the B200 build runs on CUDA tensors only")
    _check(x.device == trellis.device == suh.device == svh.device, "exl3 linear: tensors on different devices")


def exl3_gemv(x: torch.Tensor, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, K: int,
              mcg: bool, mmode: int = 1, *, codebook: int | None = None) -> torch.Tensor:
    """Native small-m EXL3 GEMV, [m, k] -> [m, n] in x.dtype (bindings.cpp:135-148)."""
    bits = int(K)
    _check(x.dim() >= 2, "x must have shape [..., in_features]")
    m = x.numel() // x.size(-1)
    _check(1 <= m <= 8, "native GEMV supports 1 <= m <= 8")
    _check(int(mmode) in (0, 1), "mmode must be 0 or 1")
    _linear_checks(x, trellis, suh, svh, bits)
    x2 = x.contiguous().view(m, x.size(-1))
    return linear_forward(x2, trellis.contiguous(), suh.contiguous(), svh.contiguous(), bits,
                          _codebook(mcg, codebook), x.dtype)


def exl3_gemm(x: torch.Tensor, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, K: int,
              mcg: bool, *, codebook: int | None = None) -> torch.Tensor:
    """Native tiled EXL3 GEMM, any row count (bindings.cpp:104-109)."""
    bits = int(K)
    _linear_checks(x, trellis, suh, svh, bits)
    x2 = x.contiguous().view(x.numel() // x.size(-1), x.size(-1))
    return linear_forward(x2, trellis.contiguous(), suh.contiguous(), svh.contiguous(), bits,
                          _codebook(mcg, codebook), x.dtype)


# --------------------------------------------------------------------- MoE
def lna2_moe_scratch_bytes(max_rows: int | None = None, topk: int = 8, hidden: int = 4096,
                           intermediate: int = 2048) -> int:
    """Scratch bytes for calls up to (max_rows, topk, hidden, intermediate).

    With no arguments: the build's row ceiling, top-8, 4096 x 2048, which
    covers every geometry of the plugin up to a single-GPU expert width."""
    rows = lna2_moe_max_rows() if max_rows is None else int(max_rows)
    return int(_lib.load().exl3_moe_scratch_bytes(rows, topk, hidden, intermediate))


def lna2_moe_max_rows() -> int:
    """Row ceiling of this build (the plugin asks, lna_moe_ticket.cu:491-492)."""
    return int(_lib.load().exl3_moe_max_rows())


def lna2_moe_prepare(K: int) -> None:
    _check(1 <= int(K) <= 4, "LNA2 supports K1..K4 in this build")
    _lib.call("exl3_moe_prepare", int(K))


def lna2_moe_info(K: int) -> list[int]:
    """14 ints; index 13 = concurrent streams (the plugin reads it, :1266-1273)."""
    import ctypes

    buf = (ctypes.c_int64 * 14)()
    _lib.call("exl3_moe_info", int(K), ctypes.addressof(buf))
    return [int(v) for v in buf]


def lna2_moe_status(scratch: torch.Tensor, clear: bool = False) -> int:
    """Device status word of a MoE scratch (0 = healthy).  Synchronizes.

    The word is sticky: kernels only OR bits into it (bit 0 dependency wait
    timed out, 1 misaligned trellis, 2 bit width out of range, 3 ring wait
    timed out, 4 plan overflow), until it is cleared here."""
    import ctypes

    word = ctypes.c_uint32(0)
    with _on_device(scratch.device):
        _lib.call("exl3_scratch_status", scratch.data_ptr(), 1, int(bool(clear)), ctypes.addressof(word),
                  _stream(scratch.device))
    return int(word.value)


def lna2_moe_status_word(scratch: torch.Tensor) -> torch.Tensor:
    """The status word of a MoE (or prefill) scratch as a 1-element int32
    device tensor, a view that stays valid as long as the scratch: a serving
    loop can copy it to pinned memory asynchronously (or test it inside a CUDA
    graph) after a layer, without a synchronization per call."""
    _check(scratch.is_cuda and scratch.dtype == torch.uint8 and scratch.numel() >= 12,
           "LNA2 scratch must be a CUDA uint8 buffer")
    return scratch[8:12].view(torch.int32)


def _raise_on_status(scratch: torch.Tensor) -> None:
    word = lna2_moe_status(scratch, clear=True)
    if word:
        raise RuntimeError(f"LNA2 device status word 0x{word:x}: a bounded wait or check failed inside the kernel "
                           "(bit 0 dependency timeout, 1 misaligned trellis, 2 bad bit width, 3 ring timeout, "
                           "4 plan overflow); the output of that call is not valid")


def check_status_default() -> bool:
    """EXL3_MOE_CHECK_STATUS=1 makes every MoE call synchronize and raise on a
    nonzero device status word (a validation mode: one sync per layer)."""
    return os.environ.get("EXL3_MOE_CHECK_STATUS", "0") not in ("", "0")


_IDS_DT = {torch.int32: 0, torch.int64: 1}


class _MoeArgs:
    """Argument checks shared by the MoE entries (lna_moe_ticket.cu:516-553)."""

    def __init__(self, x, out, tables, expert_ids, routing_weights, K, swiglu_limit, scratch, intermediate,
                 k_table, *, routed: bool, prefill: bool, expert_map=None):
        _check(x.is_cuda and x.dtype in ((torch.float16, torch.bfloat16, torch.float32) if routed and not prefill
                                          else (torch.float16, torch.bfloat16)),
               "LNA2 input must be CUDA fp16 or bf16")
        _check(x.dim() == 2 and x.size(1) % 128 == 0, "LNA2 input must be [m,hidden] with hidden % 128 == 0")
        if prefill:
            _check(x.size(0) >= 1, "LNA2 row count out of range (m >= 1)")
        else:
            _check(1 <= x.size(0) <= lna2_moe_max_rows(), "LNA2 row count out of range (1 <= m <= LNA2_MAX_M)")
        _check(x.is_contiguous(), "LNA2 input must be contiguous")
        _check(out.is_cuda and out.device == x.device and out.shape == x.shape and out.is_contiguous(),
               "LNA2 output must match x shape/device and be contiguous")
        _check(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "LNA2 output must be fp16/bf16/fp32")
        topk = expert_ids.size(-1) if expert_ids.dim() == 2 else -1
        id_types = (torch.int32, torch.int64) if routed else (torch.int32,)
        _check(expert_ids.is_cuda and expert_ids.device == x.device and expert_ids.dtype in id_types
               and expert_ids.is_contiguous() and expert_ids.dim() == 2 and expert_ids.size(0) == x.size(0)
               and 1 <= topk <= 16,
               "LNA2 expert_ids must be contiguous int32 [m,topk]" if not routed
               else "LNA2 expert_ids must be contiguous int32 or int64 [m,topk]")
        w_types = (torch.float32, torch.bfloat16, torch.float16) if routed else (torch.float32,)
        _check(routing_weights.is_cuda and routing_weights.device == x.device and routing_weights.dtype in w_types
               and routing_weights.is_contiguous() and routing_weights.shape == expert_ids.shape,
               "LNA2 routing_weights must be contiguous fp32 [m,topk]" if not routed
               else "LNA2 routing_weights must be contiguous fp32/bf16/fp16 [m,topk]")
        n_experts = tables[0].numel()
        _check(1 <= n_experts <= 1024, "LNA2 pointer table has invalid expert count")
        for t in tables:
            _check(t.is_cuda and t.device == x.device and t.dtype == torch.int64 and t.is_contiguous()
                   and t.numel() == n_experts, "LNA2 pointer tables must be contiguous CUDA int64 [experts]")
        limit = float(swiglu_limit)
        _check(limit > 0.0 and limit < float("inf"), "LNA2 requires a finite positive SwiGLU limit")
        inter = int(intermediate)
        if prefill:
            need = lna2_moe_prefill_scratch_bytes(x.size(0), topk, x.size(1), inter, n_experts)
        else:
            need = int(_lib.load().exl3_moe_scratch_bytes(x.size(0), topk, x.size(1), inter))
        _check(scratch.is_cuda and scratch.device == x.device and scratch.dtype == torch.uint8
               and scratch.is_contiguous() and scratch.numel() >= need, "LNA2 scratch too small")
        if k_table is None:
            bits = int(K)
            _check(1 <= bits <= 4, "LNA2 supports K1..K4 in this build")
            kt_ptr, kmax = None, bits
        else:
            _check(k_table.is_cuda and k_table.device == x.device and k_table.dtype == torch.int32
                   and k_table.is_contiguous() and k_table.numel() == n_experts,
                   "LNA2 k_table must be contiguous CUDA int32 [experts]")
            kt_ptr, kmax = k_table.data_ptr(), int(K)
            bits = kmax
        map_ptr, n_global = None, 0
        if expert_map is not None:
            _check(expert_map.is_cuda and expert_map.device == x.device and expert_map.dtype == torch.int64
                   and expert_map.dim() == 1 and expert_map.is_contiguous() and expert_map.numel() >= 1,
                   "EXL3 expert_map must be a contiguous CUDA int64 [n_global] on the hidden-state device")
            map_ptr, n_global = expert_map.data_ptr(), expert_map.numel()
        self.topk, self.n_experts, self.limit, self.inter = topk, n_experts, limit, inter
        self.kt_ptr, self.kmax, self.bits = kt_ptr, kmax, bits
        self.tables = [t.data_ptr() for t in tables]
        self.route = _lib.MoeRoute(expert_ids.data_ptr(), _IDS_DT[expert_ids.dtype], routing_weights.data_ptr(),
                                   _DT[routing_weights.dtype], map_ptr, n_global)


def lna2_moe_decode(x: torch.Tensor, out: torch.Tensor,
                    gate_trellis: torch.Tensor, gate_suh: torch.Tensor, gate_svh: torch.Tensor,
                    up_trellis: torch.Tensor, up_suh: torch.Tensor, up_svh: torch.Tensor,
                    down_trellis: torch.Tensor, down_suh: torch.Tensor, down_svh: torch.Tensor,
                    expert_ids: torch.Tensor, routing_weights: torch.Tensor, K: int,
                    swiglu_limit: float, scratch: torch.Tensor, *, intermediate: int = 256,
                    k_table: torch.Tensor | None = None, codebook: int = 1,
                    precise: bool = False, tp_exchange=None, check_status: bool | None = None) -> torch.Tensor:
    """Routed-expert decode of one layer; writes and returns `out`.

    Argument checks follow recipe-lna/lna2/lna_moe_ticket.cu:516-553.  With
    `tp_exchange` (a dsv4_carve_b200.tp.MoeTpExchange), the tensor-parallel
    sum of the layer output over the exchange's ranks is done inside the
    kernel and every rank's `out` holds the full sum.  `check_status` (default:
    EXL3_MOE_CHECK_STATUS) synchronizes after the launch and raises
    RuntimeError if the device status word reports a failed wait or check."""
    tables = (gate_trellis, gate_suh, gate_svh, up_trellis, up_suh, up_svh, down_trellis, down_suh, down_svh)
    a = _MoeArgs(x, out, tables, expert_ids, routing_weights, K, swiglu_limit, scratch, intermediate, k_table,
                 routed=False, prefill=False)
    with _on_device(x.device):
        if tp_exchange is None:
            _lib.call("exl3_moe_decode", x.data_ptr(), _DT[x.dtype], out.data_ptr(), _DT[out.dtype],
                      x.size(0), x.size(1), a.inter, *a.tables, a.n_experts, a.kt_ptr, a.bits, a.kmax,
                      int(codebook), expert_ids.data_ptr(), routing_weights.data_ptr(), a.topk, a.limit,
                      scratch.data_ptr(), scratch.numel(), int(bool(precise)), _stream(x.device))
        else:
            _check(tp_exchange.table.device == x.device and tp_exchange.hidden == x.size(1)
                   and x.size(0) <= tp_exchange.max_rows, "LNA2 TP exchange does not match this call")
            _lib.call("exl3_moe_decode_tp", x.data_ptr(), _DT[x.dtype], out.data_ptr(), _DT[out.dtype],
                      x.size(0), x.size(1), a.inter, *a.tables, a.n_experts, a.kt_ptr, a.bits, a.kmax,
                      int(codebook), expert_ids.data_ptr(), routing_weights.data_ptr(), a.topk, a.limit,
                      scratch.data_ptr(), scratch.numel(), int(bool(precise)), tp_exchange.table.data_ptr(),
                      tp_exchange.rank, tp_exchange.world, tp_exchange.max_rows, _stream(x.device))
        if check_status_default() if check_status is None else check_status:
            _raise_on_status(scratch)
    return out


def lna2_moe_decode_routed(x: torch.Tensor, out: torch.Tensor,
                           gate_trellis: torch.Tensor, gate_suh: torch.Tensor, gate_svh: torch.Tensor,
                           up_trellis: torch.Tensor, up_suh: torch.Tensor, up_svh: torch.Tensor,
                           down_trellis: torch.Tensor, down_suh: torch.Tensor, down_svh: torch.Tensor,
                           expert_ids: torch.Tensor, routing_weights: torch.Tensor, K: int,
                           swiglu_limit: float, scratch: torch.Tensor, *, intermediate: int = 256,
                           k_table: torch.Tensor | None = None, codebook: int = 1, precise: bool = False,
                           expert_map: torch.Tensor | None = None, tp_exchange=None,
                           check_status: bool | None = None) -> torch.Tensor:
    """lna2_moe_decode on the router's raw outputs, in ONE launch: expert_ids
    int32 or int64 (global ids when `expert_map` is given), routing_weights
    fp32 / bf16 / fp16, x fp16 / bf16 / fp32.  The id mapping and casts the
    reference's plugin runs as torch operations before the kernel
    (map_topk_to_local and .to(int32) / .to(float32),
    recipe-lna/vllm_exl3_exl3.py.lna:963-987,1234-1236) happen inside it
    (exl3_moe_decode_routed)."""
    tables = (gate_trellis, gate_suh, gate_svh, up_trellis, up_suh, up_svh, down_trellis, down_suh, down_svh)
    a = _MoeArgs(x, out, tables, expert_ids, routing_weights, K, swiglu_limit, scratch, intermediate, k_table,
                 routed=True, prefill=False, expert_map=expert_map)
    tp_ptr, tp_rank, tp_world, tp_rows = None, 0, 0, 0
    if tp_exchange is not None:
        _check(tp_exchange.table.device == x.device and tp_exchange.hidden == x.size(1)
               and x.size(0) <= tp_exchange.max_rows, "LNA2 TP exchange does not match this call")
        tp_ptr, tp_rank = tp_exchange.table.data_ptr(), tp_exchange.rank
        tp_world, tp_rows = tp_exchange.world, tp_exchange.max_rows
    import ctypes

    with _on_device(x.device):
        _lib.call("exl3_moe_decode_routed", x.data_ptr(), _DT[x.dtype], out.data_ptr(), _DT[out.dtype],
                  x.size(0), x.size(1), a.inter, *a.tables, a.n_experts, a.kt_ptr, a.bits, a.kmax, int(codebook),
                  ctypes.addressof(a.route), a.topk, a.limit, scratch.data_ptr(), scratch.numel(),
                  int(bool(precise)), tp_ptr, tp_rank, tp_world, tp_rows, _stream(x.device))
        if check_status_default() if check_status is None else check_status:
            _raise_on_status(scratch)
    return out


# --------------------------------------------------------------------- prefill MoE
def lna2_moe_prefill_scratch_bytes(rows: int, topk: int = 8, hidden: int = 4096, intermediate: int = 2048,
                                   n_experts: int = 256) -> int:
    """Scratch bytes of lna2_moe_prefill for calls of up to `rows` tokens.

    Calls longer than lna2_moe_prefill_chunk_tokens(n_experts) run in chunks
    and need no more than one chunk's scratch."""
    return int(_lib.load().exl3_moe_prefill_scratch_bytes(int(rows), int(topk), int(hidden), int(intermediate),
                                                          int(n_experts)))


def lna2_moe_prefill_chunk_tokens(n_experts: int = 256) -> int:
    """Tokens per device route plan (2048 = the reference's TEMP_ROWS_FUSED at
    256 experts, recipe-lna/vllm_exl3_exl3.py.lna:57)."""
    return int(_lib.load().exl3_moe_prefill_chunk_tokens(int(n_experts)))


def lna2_moe_prefill(x: torch.Tensor, out: torch.Tensor,
                     gate_trellis: torch.Tensor, gate_suh: torch.Tensor, gate_svh: torch.Tensor,
                     up_trellis: torch.Tensor, up_suh: torch.Tensor, up_svh: torch.Tensor,
                     down_trellis: torch.Tensor, down_suh: torch.Tensor, down_svh: torch.Tensor,
                     expert_ids: torch.Tensor, routing_weights: torch.Tensor, K: int,
                     swiglu_limit: float, scratch: torch.Tensor, *, intermediate: int = 256,
                     k_table: torch.Tensor | None = None, codebook: int = 1,
                     expert_map: torch.Tensor | None = None, check_status: bool | None = None) -> torch.Tensor:
    """Routed-expert layer for prefill chunks on the tensor cores; writes and
    returns `out`.  Same arguments and checks as lna2_moe_decode, any row
    count; the weights enter the MMA rounded to fp16 (the reference's decoded
    values).  Like lna2_moe_decode_routed it also takes int64 ids, bf16 / fp16
    routing weights and an `expert_map`, read by the device route plan."""
    tables = (gate_trellis, gate_suh, gate_svh, up_trellis, up_suh, up_svh, down_trellis, down_suh, down_svh)
    routed = (expert_map is not None or expert_ids.dtype != torch.int32
              or routing_weights.dtype != torch.float32)
    a = _MoeArgs(x, out, tables, expert_ids, routing_weights, K, swiglu_limit, scratch, intermediate, k_table,
                 routed=routed, prefill=True, expert_map=expert_map)
    import ctypes

    with _on_device(x.device):
        if not routed:
            _lib.call("exl3_moe_prefill", x.data_ptr(), _DT[x.dtype], out.data_ptr(), _DT[out.dtype],
                      x.size(0), x.size(1), a.inter, *a.tables, a.n_experts, a.kt_ptr, a.bits, a.kmax,
                      int(codebook), expert_ids.data_ptr(), routing_weights.data_ptr(), a.topk, a.limit,
                      scratch.data_ptr(), scratch.numel(), _stream(x.device))
        else:
            _lib.call("exl3_moe_prefill_routed", x.data_ptr(), _DT[x.dtype], out.data_ptr(), _DT[out.dtype],
                      x.size(0), x.size(1), a.inter, *a.tables, a.n_experts, a.kt_ptr, a.bits, a.kmax,
                      int(codebook), ctypes.addressof(a.route), a.topk, a.limit, scratch.data_ptr(),
                      scratch.numel(), _stream(x.device))
        if check_status_default() if check_status is None else check_status:
            _raise_on_status(scratch)
    return out


_PREFILL_SCRATCH: dict = {}


def _prefill_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """One scratch tensor per device, grown on demand (prefill is not captured)."""
    key = (device.type, device.index)
    buf = _PREFILL_SCRATCH.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _PREFILL_SCRATCH[key] = buf
    return buf


def exl3_moe(hidden_state, output_state, expert_count, token_sorted, weight_sorted,
             temp_state_g, temp_state_u, temp_intermediate_g, temp_intermediate_u,
             act_function, K_gate, K_up, K_down,
             gate_ptrs_trellis, gate_ptrs_suh, gate_ptrs_svh,
             up_ptrs_trellis, up_ptrs_suh, up_ptrs_svh,
             down_ptrs_trellis, down_ptrs_suh, down_ptrs_svh,
             gate_mcg, gate_mul1, up_mcg, up_mul1, down_mcg, down_mul1,
             act_limit, num_active=-1):
    """exllamav3_ext.exl3_moe with its positional signature and checks
    (orders/F1-ref/exl3_moe.cu:99-210): output_state (fp32, [T, hidden]) +=
    the routed experts' contribution of the sorted slots.  The sorted-slot
    form (expert_count [E+1] int64, token_sorted / weight_sorted [T*topk];
    slots of expert E are skipped) is turned back into per-token slots and
    handed to lna2_moe_prefill; the temp buffers are not used (this build
    keeps its own scratch)."""
    _check(hidden_state.is_cuda and hidden_state.dtype == torch.float16 and hidden_state.dim() == 2,
           "hidden_state must be CUDA fp16 [T, hidden]")
    _check(output_state.dtype == torch.float32 and output_state.shape == hidden_state.shape,
           "output_state must be fp32 with hidden_state's shape")
    _check(expert_count.dtype == torch.int64 and expert_count.dim() == 1, "expert_count must be int64 [E+1]")
    _check(token_sorted.dtype == torch.int64 and token_sorted.shape == weight_sorted.shape,
           "token_sorted / weight_sorted must be [T*topk]")
    _check(gate_mcg == up_mcg == down_mcg and gate_mul1 == up_mul1 == down_mul1,
           "MoE kernel: gate/up/down must share the same codebook")
    _check(gate_mcg != gate_mul1, "MoE kernel: Only mcg and mul1 codebooks are supported")
    _check(K_gate == K_up == K_down, "MoE kernel: gate/up/down must share one bit width in this build")
    if num_active == 0:
        return
    T, hidden = hidden_state.shape
    n_experts = expert_count.numel() - 1
    topk = token_sorted.numel() // T
    _check(topk * T == token_sorted.numel(), "token_sorted must hold T*topk slots")
    ends = torch.cumsum(expert_count, 0)
    pos = torch.arange(token_sorted.numel(), device=token_sorted.device)
    expert_of = torch.searchsorted(ends, pos, right=True)
    order = torch.argsort(token_sorted, stable=True)
    ids = expert_of[order].view(T, topk)
    ids = torch.where(ids < n_experts, ids, torch.full_like(ids, -1)).to(torch.int32).contiguous()
    w = weight_sorted[order].view(T, topk).to(torch.float32).contiguous()
    inter = int(temp_intermediate_g.size(-1))
    y = torch.empty((T, hidden), dtype=torch.float32, device=hidden_state.device)
    scratch = _prefill_scratch(hidden_state.device,
                               lna2_moe_prefill_scratch_bytes(T, topk, hidden, inter, n_experts))
    lna2_moe_prefill(hidden_state.contiguous(), y, gate_ptrs_trellis, gate_ptrs_suh, gate_ptrs_svh,
                     up_ptrs_trellis, up_ptrs_suh, up_ptrs_svh, down_ptrs_trellis, down_ptrs_suh, down_ptrs_svh,
                     ids, w, int(K_gate), float(act_limit), scratch, intermediate=inter,
                     codebook=2 if gate_mul1 else 1)
    output_state.add_(y)


# --------------------------------------------------------------------- e4m3 with block scales
_F8 = torch.float8_e4m3fn
_DT_X8 = {**_DT, _F8: _lib.DT_E4M3}
_FP8_GROUP = 128


def _rows_of(x: torch.Tensor) -> tuple:
    """(x as a 2-D view or copy, its leading dimension): rows may lie apart,
    the elements of a row may not."""
    k = x.size(-1)
    if x.dim() != 2:
        x = x.reshape(-1, k)
    ld, step = x.stride()
    if x.size(0) <= 1:
        ld = k
    if (step != 1 and k > 1) or ld < k:
        x = x.contiguous()
        ld = k
    return x, ld


def fp8_quantize(x: torch.Tensor, *, block_rows: int = 1, pow2_scale: bool = False) -> tuple:
    """(q, scale): x in e4m3 with one fp32 scale for each row and 128 columns
    (``block_rows=1``: activations, x [..., cols]) or for each 128 x 128 block
    (``block_rows=128``: a weight [rows, cols]).

    scale = max(amax / 448, 2^-126); with ``pow2_scale`` the smallest power of
    two that is not below it.  q = e4m3 nearest to x / scale, ties to even."""
    code = _DT.get(x.dtype)
    if not x.is_cuda or code is None or block_rows not in (1, _FP8_GROUP) or x.dim() < 1 or x.size(-1) < 1 \
            or (block_rows != 1 and x.dim() != 2):
        _check(x.is_cuda, "fp8_quantize: the B200 build runs on CUDA tensors only")
        _check(code is not None, "fp8_quantize: x must be fp16, bf16 or fp32")
        _check(block_rows in (1, _FP8_GROUP), "fp8_quantize: block_rows must be 1 or 128")
        _check(x.dim() >= 1 and x.size(-1) >= 1, "fp8_quantize: x must have at least one column")
        _check(False, "fp8_quantize: blocks of 128 rows need a 2-D x")
    x2, ld = _rows_of(x)
    rows, cols = x2.shape
    groups = -(-cols // _FP8_GROUP)
    index = x.device.index
    if _current_device() != index:
        with _on_device(x.device):
            return fp8_quantize(x, block_rows=block_rows, pow2_scale=pow2_scale)
    q = x.new_empty(x.shape, dtype=_F8)
    if block_rows == 1:
        shape = (rows, groups) if x.dim() == 2 else (*x.shape[:-1], groups)
    else:
        shape = (-(-rows // _FP8_GROUP), groups)
    scale = x.new_empty(shape, dtype=torch.float32)
    rc = _lib.load().exl3_fp8_quantize(x2.data_ptr(), code, rows, cols, ld, q.data_ptr(), cols, scale.data_ptr(),
                                       block_rows, 1 if pow2_scale else 0, _raw_stream(index))
    if rc:
        _lib.check(rc)
    return q, scale


def _fp8_weight_checks(weight: torch.Tensor, weight_scale: torch.Tensor) -> None:
    _check(weight.is_cuda and weight_scale.is_cuda and weight.device == weight_scale.device,
           "fp8_linear: the B200 build runs on CUDA tensors of one device")
    _check(weight.dtype == _F8 and weight.dim() == 2 and weight.size(0) >= 1 and weight.size(1) >= 1,
           "fp8_linear: weight must be float8_e4m3fn [out_features, in_features]")
    n, k = weight.shape
    _check((weight.stride(1) == 1 or k == 1) and weight.data_ptr() % 16 == 0
           and (n == 1 or (weight.stride(0) >= k and weight.stride(0) % 16 == 0)),
           "fp8_linear: weight rows must be contiguous and 16-byte aligned (pad in_features to a multiple of 16)")
    _check(weight_scale.dtype == torch.float32 and weight_scale.is_contiguous()
           and weight_scale.shape == (-(-n // _FP8_GROUP), -(-k // _FP8_GROUP)),
           "fp8_linear: weight_scale must be contiguous fp32 [ceil(out / 128), ceil(in / 128)]")


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
               x_scale: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None, pow2_scale: bool = False) -> torch.Tensor:
    """y[..., n] = x[..., k] . weight[n, k]^T (+ bias) over an e4m3 weight with
    one fp32 scale for each 128 x 128 block.

    x fp16 / bf16 / fp32 is quantised by row and 128 columns inside the call
    (``pow2_scale`` as in fp8_quantize), or x is float8_e4m3fn with its
    ``x_scale`` [..., ceil(k / 128)].  ``out_dtype`` defaults to x's type
    (bf16 for an e4m3 x)."""
    return _fp8_linear(x, _Fp8Weight(weight, weight_scale), x_scale, bias, out_dtype, pow2_scale)


class _Fp8Weight:
    """An e4m3 weight as the C ABI takes it, checked once."""
    __slots__ = ("weight", "scale", "n", "k", "groups", "device", "index", "ptr", "ldw", "scale_ptr")

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor):
        _fp8_weight_checks(weight, weight_scale)
        self.weight, self.scale, self.device = weight, weight_scale, weight.device
        self.n, self.k = (int(v) for v in weight.shape)
        self.groups = -(-self.k // _FP8_GROUP)
        self.index = weight.device.index
        self.ldw = weight.stride(0) if self.n > 1 else -(-self.k // 16) * 16
        self.ptr, self.scale_ptr = weight.data_ptr(), weight_scale.data_ptr()


def _fp8_linear(x, w: _Fp8Weight, x_scale, bias, out_dtype, pow2_scale) -> torch.Tensor:
    """fp8_linear behind the checks of the weight, which LinearFP8 makes once."""
    n, k, device = w.n, w.k, w.device
    x_code = _DT_X8.get(x.dtype)
    dim = x.dim()
    if x_code is None or x.device != device or dim < 1 or x.size(-1) != k:
        _check(x_code is not None, "fp8_linear: x must be fp16, bf16, fp32 or float8_e4m3fn")
        _check(x.device == device, "fp8_linear: x and weight on different devices")
        _check(False, "fp8_linear: x feature dimension does not match weight")
    if _current_device() != w.index:
        with _on_device(device):
            return _fp8_linear(x, w, x_scale, bias, out_dtype, pow2_scale)
    x2, ld = _rows_of(x)
    rows = x2.size(0)
    xs_ptr = None
    if x_code == 3:                                  # e4m3
        _check(x_scale is not None and x_scale.device == device and x_scale.dtype == torch.float32
               and x_scale.shape == (*x.shape[:-1], w.groups),
               "fp8_linear: an e4m3 x needs x_scale fp32 [..., ceil(in / 128)]")
        x_scale = x_scale.contiguous()
        xs_ptr = x_scale.data_ptr()
    elif x_scale is not None:
        _check(False, "fp8_linear: x_scale goes with an e4m3 x only")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if x_code == 3 else x.dtype
    y_code = _DT.get(out_dtype)
    if y_code is None:
        _check(False, "fp8_linear: out_dtype must be fp16, bf16 or fp32")
    bias_ptr, bias_code = None, 0
    if bias is not None:
        bias_code = _DT.get(bias.dtype)
        _check(bias.device == device and bias_code is not None and bias.shape == (n,)
               and (n == 1 or bias.stride(0) == 1),
               "fp8_linear: bias must be contiguous fp16, bf16 or fp32 [out_features]")
        bias_ptr = bias.data_ptr()
    y = x2.new_empty((rows, n) if dim == 2 else (*x.shape[:-1], n), dtype=out_dtype)
    if rows == 0:
        return y
    lib = _lib.load()
    scratch, scratch_ptr, need = None, None, 0
    if rows > 1:
        need = lib.exl3_fp8_linear_scratch_bytes(rows, k, n, x_code)
        if need > 0:
            # from the allocator each time: a captured graph owns its own, and streams share none
            scratch = x2.new_empty(need, dtype=torch.uint8)
            scratch_ptr = scratch.data_ptr()
    rc = lib.exl3_fp8_linear(x2.data_ptr(), x_code, ld, xs_ptr, rows, k, n, w.ptr, w.ldw, w.scale_ptr, bias_ptr,
                             bias_code, y.data_ptr(), y_code, n, 1 if pow2_scale else 0, scratch_ptr, need,
                             _raw_stream(w.index))
    if rc:
        _lib.check(rc)
    return y


def fp8_status(device: torch.device | None = None, clear: bool = False) -> int:
    """Status word of the fp8 linear and MoE kernels on a device (0 = healthy;
    bit 3: a ring wait timed out), those of replayed graphs among them.
    Synchronizes; sticky until cleared."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = ctypes.c_uint32(0)
    with _on_device(dev):
        _lib.call("exl3_fp8_status", int(bool(clear)), ctypes.addressof(word), _stream(dev))
    return int(word.value)


def fp8_moe_max_rows() -> int:
    """Row ceiling of fp8_moe_decode."""
    return int(_lib.load().exl3_fp8_moe_max_rows())


def fp8_moe_scratch_bytes(rows: int, topk: int = 8, hidden: int = 4096, intermediate: int = 2048) -> int:
    """Scratch bytes of fp8_moe_decode for calls of `rows` rows (-1: not served)."""
    return int(_lib.load().exl3_fp8_moe_scratch_bytes(int(rows), int(topk), int(hidden), int(intermediate)))


def _fp8_moe_weight_checks(gate_up, gate_up_scale, down, down_scale) -> tuple:
    """(experts, hidden, intermediate) of a layer's stacked e4m3 experts."""
    ts = (gate_up, gate_up_scale, down, down_scale)
    _check(all(t.is_cuda and t.device == gate_up.device and t.is_contiguous() for t in ts),
           "fp8_moe_decode: weights and scales must be contiguous CUDA tensors of one device")
    _check(gate_up.dtype == _F8 and down.dtype == _F8 and gate_up.dim() == 3 and down.dim() == 3,
           "fp8_moe_decode: gate_up and down must be float8_e4m3fn [experts, out, in]")
    E, I2, H = gate_up.shape
    I = down.size(2)
    _check(down.shape == (E, H, I) and I2 == 2 * I and E >= 1,
           "fp8_moe_decode: gate_up must be [experts, 2 * intermediate, hidden], down [experts, hidden, intermediate]")
    _check(H >= 128 and H % 128 == 0 and I >= 128 and I % 128 == 0,
           "fp8_moe_decode: hidden and intermediate must be multiples of 128")
    _check(fp8_moe_scratch_bytes(1, 1, H, I) > 0,
           f"fp8_moe_decode: hidden up to 16384 and intermediate up to 8192 are served, got {H} and {I}")
    _check(gate_up.data_ptr() % 16 == 0 and down.data_ptr() % 16 == 0, "fp8_moe_decode: weights must be 16-byte aligned")
    _check(gate_up_scale.dtype == torch.float32 and gate_up_scale.shape == (E, I2 // 128, H // 128)
           and down_scale.dtype == torch.float32 and down_scale.shape == (E, H // 128, I // 128),
           "fp8_moe_decode: scales must be fp32, one for each 128 x 128 block")
    return E, H, I


def fp8_moe_decode(x: torch.Tensor, out: torch.Tensor, gate_up: torch.Tensor, gate_up_scale: torch.Tensor,
                   down: torch.Tensor, down_scale: torch.Tensor, expert_ids: torch.Tensor,
                   routing_weights: torch.Tensor, swiglu_limit: float, scratch: torch.Tensor, *,
                   x_scale: torch.Tensor | None = None, expert_map: torch.Tensor | None = None,
                   pow2_scale: bool = False, check_status: bool | None = None) -> torch.Tensor:
    """Routed-expert layer for a few rows over e4m3 experts; writes and returns `out`.

    x fp16 / bf16 / fp32 [m, hidden] (quantised by row and 128 columns inside the
    call), or float8_e4m3fn with its ``x_scale`` fp32 [m, hidden / 128].

    gate_up [E, 2 * intermediate, hidden] (gate rows first) and down [E,
    hidden, intermediate] with one fp32 scale for each 128 x 128 block.  The
    router's outputs go in as lna2_moe_decode_routed takes them (int32 or int64
    ids, fp32 / bf16 / fp16 weights, an optional expert_map); `scratch` as
    there, of fp8_moe_scratch_bytes() bytes, zeroed before its first use."""
    w = _Fp8Experts(gate_up, gate_up_scale, down, down_scale)
    return _fp8_moe_decode(x, x_scale, out, w, expert_ids, routing_weights, swiglu_limit, scratch, expert_map,
                           pow2_scale, check_status)


class _Fp8Experts:
    """A layer's e4m3 experts as the C ABI takes them, checked once."""
    __slots__ = ("tensors", "E", "H", "I", "device", "index", "args", "need")

    def __init__(self, gate_up, gate_up_scale, down, down_scale):
        self.E, self.H, self.I = _fp8_moe_weight_checks(gate_up, gate_up_scale, down, down_scale)
        self.tensors = (gate_up, gate_up_scale, down, down_scale)
        self.device, self.index = gate_up.device, gate_up.device.index
        self.args = (*(t.data_ptr() for t in self.tensors), self.E)
        self.need = {}

    def scratch_bytes(self, m: int, topk: int) -> int:
        need = self.need.get((m, topk))
        if need is None:
            need = self.need[(m, topk)] = fp8_moe_scratch_bytes(m, topk, self.H, self.I)
        return need


def _fp8_moe_decode(x, x_scale, out, w: _Fp8Experts, expert_ids, routing_weights, swiglu_limit, scratch, expert_map,
                    pow2_scale, check_status) -> torch.Tensor:
    """fp8_moe_decode behind the checks of the weights, which Fp8MoeState makes once."""
    device, H = w.device, w.H
    if _current_device() != w.index:
        with _on_device(device):
            return _fp8_moe_decode(x, x_scale, out, w, expert_ids, routing_weights, swiglu_limit, scratch, expert_map,
                                   pow2_scale, check_status)
    x_code = _DT_X8.get(x.dtype)
    _check(x.device == device and x_code is not None and x.dim() == 2 and x.size(1) == H and x.is_contiguous(),
           "fp8_moe_decode: x must be contiguous fp16, bf16, fp32 or float8_e4m3fn [m, hidden] on the weights' device")
    m = x.size(0)
    xs_ptr = None
    if x_code == _lib.DT_E4M3:
        _check(x_scale is not None and x_scale.device == device and x_scale.dtype == torch.float32
               and x_scale.shape == (m, H // _FP8_GROUP) and x_scale.is_contiguous() and x.data_ptr() % 16 == 0,
               "fp8_moe_decode: an e4m3 x needs 16-byte alignment and x_scale contiguous fp32 [m, hidden / 128]")
        xs_ptr = x_scale.data_ptr()
    elif x_scale is not None:
        _check(False, "fp8_moe_decode: x_scale goes with an e4m3 x only")
    out_code = _DT.get(out.dtype)
    _check(out.device == device and out_code is not None and out.shape == x.shape and out.is_contiguous(),
           "fp8_moe_decode: out must be contiguous fp16, bf16 or fp32 of x's shape on its device")
    ids_code = _IDS_DT.get(expert_ids.dtype)
    _check(expert_ids.device == device and ids_code is not None and expert_ids.is_contiguous()
           and expert_ids.dim() == 2 and expert_ids.size(0) == m,
           "fp8_moe_decode: expert_ids must be contiguous int32 or int64 [m, topk]")
    topk = expert_ids.size(1)
    w_code = _DT.get(routing_weights.dtype)
    _check(routing_weights.device == device and w_code is not None and routing_weights.is_contiguous()
           and routing_weights.shape == expert_ids.shape,
           "fp8_moe_decode: routing_weights must be contiguous fp32, bf16 or fp16 [m, topk]")
    need = w.scratch_bytes(m, topk)
    limit = float(swiglu_limit)
    if need <= 0 or not limit > 0.0:
        _check(need > 0, "fp8_moe_decode: 1..64 rows, top-k 1..16, rows * top-k up to 256, hidden up to 16384 and "
                         "intermediate up to 8192 are served")
        _check(False, "fp8_moe_decode: the SwiGLU limit must be positive")
    _check(scratch.device == device and scratch.dtype == torch.uint8 and scratch.is_contiguous()
           and scratch.numel() >= need, "fp8_moe_decode: scratch too small")
    map_ptr, n_global = None, 0
    if expert_map is not None:
        _check(expert_map.device == device and expert_map.dtype == torch.int64 and expert_map.dim() == 1
               and expert_map.is_contiguous() and expert_map.numel() >= 1,
               "EXL3 expert_map must be a contiguous CUDA int64 [n_global] on the hidden-state device")
        map_ptr, n_global = expert_map.data_ptr(), expert_map.numel()
    route = _lib.MoeRoute(expert_ids.data_ptr(), ids_code, routing_weights.data_ptr(), w_code, map_ptr, n_global)
    rc = _lib.load().exl3_fp8_moe_decode(x.data_ptr(), x_code, xs_ptr, out.data_ptr(), out_code, m, H, w.I, *w.args,
                                         ctypes.addressof(route), topk, limit, 1 if pow2_scale else 0,
                                         scratch.data_ptr(), scratch.numel(), _raw_stream(w.index))
    if rc:
        _lib.check(rc)
    if check_status_default() if check_status is None else check_status:
        _raise_on_status(scratch)
    return out
