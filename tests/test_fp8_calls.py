"""Calls of the e4m3 layers as the host makes them, without a GPU: tensors that
pass as CUDA ones, and recorded launches."""
from __future__ import annotations

import threading
import time
from types import SimpleNamespace

import pytest
import torch

from dsv4_carve_b200 import moe
from dsv4_carve_b200 import vllm_exl3_c as ext
from dsv4_carve_b200.linear import LinearFP8


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a CUDA device."""
    index = 0

    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        kwargs = {k: v for k, v in (kwargs or {}).items() if k != "device"}
        return super().__torch_function__(func, types, args, kwargs)


class OnDevice1(OnDevice):
    index = 1


@pytest.fixture
def layer(monkeypatch):
    """An Fp8MoeState of 8 experts, 256 x 128, on device 0 whose launches are recorded in `launched`."""
    state = object.__new__(moe.Fp8MoeState)
    launched = []
    state.__dict__.update(experts=SimpleNamespace(index=0, device=torch.device("cuda", 0), E=8, H=256, I=128,
                                                  scratch_bytes=lambda m, topk: ext.fp8_moe_scratch_bytes(m, topk, 256, 128)),
                          n_experts=8, hidden=256, inter=128, pow2_scale=False, launched=launched)
    current = [0]
    monkeypatch.setattr(ext, "_current_device", lambda: current[0])
    monkeypatch.setattr(ext, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: current.__setitem__(0, i))
    monkeypatch.setattr(moe, "_FP8_SCRATCH", {})
    monkeypatch.setattr(ext, "_fp8_moe_decode", lambda *a: launched.append(a))
    real_zeros, real_empty = torch.zeros, torch.empty
    host = lambda f: lambda *a, device=None, **k: f(*a, **k).as_subclass(OnDevice)  # noqa: E731
    monkeypatch.setattr(torch, "zeros", host(real_zeros))
    monkeypatch.setattr(torch, "empty", host(real_empty))
    return state


def _call(T=3, topk=2, kind=OnDevice, dtype=torch.bfloat16, **kw):
    x = torch.ones((T, 256)).to(dtype).as_subclass(kind)
    return dict(x2d=x, ids=torch.ones((T, topk), dtype=torch.int32).as_subclass(kind),
                weights=torch.ones((T, topk)).as_subclass(kind), **kw)


def test_moe_launches_once_up_to_the_ceiling_and_in_pieces_above(layer):
    moe.apply_moe(**_call(32, 8), state=layer)
    assert len(layer.launched) == 1
    moe.apply_moe(**_call(33, 8), state=layer)
    assert [a[0].shape[0] for a in layer.launched] == [32, 32, 1]


def test_moe_host_threads_on_one_stream_take_turns(layer, monkeypatch):
    """One call at a time holds a stream's scratch, from its first launch to its last."""
    inside, most = [0], [0]

    def launch(*a):
        inside[0] += 1
        most[0] = max(most[0], inside[0])
        time.sleep(0.005)                      # the other threads run meanwhile, as during a C call
        inside[0] -= 1

    monkeypatch.setattr(ext, "_fp8_moe_decode", launch)
    threads = [threading.Thread(target=lambda: [moe.apply_moe(**_call(), state=layer) for _ in range(5)]) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert most[0] == 1


@pytest.mark.parametrize("current", [0, 1])
def test_moe_of_another_device_than_the_current_one(layer, current):
    """A layer of device 0 runs there whatever is current; rows of device 1 are refused."""
    torch.cuda.set_device(current)
    moe.apply_moe(**_call(), state=layer)
    assert len(layer.launched) == 1 and torch.cuda.current_device() == current
    with pytest.raises(RuntimeError, match="x is on cuda:1, the layer's experts are on cuda:0"):
        moe.apply_moe(**_call(kind=OnDevice1), state=layer)


def test_moe_types_of_x(layer):
    """e4m3 rows are refused, because their scales have no way in; fp64 ones keep their range."""
    with pytest.raises(RuntimeError, match="x_scale"):
        moe.apply_moe(**_call(dtype=torch.float8_e4m3fn), state=layer)
    assert not layer.launched
    call = _call(dtype=torch.float64)
    call["x2d"] = call["x2d"] * 1e6
    moe.apply_moe(**call, state=layer)
    x, out = layer.launched[0][0], layer.launched[0][2]
    assert x.dtype == torch.float32 and float(x[0, 0]) == 1e6 and out.dtype == torch.float16


@pytest.mark.parametrize("H,I", [(16512, 128), (128, 8320)])
def test_moe_state_refuses_sizes_past_the_limits(H, I):
    """The layer's own message, where the state is built."""
    def of(shape, dtype):
        return torch.empty(shape, dtype=dtype).as_subclass(OnDevice)

    def state(H, I):
        f8 = torch.float8_e4m3fn
        return moe.Fp8MoeState(of((1, 2 * I, H), f8), of((1, 2 * I // 128, H // 128), torch.float32),
                               of((1, H, I), f8), of((1, H // 128, I // 128), torch.float32))

    with pytest.raises(RuntimeError, match="16384 and intermediate up to 8192"):
        state(H, I)
    assert state(H - 128, I).hidden == H - 128 if H > I else state(H, I - 128).inter == I - 128


@pytest.mark.parametrize("T", [5, 80])
def test_moe_checks_the_whole_call_ahead_of_its_pieces(layer, T):
    """ids or out of another number of rows are refused, in one piece or several, before a launch."""
    more = _call(T + 3, 8)
    call = _call(T, 8)
    with pytest.raises(RuntimeError, match="ids of"):
        moe.apply_moe(**{**call, "ids": more["ids"], "weights": more["weights"]}, state=layer)
    less = _call(T - 1, 8)
    with pytest.raises(RuntimeError, match="ids of"):
        moe.apply_moe(**{**call, "ids": less["ids"], "weights": less["weights"]}, state=layer)
    for out in (torch.empty((T + 3, 256)), torch.empty((T, 512))[:, ::2], torch.empty((T - 1, 256))):
        with pytest.raises(RuntimeError, match="out must be"):
            moe.apply_moe(**call, state=layer, out=out.as_subclass(OnDevice))
    assert not layer.launched


@pytest.mark.parametrize("shape,topk", [((20,), 1), ((20, 2, 4), 8), ((20, 4), 4)])
def test_moe_ids_of_other_ranks(layer, shape, topk):
    """ids [rows] are one slot a row, more dimensions are slots too; the scratch is asked for what is launched."""
    call = _call(20, 1)
    call["ids"] = torch.ones(shape, dtype=torch.int32).as_subclass(OnDevice)
    call["weights"] = torch.ones(shape).as_subclass(OnDevice)
    moe.apply_moe(**call, state=layer)
    assert [tuple(a[4].shape) for a in layer.launched] == [(20, topk)]
    assert layer.launched[0][7].numel() == ext.fp8_moe_scratch_bytes(20, topk, 256, 128)


def test_weights_of_a_built_layer_are_not_assigned():
    """What the kernels read was taken when the layer was built; another tensor needs another layer."""
    def of(shape, dtype=torch.float32):
        return torch.zeros(shape).to(dtype).as_subclass(OnDevice)

    f8 = torch.float8_e4m3fn
    lin = LinearFP8(of((256, 128), f8), of((2, 1)))
    state = moe.Fp8MoeState(of((2, 256, 128), f8), of((2, 2, 1)), of((2, 128, 128), f8), of((2, 1, 1)))
    assert lin.weight.shape == (256, 128) and lin.weight_scale.shape == (2, 1) and state.down_scale.shape == (2, 1, 1)
    for layer_, names in ((lin, ("weight", "weight_scale")), (state, ("gate_up", "gate_up_scale", "down", "down_scale"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(layer_, name, getattr(layer_, name).clone())
