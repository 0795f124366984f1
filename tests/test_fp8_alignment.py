"""The C ABI of the e4m3 operators refuses pointers off their elements on the
host: a kernel would read or write there at a misaligned address."""
from __future__ import annotations

import ctypes as C

import pytest

from dsv4_carve_b200 import _lib


@pytest.fixture
def p():
    raw = (C.c_uint8 * 256)()
    yield (C.addressof(raw) + 15) // 16 * 16
    del raw


@pytest.mark.parametrize("rows", [2, 100, 300])
@pytest.mark.parametrize("off", [{"x": 1}, {"x": 2, "xd": 2}, {"y": 1}, {"y": 2, "yd": 2}, {"ws": 2}, {"b": 1}, {"b": 2, "bd": 2},
                                 {"xs": 2, "xd": 3}])
def test_linear_pointers(p, off, rows):
    lib = _lib.load()
    at = {k: p + off.get(k, 0) for k in ("x", "y", "ws", "b")}
    xd, yd, bd = off.get("xd", 1), off.get("yd", 1), off.get("bd", 0)
    xs = p + off.get("xs", 0) if xd == 3 else None
    rc = lib.exl3_fp8_linear(at["x"], xd, 256, xs, rows, 256, 128, p, 256, at["ws"], at["b"], bd, at["y"], yd, 128, 0,
                             p, 1 << 40, None)
    assert rc == _lib.EXL3_ERR_ARG and "aligned to their elements" in _lib.last_error()


@pytest.mark.parametrize("m", [2, 8])
@pytest.mark.parametrize("off", [{"x": 1}, {"x": 2, "xd": 2}, {"out": 1}, {"out": 2, "od": 2}, {"gus": 2}, {"dns": 2},
                                 {"ids": 2}, {"ids": 4, "idt": 1}, {"rw": 2}, {"rw": 1, "wdt": 1}, {"emap": 4}, {"xs": 2, "xd": 3}])
def test_moe_pointers(p, off, m):
    lib = _lib.load()
    at = {k: p + off.get(k, 0) for k in ("x", "out", "gus", "dns", "ids", "rw")}
    emap = p + off["emap"] if "emap" in off else None
    route = _lib.MoeRoute(at["ids"], off.get("idt", 0), at["rw"], off.get("wdt", 2), emap, 4 if emap else 0)
    xd = off.get("xd", 1)
    xs = p + off.get("xs", 0) if xd == 3 else None
    rc = lib.exl3_fp8_moe_decode(at["x"], xd, xs, at["out"], off.get("od", 1), m, 512, 256, p, at["gus"], p, at["dns"], 8,
                                 C.addressof(route), 4, 10.0, 0, p, 1 << 40, None)
    assert rc == _lib.EXL3_ERR_ARG and "aligned to their elements" in _lib.last_error()
