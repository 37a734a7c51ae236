"""CPU tests of the host side of rotary positions, the cache's bookkeeping and shared prefixes: structures as the
header has them, a rope's frequencies against 64-bit arithmetic, refusals, and calls without an engine."""
import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import hayai_b200 as hb
from hayai_b200 import _lib, kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = [("hc_kv_shared", kv._Shared), ("hc_kv_pages", kv._Pages), ("hc_rope", kv._Rope)]


@pytest.mark.parametrize("name,struct", STRUCTS)
def test_structures_match_the_header(tmp_path, name, struct):
    fields = [f for f, _ in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "hayai_cuda.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu ", offsetof({name}, {f}));\n' for f in fields)
                   + f'printf("%zu\\n", sizeof({name}));\nreturn 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


def test_rust_structures_name_the_same_fields():
    text = open(os.path.join(ROOT, "integration", "hayai-cuda", "src", "ffi.rs")).read()
    for name, struct in STRUCTS:
        body = re.search(r"pub struct " + name + r" \{(.*?)\}", text, re.S).group(1)
        assert re.findall(r"pub (\w+):", body) == [f for f, _ in struct._fields_]


def test_calls_without_an_engine_return_a_status():
    L = _lib.lib()
    assert L.hc_attn_shared_dev(None, None, None, None, 0, 1, None, 0, None, 0, None, 1.0) == _lib.HC_ERR_INVALID
    assert L.hc_rope_dev(None, None, 0, 1, 1, None, None, 0, None, 0) == _lib.HC_ERR_INVALID
    assert L.hc_kv_append_rope_dev(None, None, None, None, 0, 1, *[None, 0] * 4) == _lib.HC_ERR_INVALID
    assert L.hc_kv_fork_dev(None, None, 0, None, None) == _lib.HC_ERR_INVALID
    assert L.hc_kv_resize_dev(None, None, 0, None, None) == _lib.HC_ERR_INVALID
    assert L.hc_kv_compact_dev(None, None, None) == _lib.HC_ERR_INVALID
    assert b"engine" in L.hc_last_error()
    assert L.hc_rope_init(None, 0, 64, 0, 1e4, 1.0, 0.0, 0.0, 0.0, None, 1.0) == _lib.HC_ERR_INVALID
    n = ctypes.c_size_t()
    assert L.hc_kv_pages_scratch(0, ctypes.byref(n)) == _lib.HC_ERR_INVALID
    assert L.hc_kv_pages_scratch(10, None) == _lib.HC_ERR_INVALID
    assert L.hc_kv_pages_scratch(10**6, ctypes.byref(n)) == _lib.HC_OK and n.value > 4 * 10**6


def test_a_full_pool_has_its_own_report(tmp_path):
    src = tmp_path / "flags.cpp"
    src.write_text('#include <stdio.h>\n#include "err_flags.h"\nint main() { const hc::ErrReport r = hc::err_report(hc::kErrKvFull);'
                   'printf("%d %d %s\\n", r.code, r.clear_counters, r.text); }\n')
    exe = tmp_path / "flags"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "hayai_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    assert out.startswith(f"{_lib.HC_ERR_INVALID} 0 ") and "free page" in out


def turns(rope):
    return np.array(rope.struct.turns[:rope.rot_dim // 2], dtype=np.uint64)


@pytest.mark.parametrize("dim,rot,base,kw", [
    (128, 0, 10000.0, {}), (64, 16, 500000.0, dict(factor=4.0)), (256, 256, 1e6, dict(factor=8.0, original=8192, low=1.0, high=4.0)),
    (6, 2, 10.0, {}), (128, 96, 1.0, dict(factor=0.25)), (80, 32, 10000.0, dict(factors=[1.0 + 0.5 * i for i in range(16)]))])
def test_frequencies(dim, rot, base, kw):
    """Turns are kept to 2^-64: against long doubles of 64 bits, 2^-60 leaves room for the powers' own rounding."""
    r = hb.Rope(dim, rot, base=base, **kw)
    half = (rot or dim) // 2
    t = np.longdouble(base) ** (-np.arange(half, dtype=np.longdouble) / half) / np.asarray(
        kw.get("factors", [1.0] * half), np.float32).astype(np.longdouble)
    tau = 8 * np.arctan(np.longdouble(1))
    if "original" in kw:
        g = np.clip((kw["original"] * t / tau - kw["low"]) / (kw["high"] - kw["low"]), 0, 1)
        t = t * ((1 - g) / kw["factor"] + g)
    else:
        t = t / np.longdouble(kw.get("factor", 1.0))
    want = t / tau % 1
    got = turns(r).astype(np.longdouble) / np.longdouble(2) ** 64
    off = np.abs(got - want)
    assert np.minimum(off, 1 - off).max() <= 2.0 ** -60
    assert not any(r.struct.turns[half:]) and r.struct.amplitude == 1.0


@pytest.mark.parametrize("args,kw,what", [
    ((128,), dict(layout="other"), "layout"), ((127,), {}, "even"), ((0,), {}, "even"), ((258,), {}, "at most"), ((128, 130), {}, "rot_dim"),
    ((128, 31), {}, "rot_dim"), ((128,), dict(base=0.0), "base"), ((128,), dict(base=math.nan), "base"),
    ((128,), dict(factor=-1.0), "factor"), ((128,), dict(factor=math.inf), "factor"), ((128,), dict(original=-1.0), "original"),
    ((128,), dict(original=4096, factor=4.0), "low"), ((128,), dict(original=4096, low=4.0, high=1.0), "low"),
    ((128,), dict(amplitude=math.inf), "amplitude"), ((128,), dict(factors=[1.0]), "factors"),
    ((128,), dict(factors=[1.0] * 63 + [0.0]), "factors"), ((128,), dict(factors=[1.0] * 63 + [math.nan]), "factors"),
    ((128,), dict(base=1e-300), "range")])
def test_ropes_that_are_refused(args, kw, what):
    with pytest.raises(ValueError, match=what):
        hb.Rope(*args, **kw)


def test_descriptions_need_device_tensors():
    t = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        hb.KvShared(t, t[1:])
    with pytest.raises(ValueError, match="KvCache"):
        hb.KvPages([], t[None], t[:1], t)


def test_other_devices_are_refused():
    class Elsewhere:
        index = 1

    class Here:
        index = 0

    e = hb.CudaEngine.__new__(hb.CudaEngine)
    e.device, e.handle = 0, None
    rope = hb.Rope(64)
    for call in (lambda: e.kv_fork_dev(Elsewhere(), None, None), lambda: e.kv_resize_dev(Elsewhere(), None, None),
                 lambda: e.kv_compact_dev(Elsewhere()), lambda: e.attn_shared_dev(Elsewhere(), Here(), Here(), None, None),
                 lambda: e.attn_shared_dev(Here(), Here(), Elsewhere(), None, None),
                 lambda: e.kv_append_rope_dev(Here(), Elsewhere(), rope, None, None, None)):
        with pytest.raises(ValueError, match="device 0"):
            call()
    with pytest.raises(ValueError, match="engine's device"):
        e.rope_dev(rope, torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, 64))
    with pytest.raises(ValueError, match="int32"):
        e.rope_dev(rope, torch.zeros(2), torch.zeros(2, 3, 64))
