"""CPU tests of the paged cache's host side: the structures that Python hands to the library have the
header's layout, descriptions refuse what the kernels do not take, and calls without an engine fail
with a status."""
import ctypes
import os
import re
import subprocess
import sys

import pytest
import torch

import hayai_b200 as hb
from hayai_b200 import _lib, kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,struct", [("hc_kv_cache", kv._Cache), ("hc_kv_batch", kv._Batch)])
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
    for name, struct in (("hc_kv_cache", kv._Cache), ("hc_kv_batch", kv._Batch)):
        body = re.search(r"pub struct " + name + r" \{(.*?)\}", text, re.S).group(1)
        assert [f.replace("ggml_type", "type") for f in re.findall(r"pub (\w+):", body)] == [f for f, _ in struct._fields_]


def test_descriptions_need_device_tensors():
    x = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        hb.KvCache(x, x)
    t = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        hb.KvBatch(t, t[0], t[0, :1], 1)


def test_calls_without_an_engine_return_a_status():
    L = _lib.lib()
    assert L.hc_kv_append_dev(None, None, None, 0, None, 0, None, 0) == _lib.HC_ERR_INVALID
    assert L.hc_kv_read_dev(None, None, None, 0, None, 0, None, 0) == _lib.HC_ERR_INVALID
    assert L.hc_attn_paged_dev(None, None, None, 0, 1, None, 0, None, 0, None, 1.0, 1, 0, 0) == _lib.HC_ERR_INVALID
    assert b"engine" in L.hc_last_error()


def test_a_cache_of_another_device_is_refused():
    """The kernels run on the engine's GPU: descriptions of another one never reach them."""
    class Elsewhere:
        index = 1

    class Here:
        index = device = 0

    for cache, batch in ((Elsewhere, Here), (Here, Elsewhere)):
        with pytest.raises(ValueError, match="device"):
            hb.CudaEngine._kv_here(Here, cache, batch)
    hb.CudaEngine._kv_here(Here, Here, Here)


def replay(tmp_path, *flags):
    exe = tmp_path / "replay"
    subprocess.run(["g++", "-O2", "-std=c++17", *flags, "-I", os.path.join(ROOT, "hayai_b200", "csrc"),
                    os.path.join(ROOT, "tests", "attn_phases.cpp"), "-o", str(exe)], check=True)
    return [int(x) for x in subprocess.run([str(exe), "2000", "7"], capture_output=True, text=True, check=True).stdout.split()]


def test_waits_of_the_prompt_kernel_are_sound(tmp_path):
    """Barriers are waited for by parity: in replays of the kernel's roles over random lists of segments no
    wait is more than one phase away from what it waits for, and none waits for ever."""
    assert replay(tmp_path) == [0, 0]


def test_the_replay_sees_a_wait_that_is_not_sound(tmp_path):
    """Looking at V ahead of the scores in a segment's first unit is found out."""
    unsound, stuck = replay(tmp_path, "-DEARLY=1")
    assert unsound > 0 and stuck == 0


def test_counters_are_cleared_whatever_is_reported(tmp_path):
    """A wait that ran out may leave joining counters behind: they are cleared also where another flag is up
    and gives the report."""
    src = tmp_path / "flags.cpp"
    src.write_text('#include <stdio.h>\n#include "err_flags.h"\nint main() { for (int f = 1; f < 16; ++f) {'
                   'const hc::ErrReport r = hc::err_report(f); printf("%d %d\\n", r.code, r.clear_counters); } }\n')
    exe = tmp_path / "flags"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "hayai_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    rows = [line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()]
    for flag, (code, clear) in enumerate(rows, 1):
        want = _lib.HC_ERR_RANGE if flag & 1 else _lib.HC_ERR_TIMEOUT if flag & 2 else _lib.HC_ERR_INVALID if flag & 4 else None
        assert want is None or int(code) == want
        assert int(clear) == (flag >> 1 & 1)


def test_the_package_imports_without_torch():
    """All public names, and no torch loaded by them: only the cache's descriptions need it."""
    code = "import sys; sys.modules['torch'] = None\nfrom hayai_b200 import *\nCudaEngine, KvCache, KvBatch"
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True)
    code = "import sys\nfrom hayai_b200 import *\nassert 'torch' not in sys.modules"
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True)
