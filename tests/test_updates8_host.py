"""8-bit updates without a GPU: what the calls refuse before they touch a device."""
import pytest
import torch


def test_the_extension_refuses_tensors_that_are_not_on_the_device():
    from lancelot_b200._lib import InvalidArgument
    from lancelot_b200.pybind import _updates8 as m

    v, codes, scales = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 1)
    for call in (lambda: m.quantize_rows(0, 0, v, codes, scales, 0, None, None, None, None),
                 lambda: m.dequantize_rows(0, 0, codes, scales, 64, 0, None, None, 1, None),
                 lambda: m.int8_matmul(0, 0, codes, codes, v[0, :2], v[0, :2], 3, None),
                 lambda: m.int8_distances(0, 0, codes, scales, torch.zeros(2, 1, dtype=torch.int32), 0)):
        with pytest.raises(InvalidArgument, match="cuda:0"):
            call()
    with pytest.raises(TypeError):
        m.int8_matmul(0, 0, [[1]], codes, v, v, 3, None)


def test_the_c_entries_refuse_a_null_context():
    import ctypes as C

    from lancelot_b200 import lib

    z, n, f = C.c_int64(0), None, C.c_size_t(0)
    assert lib.lb_quantize_rows(n, n, 1, z, z, z, n, n, n, z, n, z, C.c_int64(64), z, n, z, n, z, n, f, n) == 1
    assert lib.lb_dequantize_rows(n, n, z, n, z, z, C.c_int64(64), z, n, z, z, n, 1, z, n) == 1
    assert lib.lb_int8_matmul(n, z, z, z, n, z, n, n, z, n, n, 1, z, n, f, n) == 1
    assert lib.lb_int8_distances(n, n, z, n, z, z, C.c_int64(64), z, n, z, z, n, n, f, n) == 1
    assert b"context" in lib.lb_last_error()


def test_workspaces_are_asked_for_only_where_they_are_needed():
    import ctypes as C

    from lancelot_b200 import lib

    q, m, d = lib.lb_quantize_rows_workspace_bytes, lib.lb_int8_matmul_workspace_bytes, lib.lb_int8_distances_workspace_bytes
    for f in (q, m, d):
        f.restype = C.c_size_t
    i = C.c_int64
    assert q(i(5), i(1000), i(1008), i(0)) == 0 and q(i(5), i(1 << 20), i(1 << 20), i(128)) == 0
    assert q(i(2), i(1 << 20), i(1 << 20), i(0)) == 2 * 32 * 4  # the maxima of parts of 32768 columns
    assert q(i(0), i(5), i(16), i(0)) == 0 and q(i(1), i(1), i(15), i(0)) == 0
    a, b = C.c_void_p(4096), C.c_void_p(8192)
    assert m(i(8), i(8), i(64), a, i(64), b, i(64)) == 0
    assert m(i(40), i(41), i(33), a, i(33), b, i(33)) == 2048 + 41 * 48  # both packed to 48 bytes a row
    assert m(i(40), i(41), i(64), C.c_void_p(4097), i(64), b, i(64)) == 2560
    assert m(i(8), i(900), i(33), a, i(33), b, i(33)) == 0  # few rows on one side: read as they lie
    assert m(i(8), i(9), i(131072), a, i(131072), b, i(131072)) == 0
    assert d(None, i(4), i(4), i(64)) == 0


def test_a_cache_checks_its_sizes():
    from lancelot_b200.updates import UpdateCache

    class Device:
        device = 0

    for args in ((0, 5), (3, 0), (3, 5, 24), (3, 5, 8), (3, 5, 32, 48), (3, 5, 32, 16)):
        with pytest.raises(ValueError):
            UpdateCache(Device(), *args)


def test_the_status_names_every_condition_that_it_clears(tmp_path):
    """a wait that ran out beside values that are too large: the check clears both, so it reports both, the graver one as its code"""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source, program = tmp_path / "status.cpp", tmp_path / "status"
    source.write_text("""
#include <cstdio>
#include "context.h"
int main()
{
    for (int flags : {0, 1, 2, 3, 4, 7}) {
        std::string message;
        const int code = lb::status_of(flags, message);
        std::printf("%d %d %s\\n", flags, code, message.c_str());
    }
}
""")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.check_call([os.environ.get("CXX", "g++"), "-std=c++17", "-I" + os.path.join(root, "lancelot_b200", "csrc"), "-I" + os.path.join(cuda, "include"),
                           str(source), "-o", str(program)])
    large, wait, other = "encoded values are too large", "a wait inside a kernel ran out", "device-side status flag raised"
    lines = subprocess.check_output([str(program)], text=True).splitlines()
    got = {int(f): (int(c), m) for f, c, m in (line.split(" ", 2) for line in lines)}
    invalid, logic = 1, 2
    assert got[0] == (0, "")
    for flags, code, named in ((1, invalid, [large]), (2, logic, [wait]), (3, logic, [large, wait]), (4, logic, [other]), (7, logic, [large, wait, other])):
        assert got[flags][0] == code
        assert [m for m in (large, wait, other) if m in got[flags][1]] == named


def test_a_closed_context_is_refused_like_a_null_one():
    from lancelot_b200._lib import InvalidArgument
    from lancelot_b200.cabi import Context

    closed = Context.__new__(Context)
    closed.h, closed.device = None, 0
    v, codes, scales = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 1)
    on = "cuda" if torch.cuda.is_available() else "cpu"
    v, codes, scales = v.to(on), codes.to(on), scales.to(on)
    for call in (lambda: closed.quantize_rows(v, codes, scales), lambda: closed.dequantize_rows(codes, scales, 64),
                 lambda: closed.int8_matmul(codes, codes, v[0, :2], v[0, :2]),
                 lambda: closed.int8_distances(codes, scales, torch.zeros(2, 1, dtype=torch.int32, device=on))):
        with pytest.raises(InvalidArgument, match="context is null" if on == "cuda" else "cuda:0"):
            call()


def test_the_module_of_the_reference_builds_without_torch(monkeypatch, tmp_path, capsys):
    import sys

    from lancelot_b200.pybind import build

    compiled = []
    monkeypatch.setattr(build, "_compile", lambda module, *args: compiled.append(module) or module)
    assert build.build() == "pyCAHEL" and compiled == ["pyCAHEL", "_updates8"]
    compiled.clear()
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))  # one that has no CUDA part
    assert build.build() == "pyCAHEL" and compiled == ["pyCAHEL"] and "_updates8" in capsys.readouterr().err
    compiled.clear()
    monkeypatch.setitem(sys.modules, "torch", None)  # none at all
    assert build.build() == "pyCAHEL" and compiled == ["pyCAHEL"] and "_updates8" in capsys.readouterr().err


def test_a_module_is_built_anew_when_torch_was_replaced(monkeypatch, tmp_path):
    import os
    import types

    from lancelot_b200.pybind import build

    commands = []

    def run(cmd, **_):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return types.SimpleNamespace(returncode=0, stderr="")

    monkeypatch.setattr(build, "PKG", str(tmp_path))
    monkeypatch.setattr(build, "target", lambda module="pyCAHEL": str(tmp_path / (module + ".so")))
    monkeypatch.setattr(build.subprocess, "run", run)
    build.build()
    assert [os.path.basename(c[c.index("-o") + 1]) for c in commands] == ["pyCAHEL.so.tmp", "_updates8.so.tmp"]
    build.build()
    assert len(commands) == 2  # nothing has changed
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build()
    assert len(commands) == 3 and "_updates8.so.tmp" in commands[2][commands[2].index("-o") + 1]
    build.build()
    assert len(commands) == 3


def test_a_cache_takes_no_fraction_of_a_client():
    import numpy as np

    from lancelot_b200.updates import UpdateCache

    cache = UpdateCache.__new__(UpdateCache)
    cache.shape, cache.table = torch.Size((3, 40)), torch.arange(6, dtype=torch.int32).view(3, 2)
    for one in (1, np.int64(1), torch.tensor(1)):
        assert cache._rows(one).tolist() == [[2, 3]]
    for bad in (1.7, 1.0, "1", [1], torch.tensor(1.5), 3, -1):
        with pytest.raises(ValueError):
            cache._rows(bad)
