"""include/mor_b200_mx.h, the library behind it and its ctypes binding agree, and every entry point refuses bad arguments
before it touches the device (no kernel is launched in this file)."""
import ctypes
import os
import re
import subprocess

import pytest

from mor_b200 import cabi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mor_b200_mx.h")


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"MOR_B200_MX_API\s+\w+\s+(mor_b200_mx_\w+)\s*\(", text)))


def test_header_library_and_binding_agree():
    assert len(declared()) == 6
    out = subprocess.run(["nm", "-D", "--defined-only", cabi.MX_LIB_PATH], capture_output=True, text=True).stdout
    assert sorted(l.split()[-1] for l in out.splitlines() if " T " in l) == declared()
    assert sorted(cabi.MX_SIGNATURES) == declared()


def test_header_compiles_as_c_and_cpp(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "mor_b200.h"\n#include "mor_b200_mx.h"\nint main(void){return mor_b200_mx_quantize_fp4(0,0,0,32,32,0,0,0);}\n')
    for cc, std in (("gcc", "-std=c99"), ("g++", "-std=c++17")):
        exe = tmp_path / ("t_" + cc)
        r = subprocess.run([f"/usr/bin/{cc}", std, "-Wall", "-Werror", "-x", "c" if cc == "gcc" else "c++", str(src), f"-I{ROOT}/include",
                            f"-L{os.path.dirname(cabi.MX_LIB_PATH)}", "-lmor_b200_mx", f"-Wl,-rpath,{os.path.dirname(cabi.MX_LIB_PATH)}",
                            "-o", str(exe)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        assert subprocess.run([str(exe)]).returncode == 0      # no rows: valid, nothing launched


def test_missing_library_fails_loudly(tmp_path, monkeypatch):
    monkeypatch.setattr(cabi, "MX_LIB_PATH", str(tmp_path / "nope.so"))
    monkeypatch.setattr(cabi, "_mx_lib", None)
    with pytest.raises(ImportError, match="no CPU or PyTorch fallback"):
        cabi.mx_lib()


def test_argument_errors_come_back_as_status_codes():
    L = cabi.mx_lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) & ~15
    q = L.mor_b200_mx_quantize_fp4
    assert q(p, 2, 4, 64, 64, p, p, None) == -1          # dtype
    assert q(None, 0, 4, 64, 64, p, p, None) == -1
    assert q(p, 0, 4, 64, 64, None, p, None) == -1
    assert q(p, 0, 4, 64, 64, p, None, None) == -1
    assert q(p, 0, -1, 64, 64, p, p, None) == -1
    assert q(p, 0, 4, 0, 0, p, p, None) == -1
    assert q(p, 0, 4, 64, 32, p, p, None) == -1          # rows overlap
    assert q(p, 0, 4, 48, 48, p, p, None) == -2
    assert q(p, 0, 4, 64, 68, p, p, None) == -2          # pitch of 136 bytes
    assert q(p + 2, 0, 4, 64, 64, p, p, None) == -2
    assert q(p, 0, 4, 64, 64, p + 2, p, None) == -2
    assert q(p, 0, 1 << 40, 64, 64, p, p, None) == -5
    assert q(None, 0, 0, 64, 64, None, None, None) == 0  # no rows
    d = L.mor_b200_mx_dequantize
    assert d(p, p, p, 2, 4, 64, 32, 0, None) == -1
    assert d(p, p, p, 0, 4, 64, 32, 2, None) == -1       # E3M2 is no payload format
    assert d(p, p, p, 0, 4, 64, 48, 0, None) == -1       # 48 does not divide 64
    assert d(p, p, p, 0, 4, 96, 48, 0, None) == -2
    assert d(p, p, p, 0, 4, 64, 4, 0, None) == -2
    assert d(p, p, p, 0, 4, 1024, 512, 0, None) == -2
    assert d(p + 4, p, p, 0, 4, 64, 32, 0, None) == -2
    assert d(p, p, p + 8, 0, 4, 64, 32, 0, None) == -2
    assert d(p, None, p, 0, 4, 64, 32, 0, None) == -1
    assert d(p, p, p, 0, 1 << 40, 64, 32, 0, None) == -5
    assert d(None, None, None, 0, 0, 64, 32, 0, None) == 0
    m = L.mor_b200_mx_matmul
    assert m(p, p, p, p, 4, 4, 64, 4, 0, None, p, None, 0, None) == -1
    assert m(p, p, p, p, 4, 4, 64, 3, 3, None, p, None, 0, None) == -1
    assert m(p, p, p, p, 4, 4, 0, 0, 0, None, p, None, 0, None) == -1
    assert m(p, p, p, p, -4, 4, 64, 0, 0, None, p, None, 0, None) == -1
    assert m(p, p, p, p, 4, 4, 48, 0, 0, None, p, None, 0, None) == -2
    assert m(p + 8, p, p, p, 4, 4, 64, 0, 0, None, p, None, 0, None) == -2
    assert m(p, p, p + 8, p, 4, 4, 64, 0, 0, None, p, None, 0, None) == -2
    assert m(p, p + 4, p, p, 4, 4, 64, 0, 0, None, p, None, 0, None) == -2
    assert m(p, p, p, p + 8, 4, 4, 64, 0, 0, None, p, None, 0, None) == -2
    assert m(p, p, p, p, 4, 4, 64, 0, 0, p + 1, p, None, 0, None) == -2
    assert m(p, p, p, p, 4, 4, 64, 0, 0, None, p + 1, None, 0, None) == -2
    assert m(p, None, p, p, 4, 4, 64, 0, 0, None, p, None, 0, None) == -1
    assert m(p, p, p, p, 4, 4, 64, 0, 0, None, None, None, 0, None) == -1
    assert m(p, p, p, p, 4, 1 << 40, 64, 0, 0, None, p, None, 0, None) == -5
    assert m(None, None, None, None, 0, 4, 64, 0, 0, None, None, None, 0, None) == 0
    assert m(p, p, p, p, 4096, 4096, 64, 0, 0, None, p, None, 0, None) == -3      # needs a workspace
    assert m(p, p, p, p, 4096, 4096, 64, 0, 0, None, p, p, 4096, None) == -3
    assert m(p, p, p, p, 4096, 4096, 64, 0, 0, None, p, p + 8, 1 << 20, None) == -3
    w = L.mor_b200_mx_matmul_workspace_bytes
    assert w(4096, 4096, 64, 0) == 64 * 2 * 512 and w(4097, 4096, 4096, 4) == 65 * 32 * 512
    assert w(1, 4096, 4096, 4) == 0 and w(1, 128, 32, 0) == 0 and w(1024, 4096, 4096, 0) == 0   # one round of tiles
    assert w(0, 1, 32, 0) == 0 and w(4096, 4096, 48, 0) == 0 and w(1 << 40, 1, 32, 0) == 0
    g = L.mor_b200_mx_matmul_grad
    assert g(p, 64, p, p, 4, 64, 64, 2, 0, p, None) == -1
    assert g(p, 64, p, p, 4, 64, 64, 0, 2, p, None) == -1
    assert g(p, 32, p, p, 4, 64, 64, 0, 0, p, None) == -1     # pitch below k
    assert g(p, 32, p, p, 64, 64, 4, 0, 1, p, None) == -1     # pitch below m
    assert g(p, 64, p, p, 4, 48, 64, 0, 0, p, None) == -2
    assert g(p, 68, p, p, 4, 64, 64, 0, 0, p, None) == -2
    assert g(p + 2, 64, p, p, 4, 64, 64, 0, 0, p, None) == -2
    assert g(p, 64, p + 8, p, 4, 64, 64, 0, 0, p, None) == -2
    assert g(p, 64, p, p, 4, 64, 64, 0, 0, p + 8, None) == -2
    assert g(None, 64, p, p, 4, 64, 64, 0, 0, p, None) == -1
    assert g(p, 64, p, p, 4, 64, 0, 0, 0, None, None) == -1   # no sum, and nowhere to write the zeros
    assert g(p, 1 << 40, p, p, 4, 64, 64, 0, 0, p, None) == -5
    assert g(None, 64, None, None, 0, 64, 64, 0, 0, None, None) == 0

    c = L.mor_b200_mx_column_sums
    assert c(None, 64, 4, 64, p, None) == -1 and c(p, 64, 4, 64, None, None) == -1 and c(p, 32, 4, 64, p, None) == -1
    assert c(p, 68, 4, 64, p, None) == -2 and c(p + 2, 64, 4, 64, p, None) == -2 and c(p, 64, 4, 64, p + 1, None) == -2
    assert c(p, 1 << 40, 4, 64, p, None) == -5 and c(None, 0, 4, 0, None, None) == 0


def test_schemas_and_cpu_tensors():
    import torch
    import mor
    z = torch.zeros(4, 64, dtype=torch.uint8)
    for call in (lambda: mor.ops.quantize_mx_fp4(torch.zeros(4, 64, dtype=torch.bfloat16), 4, 64, 32),
                 lambda: mor.ops.dequantize_mx(z, z[:, :2], 4, 64, 32, 0),
                 lambda: mor.ops.mx_matmul(z, z[:, :2], z, z[:, :2], 4, 4, 64, 0, 0),
                 lambda: mor.ops.mx_matmul_grad(torch.zeros(4, 4, dtype=torch.bfloat16), z, z[:, :2], 4, 64, 4, 0, False)):
        with pytest.raises(NotImplementedError):              # CUDA only: no CPU kernel, no fallback
            call()


def test_layer_arguments():
    import torch
    from mor_b200.nn import MXLinear, mx_linear
    with pytest.raises(ValueError, match="elem_format"):
        MXLinear(64, 64, elem_format="fp4")
    with pytest.raises(ValueError, match="multiple of 32"):
        MXLinear(48, 64)
    with pytest.raises(ValueError, match="elem_format"):
        mx_linear(torch.zeros(2, 64), torch.zeros(8, 64), None, 3)
    with pytest.raises(ValueError, match="weight"):
        mx_linear(torch.zeros(2, 32), torch.zeros(8, 64), None, 0)
    assert "elem_format=e2m1" in repr(MXLinear(64, 32, elem_format="e2m1", device="cpu"))
