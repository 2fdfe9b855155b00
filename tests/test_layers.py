"""CPU checks of the dense layers' interface: struct layouts, and the refusal of tensors off the GPU."""
import ctypes as C
import os
import subprocess

import pytest

from burn_automata_amd import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_c_compiler(tmp_path):
    structs = {"npa_norm_cfg": _abi.NpaNormCfg, "npa_linear_cfg": _abi.NpaLinearCfg}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "npa_abi.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));' for field, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.splitlines():
        cname, what, value = line.split()
        py = structs[cname]
        assert int(value) == (C.sizeof(py) if what == "size" else getattr(py, what).offset), line


def test_constants_match_the_header():
    text = open(os.path.join(ROOT, "include", "npa_abi.h")).read()
    for name in ("TYPE_F32", "TYPE_BF16", "TYPE_F16", "ACT_IDENTITY", "ACT_RELU", "ACT_GELU", "ACT_SILU"):
        assert f"NPA_{name} = {getattr(_abi, name)}" in text, name


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from burn_automata_amd import layers
    x = torch.zeros(2, 3)
    for call in (lambda: layers.layer_norm(x), lambda: layers.linear(x, x), lambda: layers.linear([1.0], x)):
        with pytest.raises(_abi.InvalidArgument, match="not a CUDA tensor"):
            call()
