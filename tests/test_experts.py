"""CPU checks of the mixture of update rules: struct layouts, constants, and what is refused before the GPU is asked."""
import ctypes as C
import os
import subprocess

import pytest

from burn_automata_amd import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_c_compiler(tmp_path):
    structs = {"npa_route_cfg": _abi.NpaRouteCfg, "npa_expert_linear_cfg": _abi.NpaExpertLinearCfg,
               "npa_combine_cfg": _abi.NpaCombineCfg}
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
    for name in ("SCORE_SOFTMAX", "SCORE_SIGMOID"):
        assert f"NPA_{name} = {getattr(_abi, name)}" in text, name


def test_host_tensors_and_missing_plans_are_refused():
    torch = pytest.importorskip("torch")
    from burn_automata_amd import experts
    x = torch.zeros(2, 3)
    words = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: experts.route(x, 2), lambda: experts.route_adjoint(x, x, words), lambda: experts.plan(x, 2),
                 lambda: experts.linear(x, x, None), lambda: experts.linear_adjoint(x, x, x, None),
                 lambda: experts.combine(x, None), lambda: experts.combine_adjoint(x, x, None)):
        with pytest.raises(_abi.InvalidArgument, match="CUDA tensor"):
            call()
    with pytest.raises(_abi.InvalidArgument, match="contiguous int32 on one GPU"):
        experts.Plan(words, words, words)


@pytest.mark.parametrize("rows,top_k,count", ((1, 0, 4), (1, 5, 4), (1, 33, 64), (1, 1, 0), (1, 1, 1025), ((1 << 30) // 8 + 1, 8, 8)))
def test_sizes_that_are_refused(rows, top_k, count):
    pytest.importorskip("torch")
    from burn_automata_amd import experts
    with pytest.raises(_abi.InvalidArgument):
        experts._choices(rows, top_k, count)


@pytest.mark.parametrize("rows,top_k,count", ((0, 1, 1), (1, 32, 32), ((1 << 30) // 8, 8, 1024)))
def test_sizes_at_the_limits_are_served(rows, top_k, count):
    pytest.importorskip("torch")
    from burn_automata_amd import experts
    experts._choices(rows, top_k, count)


def test_unknown_names_are_refused():
    pytest.importorskip("torch")
    from burn_automata_amd import experts
    assert experts._scores("sigmoid") == experts._scores(experts.Scores.sigmoid) == _abi.SCORE_SIGMOID
    with pytest.raises(_abi.InvalidArgument, match="unknown scores"):
        experts._scores("tanh")
