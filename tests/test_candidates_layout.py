"""ctypes' structs of the losses over all candidates and of the rotation have
the sizes and field offsets of the C header's."""
import ctypes
import os
import subprocess

from starry_unigraph.lib import _capi


def test_struct_layouts_match_the_header(tmp_path):
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"sgl_candidates": _capi.Candidates, "sgl_rotary_side": _capi.RotarySide}
    src = tmp_path / "layout.cpp"
    lines = ['#include <cstdio>', '#include <cstddef>', '#include "starrygl_mi355x.h"', 'int main() {']
    want = []
    for name, cls in structs.items():
        lines.append(f'  printf("%zu ", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'  printf("%zu ", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src.write_text("\n".join(lines + ["  return 0;", "}", ""]))
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(repo, "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want
