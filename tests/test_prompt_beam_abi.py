"""The ctypes mirrors of the requests of packed prompts and beams against the C header, compiled here."""
import ctypes
import os
import subprocess

from qwanto_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MIRRORS = {"QwnHipRotaryRequest": abi.RotaryRequest, "QwnHipPromptAttentionRequest": abi.PromptAttentionRequest,
           "QwnHipBeamSelectRequest": abi.BeamSelectRequest, "QwnHipBeamAdvanceRequest": abi.BeamAdvanceRequest}


def test_request_layouts(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "qwn_hip_ext.h"', 'int main(void) {']
    for name, cls in MIRRORS.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    seen = 0
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        cls = MIRRORS[name]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), (name, field)
        seen += 1
    assert seen == sum(len(c._fields_) + 1 for c in MIRRORS.values())
