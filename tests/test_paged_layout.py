"""The paged 4-bit cache's addressing and the split of its attention's work,
on the host: each code has bits of its own inside its block, pages that the
table does not name and sequences that do not lie in the batch are left out,
and every partial sum that the merge reads was written for its block."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layout_pages_and_split(tmp_path):
    exe = str(tmp_path / "probe")
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-I" + os.path.join(ROOT, "qwanto_amd", "csrc"),
                    os.path.join(ROOT, "tests", "paged_layout_probe.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_null_handles_refused(hip_lib):
    lib = hip_lib.lib
    assert lib.qwn_hip_ext_norm_quantize_device(None, None, None) == -1
    assert "norm" in hip_lib.last_error()
    assert lib.qwn_hip_ext_paged_kv_create(None, None, None) == -1
    assert lib.qwn_hip_ext_paged_kv_destroy(None, None) == -1
    assert lib.qwn_hip_ext_paged_kv_append_device(None, None, None, None) == -1
    assert lib.qwn_hip_ext_paged_kv_read_device(None, None, None, None, None, 0, None) == -1
    assert lib.qwn_hip_ext_paged_kv_attention_workspace_bytes(None, None, None) == 0
    assert lib.qwn_hip_ext_paged_kv_attention_device(None, None, None, None) == -1
    assert "paged attention" in hip_lib.last_error()
    assert lib.qwn_hip_ext_logits_process_device(None, None, None) == -1
    assert lib.qwn_hip_ext_logits_workspace_bytes(0, 0) == 0


def test_request_layouts():
    """The ctypes mirrors of the request structs against the C header."""
    from qwanto_amd import abi
    import ctypes
    import tempfile
    structs = {"QwnHipNormRequest": abi.NormRequest, "QwnHipPagedKvOptions": abi.PagedKvOptions,
               "QwnHipPagedBatch": abi.PagedBatch, "QwnHipPagedAppendRequest": abi.PagedAppendRequest,
               "QwnHipPagedAttentionRequest": abi.PagedAttentionRequest, "QwnHipLogitsRequest": abi.LogitsRequest}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "qwn_hip_ext.h"', 'int main(void) {']
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines.append("return 0; }")
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "p.c"), os.path.join(tmp, "p")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        cname, field, value = line.split()
        cls = structs[cname]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), (cname, field)
