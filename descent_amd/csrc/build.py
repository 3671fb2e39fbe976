"""Builds libdescent_hip.so in this directory.

Steps: embed kernels/*.inc as C++ string constants (_embedded.cpp), then compile the host library with hipcc
for gfx950 and link it against the HIP runtime and hipRTC.  Device code is generated per kernel descriptor at
run time and compiled by hipRTC with the options in codegen.cpp; `python -m descent_amd.csrc.build --check`
additionally compiles a representative set of generated kernels for gfx950 (no GPU needed).
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libdescent_hip.so")
SOURCES = ["desc.cpp", "codegen.cpp", "operators.cpp", "runtime.cpp", "schedule.cpp", "api.cpp"]
EMBED = {
    "kPreludeSource": "kernels/prelude.inc", "kMatmulMfmaSource": "kernels/matmul_mfma.inc",
    "kRmsNormSource": "kernels/rms_norm.inc", "kRotarySource": "kernels/rotary.inc",
    "kAttentionSource": "kernels/attention.inc", "kDualMatmulSource": "kernels/dual_matmul.inc",
}


def embed() -> str:
    out = ['// generated by build.py from kernels/*.inc -- do not edit', '#include "codegen.hpp"', "namespace dsc {"]
    for name, rel in EMBED.items():
        text = open(os.path.join(HERE, rel)).read()
        assert ')DSCRAW"' not in text
        # string literals are limited to 64 KiB by some compilers: split by line groups
        out.append(f"const char* const {name} =")
        lines = text.splitlines(keepends=True)
        for i in range(0, len(lines), 40):
            out.append('R"DSCRAW(' + "".join(lines[i : i + 40]) + ')DSCRAW"')
        out.append(";")
    out.append("}  // namespace dsc")
    path = os.path.join(HERE, "_embedded.cpp")
    text = "\n".join(out) + "\n"
    if not os.path.exists(path) or open(path).read() != text:
        open(path, "w").write(text)
    return path


def build(verbose: bool = False) -> str:
    embed()
    cmd = [
        "hipcc", "--offload-arch=gfx950", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-o", LIB,
    ] + SOURCES + ["_embedded.cpp", "-lhiprtc", "-lamdhip64", "-ldl"]
    proc = subprocess.run(cmd, cwd=HERE, capture_output=True, text=True)
    if verbose or proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError("building libdescent_hip.so failed:\n" + proc.stderr[-4000:])
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
