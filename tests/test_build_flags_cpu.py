"""CPU: how the kernels are built."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "openvis_amd", "csrc")


def test_every_kernel_is_built_without_packed_f32_instructions():
    """v_pk_add_f32 and its like have given wrong results on this hardware: the compiler is told not to make them, in every file"""
    out = subprocess.run(["make", "-n", "-B", "-C", CSRC], check=True, capture_output=True, text=True).stdout
    compiled = [line for line in out.splitlines() if re.search(r"hipcc .* -c ", line)]
    sources = [f for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp"))]
    assert len(compiled) == len(sources) > 20
    for line in compiled:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line
    for f in sources + [h for h in os.listdir(CSRC) if h.endswith(".h")]:
        assert not re.search(r"v_pk_(add|mul|fma)_f32", open(os.path.join(CSRC, f)).read()), f
