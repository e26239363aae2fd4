"""The machine code of the library as it is built: no packed fp32 arithmetic anywhere (some operand forms of v_pk_add/mul/fma_f32
have given wrong results on this hardware), and the main loops of the strip walks under the Makefile's own flags.
tests/test_isa_guard.py compiles the same source without the flag that forbids those instructions: what it counts is what the
compiler makes of the pairs in the source, not what runs."""
import os
import re
import shutil
import subprocess

import pytest

import unet_amd
from test_isa_guard import loop_body

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "unet_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
PACKED = re.compile(r"\bv_pk_(add|mul|fma)_f32\b")

# (mangled-name prefix, most multiply-adds in the loop body (two for each packed one of the guard), most instructions there,
#  most registers: 256 for two waves a SIMD, 168 for three)
LOOPS = [
    ("_Z24dwblock_bwd_strip_kernelILi18ELb0ELb0E", 228, 570, 256),
    ("_Z24dwblock_bwd_strip_kernelILi18ELb1ELb0E", 240, 690, 256),
    ("_Z24dwblock_bwd_strip_kernelILi18ELb0ELb1E", 228, 610, 256),
    ("_Z23dwconv_fwd_strip_kernelILi18ELb0E", 120, 340, 168),
    ("_Z23dwconv_fwd_strip_kernelILi18ELb1E", 120, 465, 168),
]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs llvm-objdump")
def test_no_packed_fp32_arithmetic_in_the_library(tmp_path):
    lib = tmp_path / "lib.so"
    shutil.copy(unet_amd.LIB_PATH, lib)
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path, timeout=60)
    objects = sorted(p for p in tmp_path.iterdir() if p.name.endswith("gfx950") and p.stat().st_size)
    assert objects, "no gfx950 code in the library"
    fma = 0
    for p in objects:
        with subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", str(p)], stdout=subprocess.PIPE, text=True) as dump:
            for line in dump.stdout:
                assert not PACKED.search(line), f"{p.name}: {line.strip()}"
                fma += "v_fma" in line
        assert dump.returncode == 0
    assert fma > 1000                                    # the listing is one of instructions


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_strip_walks_under_the_flags_of_the_build(tmp_path):
    dry = subprocess.run(["make", "-n", "-B", "-C", CSRC, "lunext.o", f"HIPCC={HIPCC}"], check=True, capture_output=True, text=True).stdout
    cmd = next(line for line in dry.splitlines() if line.endswith("-c lunext.hip -o lunext.o")).split()
    out = tmp_path / "lunext.s"
    cmd = cmd[:-4] + ["-S", "--cuda-device-only", "lunext.hip", "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, cwd=CSRC, timeout=600)
    asm = out.read_text()
    assert not PACKED.search(asm)
    for prefix, most_fma, most_instructions, most_registers in LOOPS:
        body = loop_body(asm, prefix)
        assert body, f"no loop found in {prefix}"
        fma = sum(bool(re.search(r"\bv_fmac?_f32", line)) for line in body)
        instructions = sum(bool(re.match(r"\s+[vsbdg]\w+", line)) for line in body)
        assert 0 < fma <= most_fma and instructions <= most_instructions, f"{prefix}: {fma} multiply-adds of {instructions} instructions"
        m = re.search(r"^%s.*?; NumVgprs: (\d+).*?; ScratchSize: (\d+)" % re.escape(prefix), asm, re.S | re.M)
        assert m and int(m.group(1)) <= most_registers and int(m.group(2)) == 0, f"{prefix}: {m and m.groups()}"
