"""What the kernels over class logits tell the compiler of their 16-byte accesses to rows that start at any element: read from
the unoptimised intermediate code of their own sources (device code only, no GPU needed)."""
import functools
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "unet_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
SOURCES = ["class_probs.hip", "distill.hip"]
ELEMENT = {"f": 4, "DF16b": 2, "DF16_": 2}              # mangled float, bf16 and fp16


@functools.lru_cache(None)
def functions(source):
    """{mangled name: lines} of the functions as the front end hands them on"""
    out = subprocess.run([HIPCC, "-O1", "-Xclang", "-disable-llvm-passes", "-std=c++17", "--offload-arch=gfx950", "--cuda-device-only",
                          "-S", "-emit-llvm", "-o", "-", os.path.join(CSRC, source)], check=True, capture_output=True, text=True, timeout=300).stdout
    found, body = {}, None
    for line in out.splitlines():
        m = re.match(r"define .*@(\w+)\(", line)
        if m:
            body = found[m.group(1)] = []
        elif line == "}":
            body = None
        elif body is not None:
            body.append(line)
    return found


@pytest.mark.parametrize("source", SOURCES)
def test_loads_of_rows_promise_no_more_than_an_elements_alignment(source):
    seen = 0
    for name, lines in functions(source).items():
        m = re.search(r"RowRegsI(f|DF16b|DF16_)Li\d+ELi\d+EE5fetch", name)
        if m:
            for line in lines:
                at = re.search(r"load <4 x i32>, .*align (\d+)", line)
                if at:
                    promised = int(at.group(1))
                    local = re.search(r"load <4 x i32>, ptr (%\w+)", line).group(1)
                    if any(re.match(rf"\s*{re.escape(local)} = (alloca|addrspacecast)", l) for l in lines):
                        continue                                     # the loaded vector itself, kept in a local variable
                    seen += 1
                    assert promised <= ELEMENT[m.group(1)], f"{name}: {line.strip()}"
    assert seen >= 6
