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
def emitted(source):
    return subprocess.run([HIPCC, "-O1", "-Xclang", "-disable-llvm-passes", "-std=c++17", "--offload-arch=gfx950", "--cuda-device-only",
                           "-S", "-emit-llvm", "-o", "-", os.path.join(CSRC, source)], check=True, capture_output=True, text=True, timeout=300).stdout


def functions(source):
    """{mangled name: lines} of the functions as the front end hands them on"""
    found, body = {}, None
    for line in emitted(source).splitlines():
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


@pytest.mark.parametrize("source", SOURCES)
def test_16_byte_stores_may_meet_stores_of_any_type(source):
    """A gradient is stored 16 bytes at a time, and the label's or the teacher's class once more as one element.  Which of the two
    stays is left to the compiler where it may take them for stores to different objects: so the former are vectors, tagged as
    accesses of any type, and no copies of a struct of integers."""
    seen = 0
    text = emitted(source)
    any_type = re.search(r'^(!\d+) = !\{!"omnipotent char"', text, re.M).group(1)
    tag = re.search(rf"^(!\d+) = !\{{{any_type}, {any_type}, i64 0\}}", text, re.M).group(1)
    for name, lines in functions(source).items():
        if re.search(r"RowRegsI(f|DF16b|DF16_)Li\d+ELi\d+EE3put|copy_(to|from)_lds", name):
            stores = [line for line in lines if re.search(r"store <4 x i32>", line)]
            assert stores and not any("llvm.memcpy" in line for line in lines), name
            assert all(line.endswith(f"!tbaa {tag}") for line in stores if "tbaa" in line), name
            seen += 1
    assert seen >= 6


def test_another_lanes_stores_come_behind_a_fence():
    """the teacher's classes are written by other lanes of the wave than the dense gradient before them"""
    kernels = {name: lines for name, lines in functions("distill.hip").items() if re.search(r"ds_(quad|wave)_kernel", name)}
    for kernel in ("quad", "wave"):
        bodies = [lines for name, lines in kernels.items()
                  if f"ds_{kernel}_kernel" in name and any("wave_stores_in_order" in line for line in lines)]
        assert len(bodies) >= 3, kernel                                  # one for each type
    fence = next(lines for name, lines in functions("distill.hip").items() if "wave_stores_in_order" in name)
    assert sum('fence syncscope("wavefront")' in line for line in fence) == 2
