"""The host code of the entry points over class logits under AddressSanitizer: workspace sizes of every path, and what is refused
before a launch (device code is compiled as usual, nothing runs on a GPU)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_host_code_under_address_sanitizer():
    r = subprocess.run(["make", "-C", os.path.join(ROOT, "unet_amd", "csrc"), "asan_class_rows", "-j8"], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=0:verify_asan_link_order=0")
    r = subprocess.run([os.path.join(ROOT, "tests", "asan_class_rows")], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
