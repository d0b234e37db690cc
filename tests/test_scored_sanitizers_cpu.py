"""The operators of scored attention, the 8-bit cache and page copies under AddressSanitizer and
UndefinedBehaviorSanitizer on a machine without a GPU: the host layer runs over a device in host memory whose kernels
touch everything that the operators let them touch (tests/sanitize/scored_host.c)."""
import glob
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# what scored_host.c defines itself
OWN = ["device_count", "device_select", "device_synchronize", "device_properties", "malloc", "free", "host_alloc", "host_free",
       "memset_async", "upload_async", "download_async", "stream_create", "stream_destroy", "stream_synchronize"]


def test_scored_operators_are_clean_under_asan_and_ubsan(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc is required")
    sanitize = os.path.join(ROOT, "tests", "sanitize")
    host = os.path.join(ROOT, "clori_b200", "csrc", "host")
    flags = ["-std=c11", "-O1", "-g", "-D_GNU_SOURCE", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
             "-fno-omit-frame-pointer", "-Wall", "-Wextra", "-Wno-unused-parameter", "-Werror", "-I", os.path.join(ROOT, "include"),
             "-I", host]
    absent, exe = str(tmp_path / "absent.o"), str(tmp_path / "scored_driver")
    renamed = [f"-Dyvx_cuda_{x}=absent_{x}" for x in OWN]
    for cmd in (["gcc"] + flags + renamed + ["-c", os.path.join(sanitize, "shim_absent.c"), "-o", absent],
                ["gcc"] + flags + sorted(glob.glob(os.path.join(host, "*.c")) + glob.glob(os.path.join(host, "extension", "*.c"))) +
                [os.path.join(sanitize, x) for x in ("scored_host.c", "scored_driver.c")] + [absent, "-lm", "-o", exe]):
        built = subprocess.run(cmd, capture_output=True, text=True)
        assert built.returncode == 0, built.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1", UBSAN_OPTIONS="halt_on_error=1")
    ran = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=300)
    assert ran.returncode == 0, (ran.stdout[-2000:], ran.stderr[-4000:])
    assert "scored operators clean under the sanitizers" in ran.stdout
