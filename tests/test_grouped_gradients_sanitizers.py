"""The host code of grouped_linear's gradients (descriptor checks, workspace sizes, refusals) under AddressSanitizer and
UndefinedBehaviorSanitizer: their sources compiled with the sanitizers on their host side only
(-Xarch_host; the device code is built as usual but never launched) and linked with
tests/grouped_gradients_sanitize_main.cpp.  Runs without a GPU; skipped where hipcc is absent."""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(HERE))
# (dg_graph.hip holds the error message that the other reports through)
SOURCES = ["dg_graph.hip", "dg_grouped.hip"]


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="hipcc not available")
def test_grouped_gradients_host_code_under_asan_ubsan(tmp_path):
    from dynamis_amd import build as b

    assert set(SOURCES) <= set(b.SOURCES)
    # every sanitizer flag is scoped to the host pass with -Xarch_host
    flags = [f for f in b.FLAGS if f not in ("-O3",)] + ["-O1", "-g", "-fno-omit-frame-pointer",
                                                      "-Xarch_host", "-fsanitize=address,undefined",
                                                      "-Xarch_host", "-fno-sanitize-recover=all"]
    objs = []
    for src in [os.path.join(b.CSRC, s) for s in SOURCES] + [os.path.join(HERE, "grouped_gradients_sanitize_main.cpp")]:
        obj = str(tmp_path / (os.path.basename(src) + ".o"))
        r = subprocess.run([b.HIPCC, *flags, "-c", src, "-o", obj], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout + r.stderr
        objs.append(obj)
    exe = str(tmp_path / "grouped_gradients_sanitize")
    cmd = [b.HIPCC, f"--offload-arch={b.ARCH}", "-fsanitize=address,undefined", "-fno-gpu-sanitize", *objs, "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert "all checks passed" in r.stdout
    print(r.stdout)
