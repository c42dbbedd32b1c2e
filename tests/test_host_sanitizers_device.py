"""The host code of the paths that need a device (models loaded and closed, steps, recorded steps, trees of drafted tokens, accepted paths
kept, forks, logits judged on the device) under AddressSanitizer and UndefinedBehaviorSanitizer, without a GPU: on a HIP
runtime of host memory (tests/c/hip_stand_in.cpp), driven by tests/c/device_paths.cpp.  A bad access, a copy whose source goes away or
a misuse of the runtime ends the program with a report."""
import os
import subprocess

import pytest
import torch

from conftest import TINY_A
from helpers import ROOT


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    from celeg_amd.csrc import build
    work = str(tmp_path_factory.mktemp("sanitized"))
    try:
        library = build.build_sanitized(work, hip_stand_in=os.path.join(ROOT, "tests", "c", "hip_stand_in.cpp"))
    except build.BuildError as err:
        if "sanitize" in str(err) or "asan" in str(err).lower():
            pytest.skip(f"the compiler has no sanitizer runtime here: {str(err)[-300:]}")
        raise
    path = os.path.join(work, "device_paths")
    subprocess.run([build._hipcc(), "-no-hip-rt", "-std=c++17", "-O1", "-g1", "-x", "hip", f"--offload-arch={build.ARCH}"] + build.SANITIZE_FLAGS +
                   ["-I", os.path.join(ROOT, "celeg_amd", "csrc", "include"), os.path.join(ROOT, "tests", "c", "device_paths.cpp"),
                    "-o", path, "-L", work, "-l:" + os.path.basename(library), "-Wl,-rpath," + work],
                   check=True, capture_output=True, text=True)
    return path


def test_paths_that_need_a_device_under_sanitizers(program, tmp_path):
    from celeg_amd.weights import write_random_model
    attention = dict(TINY_A, layer_types=["full_attention"] * TINY_A["num_hidden_layers"])
    folders = [write_random_model(cfg, str(tmp_path / name), seed=0, dtype=torch.float32, std=0.05)
               for name, cfg in (("attention", attention), ("stateful", TINY_A))]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=0:halt_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    proc = subprocess.run([program] + folders, capture_output=True, text=True, timeout=600, env=env)
    report = proc.stdout[-3000:] + proc.stderr[-6000:]
    assert "AddressSanitizer" not in proc.stderr and "runtime error:" not in proc.stderr and "HIP stand-in:" not in proc.stderr, report
    assert proc.returncode == 0, report
    assert "failures: 0" in proc.stdout
