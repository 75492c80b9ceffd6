"""Programs that include the kernels' sources and run what of them is host code: built for the host alone, without a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def run(tmp_path, source, *args):
    """The lines that the program prints."""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    src, exe = tmp_path / "probe.hip", tmp_path / "probe"
    src.write_text(source)
    # kernels are not launched, so that what the device code would be linked as may stay open
    subprocess.run([HIPCC, "--offload-arch=gfx950", "--offload-host-only", "-O1", "-std=c++17", "-w", "-I", os.path.join(ROOT, "anneal_amd", "csrc"), str(src),
                    "-Wl,--unresolved-symbols=ignore-all", "-o", str(exe)], check=True)
    return subprocess.run([str(exe), *map(str, args)], check=True, capture_output=True, text=True).stdout.splitlines()
