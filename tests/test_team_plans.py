"""Plans of the channels-last GroupNorm's one-launch kernels, over a sweep of shapes; no device is touched."""
import os
import shutil
import subprocess

from conftest import ROOT, load_package


def test_every_planned_grid_fits_the_device(tmp_path):
    load_package()                                    # builds the library where it is missing
    lib = os.path.join(ROOT, "mobile-stable-diffusion_b200", "lib")
    exe = str(tmp_path / "test_team_plans")
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    r = subprocess.run([nvcc, "-O1", "-std=c++17", os.path.join(ROOT, "tests", "cpp", "test_team_plans.cpp"), "-o", exe, "-L" + lib,
                        "-lsdfl", "-Xlinker", "-rpath," + lib], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr
