"""The builds do not depend on the environment's compiler flags."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def commands(folder, **env):
    return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, folder), "all"], env={**os.environ, **env}, stdout=subprocess.PIPE, text=True, check=True).stdout


def test_the_environment_changes_no_flags():
    want = [line for line in commands("oracle").splitlines() if "-shared" in line]
    assert len(want) == 2 and all("-ffp-contract=off" in line and "-fwrapv" in line for line in want)
    assert [line for line in commands("oracle", CXXFLAGS="-O0").splitlines() if "-shared" in line] == want
    kernels = [line for line in commands("aix_amd/csrc", ARCH="x86_64", CXXFLAGS="-O0").splitlines() if ".hip " in line]
    assert kernels and all("--offload-arch=gfx950" in line and "x86_64" not in line for line in kernels)
