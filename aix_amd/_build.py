"""Builds the HIP/C++ libraries in-tree with hipcc / g++ (no cmake, no JIT cache)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def library_path(name):
    return os.path.join(HERE, name)


def build(jobs=8, verbose=False, force=False):
    """Compile every HIP extension for gfx950 and the host library; raises on the first compiler
    error.  force=True recompiles every source even where an up-to-date library is present.

    Every finished step is printed as it ends (some sources compile for minutes, and a build that says nothing looks hung);
    of a failing build the errors are, wherever in the compilers' output they stand."""
    cmd = ["make", "-C", os.path.join(HERE, "csrc"), f"-j{jobs}", "all"] + (["-B"] if force else [])
    lines = []
    with subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, errors="replace") as make:
        for line in make.stdout:
            lines.append(line)
            if verbose or line.startswith("built "):
                print(line, end="", flush=True)
    if make.returncode != 0:
        print("".join([line for line in lines if "error:" in line or "***" in line][:100]), flush=True)
        print("".join(lines)[-4000:], flush=True)
        raise RuntimeError("building the aix_amd libraries failed")
