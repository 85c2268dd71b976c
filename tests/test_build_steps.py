"""The builds do not depend on the environment's compiler flags, say what they have built as they go, and name their errors."""
import os
import subprocess

import pytest

from aix_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def commands(folder, **env):
    return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, folder), "all"], env={**os.environ, **env}, stdout=subprocess.PIPE, text=True, check=True).stdout


def test_the_environment_changes_no_flags():
    want = [line for line in commands("oracle").splitlines() if "-shared" in line]
    assert len(want) == 2 and all("-ffp-contract=off" in line and "-fwrapv" in line for line in want)
    assert [line for line in commands("oracle", CXXFLAGS="-O0").splitlines() if "-shared" in line] == want
    kernels = [line for line in commands("aix_amd/csrc", ARCH="x86_64", CXXFLAGS="-O0").splitlines() if ".hip " in line]
    assert kernels and all("--offload-arch=gfx950" in line and "x86_64" not in line for line in kernels)


def made(tmp_path, monkeypatch, recipe):
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "Makefile").write_text("all:\n" + "".join(f"\t@{line}\n" for line in recipe))
    monkeypatch.setattr(_build, "HERE", str(tmp_path))


def test_finished_steps_are_printed(tmp_path, monkeypatch, capfd):
    made(tmp_path, monkeypatch, ["echo some command", "echo built a.o", "echo built b.o"])
    _build.build()
    assert capfd.readouterr().out == "built a.o\nbuilt b.o\n"


def test_errors_are_printed_however_much_follows_them(tmp_path, monkeypatch, capfd):
    made(tmp_path, monkeypatch, ["echo built a.o", "echo 'b.hip:1:1: error: no such thing'", "seq -f 'c.hip:%g:1: warning: of no interest' 10000", "exit 1"])
    with pytest.raises(RuntimeError):
        _build.build()
    out = capfd.readouterr().out
    assert out.startswith("built a.o\n") and "b.hip:1:1: error: no such thing" in out and len(out) < 20000


def test_the_makefile_names_every_step():
    out = commands("aix_amd/csrc")
    sources = [f[:-4] + ".o" for f in os.listdir(os.path.join(ROOT, "aix_amd", "csrc", "hip")) if f.endswith(".hip")]
    for target in sources + ["libaixhip_kernels.so", "libaixhip.so", "libaixhip_bench.so"]:
        assert f"echo built {target}" in out, target
