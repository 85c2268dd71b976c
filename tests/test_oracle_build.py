"""The oracle's build takes the reference's sources where they are, and does without them where they are not."""
from oracle import cpuref as O


def test_a_folder_without_the_sources_is_no_reference(tmp_path, monkeypatch):
    monkeypatch.setenv("AIX_REFERENCE_DIR", str(tmp_path))
    assert not O.reference_sources()                        # an empty folder: only the restatement is built
    lib = tmp_path / "Targets" / "AIXLib"
    lib.mkdir(parents=True)
    (lib / "aixDeviceCPU.cpp").write_text("")
    assert O.reference_sources()
    monkeypatch.setenv("AIX_REFERENCE_DIR", str(tmp_path / "nowhere"))
    assert not O.reference_sources()
