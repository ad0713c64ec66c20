"""The build's bookkeeping, with a compiler that only writes its command line
into its output file."""
import os

import pytest

from vllm_gr_ehaleva_b200 import build as b


@pytest.fixture
def fake(tmp_path, monkeypatch):
    """The build in a folder of its own; returns a function that runs it, `fails` names the
    source (or "link") whose command fails."""
    state = {"fails": None}
    for src in {f for s, hs in b.SOURCES.items() for f in [s, *hs]}:
        (tmp_path / src).write_text("")

    def run(cmd):
        out = cmd[cmd.index("-o") + 1]
        name = os.path.basename(cmd[cmd.index("-c") + 1]) if "-c" in cmd else "link"
        if name == state["fails"]:
            raise RuntimeError(f"{name} failed")
        if name == "link":   # what the library is made of
            text = "\n".join(open(a).read() for a in cmd if a.endswith(".o"))
        else:
            text = " ".join(a for a in cmd if a.startswith("-D")) or "default"
        with open(out, "w") as f:
            f.write(text)
        return ""

    monkeypatch.setattr(b, "CSRC", str(tmp_path))
    monkeypatch.setattr(b, "OBJ_DIR", str(tmp_path / "build"))
    monkeypatch.setattr(b, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "nvcc_path", lambda: "nvcc")
    monkeypatch.setattr(b, "_run", run)

    def build(fails=None, **kw):
        state["fails"] = fails
        return open(b.build(**kw)).read().split("\n")

    return build


N = len(b.SOURCES)


@pytest.mark.parametrize("fails", [*b.SOURCES, "link"])
def test_a_failed_build_with_extra_flags_leaves_nothing_to_the_next_one(fake, fails):
    with pytest.raises(RuntimeError, match="failed"):
        fake(fails, extra_flags=["-DOTHER"])
    assert fake() == ["default"] * N


def test_extra_flags_are_for_one_build(fake):
    assert fake() == ["default"] * N
    kept = {f: os.stat(os.path.join(b.OBJ_DIR, f)).st_mtime_ns for f in os.listdir(b.OBJ_DIR)}
    assert fake(extra_flags=["-DOTHER"]) == ["-DOTHER"] * N
    assert {f: os.stat(os.path.join(b.OBJ_DIR, f)).st_mtime_ns for f in os.listdir(b.OBJ_DIR)} == kept
    assert fake(force=True) == ["default"] * N
