"""The flags that a kernel source is compiled with decide what it computes: another list of flags makes a build stale, and every compiler line of the
tools takes the library's."""
import glob
import os

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_other_flags_make_a_build_stale(monkeypatch, tmp_path):
    from sqd import lib
    src, obj = tmp_path / "a.hip", tmp_path / "a.o"
    for f in (src, obj, tmp_path / "libsqd.so"):
        f.write_text("")
    monkeypatch.setattr(lib, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(lib, "SO_PATH", str(tmp_path / "libsqd.so"))
    monkeypatch.setattr(lib, "FLAGS_PATH", str(tmp_path / "libsqd.flags"))
    monkeypatch.setattr(lib, "sources", lambda: [str(src)])
    monkeypatch.setattr(lib, "_headers", lambda: [str(src)])
    monkeypatch.delenv("SQD_HIPCC_EXTRA", raising=False)
    assert lib.needs_build() and lib._stale(str(src), 0)              # nobody says what these were built with
    (tmp_path / "libsqd.flags").write_text("\n".join(lib.compile_flags()))
    assert not lib.needs_build() and not lib._stale(str(src), 0)
    monkeypatch.setenv("SQD_HIPCC_EXTRA", "-DX")
    assert lib.needs_build() and lib._stale(str(src), 0)
    monkeypatch.delenv("SQD_HIPCC_EXTRA")
    monkeypatch.setattr(lib, "HIPCC_FLAGS", [f for f in lib.HIPCC_FLAGS if f != "-packed-fp32-ops"])
    assert lib.needs_build() and lib._stale(str(src), 0)


def test_a_build_says_what_it_was_built_with(monkeypatch, tmp_path):
    """the record is written behind the last step: not there while one is missing"""
    from sqd import lib
    seen = []

    def call(cmd):
        seen.append((cmd, os.path.exists(lib.FLAGS_PATH)))
        open(cmd[cmd.index("-o") + 1], "w").close()
    src = tmp_path / "a.hip"
    src.write_text("")
    monkeypatch.setattr(lib, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(lib, "SO_PATH", str(tmp_path / "libsqd.so"))
    monkeypatch.setattr(lib, "FLAGS_PATH", str(tmp_path / "libsqd.flags"))
    monkeypatch.setattr(lib, "sources", lambda: [str(src)])
    monkeypatch.setattr(lib, "_headers", lambda: [str(src)])
    monkeypatch.setattr(lib, "_LIB", None)
    monkeypatch.setattr(lib.subprocess, "check_call", call)
    lib.build()
    assert len(seen) == 2 and not lib.needs_build()
    lib.build()
    assert len(seen) == 2
    monkeypatch.setenv("SQD_HIPCC_EXTRA", "-DX")
    lib.build()
    assert len(seen) == 4 and "-DX" in seen[2][0] and not any(there for _, there in seen)


def test_every_compiler_line_takes_the_librarys_flags():
    for path in glob.glob(os.path.join(REPO, "tools", "**", "*"), recursive=True):
        if path.endswith((".sh", ".py")):
            with open(path) as f:
                text = f.read()
            # a command line that compiles device code; "hipcc ..." is a usage text
            lines = [line for line in text.splitlines() if "hipcc" in line and "hipcc ..." not in line and
                     (" -c " in line or "--cuda-device-only" in line or ".hip\"" in line)]
            for line in lines:
                assert "$flags" in line or "compile_flags()" in line, (path, line)
