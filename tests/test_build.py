"""What the build compiles again (a stand-in for the compiler; no GPU, no hipcc)."""
import os


def test_changed_sources_and_changed_flags_are_compiled_again(tmp_path, monkeypatch):
    from sparc_amd import build
    monkeypatch.setattr(build, "LIBDIR", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    calls = []

    def compiler(cmd):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("made")

    monkeypatch.setattr(build.subprocess, "check_call", compiler)

    def compiled():
        calls.clear()
        build.build(verbose=False)
        return sum("-c" in cmd for cmd in calls), len(calls)

    n = len(build.SOURCES)
    first, commands = compiled()
    assert first >= n and commands > first                # every source, and a link behind them
    assert compiled() == (0, 0)
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DSPARC_OTHER"])
    assert compiled()[0] >= n                             # other flags: other objects
    assert compiled() == (0, 0)
    os.utime(tmp_path / "adam.o", (1, 1))                 # older than its source
    assert compiled()[0] == 1
    os.remove(tmp_path / "adam.o.cmd")                    # of a build that noted no command
    assert compiled()[0] == 1
