"""The build recipe: the flags give one binary, and a change of the flags rebuilds."""
import importlib
import os


def recipe():
    return importlib.import_module("sam-rs_b200.build")


def test_flags_give_one_binary():
    """Splitting a file's compilation over threads makes nvcc's register allocation differ from build to build."""
    assert not [f for f in recipe().FLAGS if "split-compile" in f]


def test_a_change_of_the_recipe_rebuilds(monkeypatch, tmp_path):
    """A library older than build.py (its flags) is stale; a newer one than every source is not."""
    b, ran = recipe(), []
    out = tmp_path / "lib.so"
    out.write_bytes(b"")
    monkeypatch.setattr(b, "OUT", str(out))
    monkeypatch.setattr(b.subprocess, "run", lambda cmd, check: ran.append(cmd) or open(cmd[cmd.index("-o") + 1], "w").close())
    newest = max(os.path.getmtime(p) for p in b.sources())
    os.utime(out, (newest + 1, newest + 1))
    b.build()
    assert not ran
    recipe_time = os.path.getmtime(os.path.join(b.HERE, "build.py"))
    others = [p for p in b.sources() if not p.endswith("build.py")]
    real = os.path.getmtime
    # every other source is old: only the recipe is newer than the library
    monkeypatch.setattr(b.os.path, "getmtime", lambda p: 1.0 if p in others else real(p))
    os.utime(out, (recipe_time - 1, recipe_time - 1))
    b.build()
    assert len(ran) == 1
