"""A rebuild in a process that has loaded the library: the next call loads the
new file, the one that the compiled host path would load too."""

import os
import shutil

from cube_awq_b200 import _lib, build


def test_a_rebuilt_library_is_loaded_anew(tmp_path, monkeypatch):
    path = str(tmp_path / "libcube_awq.so")
    shutil.copy(_lib.LIB_PATH, path)
    for module in (_lib, build):
        monkeypatch.setattr(module, "LIB_PATH", path)
    monkeypatch.setattr(_lib, "_lib", None)
    before = _lib.lib()
    assert _lib.lib() is before

    class Done:
        returncode = 0

    def link(cmd, **_):
        shutil.copy(before._name, cmd[cmd.index("-o") + 1])
        return Done()

    monkeypatch.setattr(build, "_compile", lambda src, verbose, extra: src)
    monkeypatch.setattr(build.subprocess, "run", link)
    inode = os.stat(path).st_ino
    assert build.build(force=True) == path
    assert os.stat(path).st_ino != inode
    after = _lib.lib()
    assert after is not before and after._handle != before._handle
    assert after.cawq_version() == before.cawq_version()
