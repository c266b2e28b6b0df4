"""The in-tree build: what makes an object stale."""
import os

import build


def test_an_object_of_another_command_is_stale(tmp_path):
    src, obj = tmp_path / "a.hip", tmp_path / "a.hip.o"
    src.write_text("")
    cmd = ["hipcc", "-O3", "-c", str(src)]
    assert build._stale(str(obj), [str(src)], cmd)                     # not there
    obj.write_text("")
    assert build._stale(str(obj), [str(src)], cmd)                     # made by an unknown command
    build._made(str(obj), cmd)
    assert not build._stale(str(obj), [str(src)], cmd)
    assert build._stale(str(obj), [str(src)], cmd + build.NO_PACKED_FP32)
    os.utime(src, (os.path.getmtime(obj) + 10,) * 2)
    assert build._stale(str(obj), [str(src)], cmd)
