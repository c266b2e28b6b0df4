"""The in-tree build: what makes an object stale, and which kernels may not spill."""
import os

import pytest

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


def remarks(*sizes):
    return "".join("x.hip:1:1: remark: Function Name: _Z18ortho_small_kernelILi64ELi%dEE [-R]\nx.hip:1:1: remark:     VGPRs: 240 [-R]\n"
                   "x.hip:1:1: remark:     ScratchSize [bytes/lane]: %d [-R]\n" % (i, s) for i, s in enumerate(sizes))


def test_kernels_that_may_not_spill():
    other = "r: Function Name: _Z5other [-R]\nr:     ScratchSize [bytes/lane]: 40 [-R]\n"
    build._check_scratch(other + remarks(0, 0) + other, "ortho_small_kernel")
    with pytest.raises(RuntimeError, match="ILi64ELi1EE"):
        build._check_scratch(remarks(0, 108, 0), "ortho_small_kernel")
    with pytest.raises(RuntimeError, match="no ortho_small_kernel"):
        build._check_scratch(other, "ortho_small_kernel")
