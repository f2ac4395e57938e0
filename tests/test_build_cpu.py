"""What is built where a part of the build cannot be."""

import pytest

from fuselse_amd import _build


@pytest.mark.parametrize("why", [RuntimeError("g++ failed"), ImportError("No module named torch")])
def test_the_c_libraries_do_not_need_torch(monkeypatch, tmp_path, why):
    """libfuselse_amd.so and the measurement library are linked where the calls over
    torch's C++ API cannot be compiled, and the build says so."""
    made = []

    def no_torch(src, verbose):
        raise why

    monkeypatch.setattr(_build, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(_build, "_compile", lambda src, verbose: src)
    monkeypatch.setattr(_build, "_compile_torch", no_torch)
    monkeypatch.setattr(_build, "_link", lambda objs, out, extra, verbose: made.append(out))
    with pytest.raises(type(why)):
        _build.build()
    assert made == [_build.LIB_PATH, _build.DIAG_LIB_PATH]
