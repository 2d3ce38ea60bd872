"""The build recipe where the Python extension's compiler is missing."""
import os

import pytest

from q35hip import build


@pytest.mark.parametrize("cxx", ["/bin/false", "/no/such/compiler"])
def test_the_c_library_needs_no_host_compiler(cxx, tmp_path, monkeypatch):
    """The library is linked, a warning tells what failed, and no extension of an earlier build stays beside it."""
    monkeypatch.setenv("CXX", cxx)
    for name in ("BUILD_DIR", "LIB_PATH", "HOST_PATH"):
        monkeypatch.setattr(build, name, str(tmp_path / name))
    with open(build.HOST_PATH, "w") as f:
        f.write("an earlier build's")
    monkeypatch.setattr(build, "sources", lambda: [os.path.join(build.CSRC, "status.hip")])
    with pytest.warns(UserWarning, match="could not be built"):
        assert build.build() == build.LIB_PATH
    assert os.path.getsize(build.LIB_PATH) > 0 and not os.path.exists(build.HOST_PATH)
