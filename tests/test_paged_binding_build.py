"""The torch binding of the paged cache operators as a build product: libtir.so does not
depend on it, and it is compiled again for, and refused by, another torch or Python."""
import os
import sys
import types

import pytest


@pytest.fixture
def elsewhere(tirlib, tmp_path, monkeypatch):
    """The build module with its products in tmp_path and no C++ compiler."""
    pytest.importorskip("torch")
    from tir import build
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_paged_bind.so"))
    monkeypatch.setattr(build, "BIND_STAMP", str(tmp_path / "stamp"), raising=False)
    monkeypatch.setenv("CXX", "/bin/false")
    return build


def test_the_library_is_linked_where_the_binding_does_not_compile(elsewhere, tmp_path, monkeypatch, capfd):
    monkeypatch.setattr(elsewhere, "LIB", str(tmp_path / "libtir.so"))
    for cxx in ("/bin/false", str(tmp_path / "no-such-compiler")):
        monkeypatch.setenv("CXX", cxx)
        assert elsewhere.build() == elsewhere.LIB and os.path.exists(elsewhere.LIB)
        assert "binding" in capfd.readouterr().err
        with pytest.raises(RuntimeError, match="compile failed"):
            elsewhere.build_bind()


def test_the_binding_is_compiled_again_for_another_torch_or_python(elsewhere, monkeypatch):
    for p in (elsewhere.BIND, elsewhere.BIND_STAMP):
        with open(p, "w") as f:
            f.write(elsewhere._bind_target() if p == elsewhere.BIND_STAMP else "")
    assert elsewhere.build_bind() == elsewhere.BIND  # up to date: no compiler is run
    for other in ("torch 0.0, " + elsewhere._bind_target().split(", ")[1], elsewhere._bind_target() + "d"):
        with open(elsewhere.BIND_STAMP, "w") as f:
            f.write(other)
        with pytest.raises(RuntimeError, match="compile failed"):
            elsewhere.build_bind()
    os.remove(elsewhere.BIND_STAMP)
    with pytest.raises(RuntimeError, match="compile failed"):
        elsewhere.build_bind()


@pytest.mark.parametrize("found", ["for another torch", "of an earlier build", "nothing"])
def test_a_binding_that_does_not_fit_is_refused_on_first_use(tirlib, monkeypatch, found):
    torch = pytest.importorskip("torch")
    module = {"for another torch": types.SimpleNamespace(built_for="0.0"), "of an earlier build": types.SimpleNamespace(),
              "nothing": None}[found]
    monkeypatch.setattr(tirlib, "_bind_module", None)
    monkeypatch.setitem(sys.modules, "tir._paged_bind", module)
    if hasattr(tirlib, "_paged_bind"):
        monkeypatch.delattr(tirlib, "_paged_bind")
    x = torch.zeros(1, 1, 64)
    with pytest.raises(ImportError, match="torch binding .* build it"):
        tirlib.qk_norm_rope(x, x, x, x, None)
    assert tirlib._bind_module is None
