"""The build's two products (no GPU needed; nothing is compiled): the kernels' library does not depend on the torch binding."""
import importlib.util
import os
import types

import pytest

from conftest import PKG


@pytest.fixture
def built(tmp_path, monkeypatch):
    """build.py with its products in tmp_path and every compiler call replaced by writing its output."""
    spec = importlib.util.spec_from_file_location("mdx_build_under_test", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "OUT", str(tmp_path / "libmdx.so"))
    monkeypatch.setattr(mod, "BIND_OUT", str(tmp_path / "_bind.so"))
    monkeypatch.setattr(mod, "hipcc", lambda: "/opt/rocm/bin/hipcc")
    fail = []

    def run(cmd, **_):
        if any(f in " ".join(cmd) for f in fail):
            if "no such compiler" in fail:
                raise FileNotFoundError(cmd[0])
            return types.SimpleNamespace(returncode=1, stdout="", stderr="header not found")
        open(cmd[cmd.index("-o") + 1], "w").write("new")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod, fail, tmp_path


def test_both_products(built):
    mod, _, out = built
    mod.build()
    assert sorted(os.listdir(out)) == ["_bind.so", "libmdx.so"]


@pytest.mark.parametrize("how", ["header not found", "no such compiler"])
def test_a_binding_that_does_not_compile_leaves_the_library(built, how):
    """libmdx.so is there and new; the failure is still an error, and no binding of an earlier build stays."""
    mod, fail, out = built
    (out / "libmdx.so").write_text("old")
    (out / "_bind.so").write_text("old")
    fail += ["mdx_bind.cpp", how]
    with pytest.raises(RuntimeError, match="libmdx.so is built, _bind.so is not"):
        mod.build()
    assert (out / "libmdx.so").read_text() == "new" and not (out / "_bind.so").exists()


def test_a_kernel_that_does_not_compile_leaves_both(built):
    mod, fail, out = built
    (out / "libmdx.so").write_text("old")
    fail += ["mdx_pages.hip"]
    with pytest.raises(RuntimeError, match="compile failed"):
        mod.build()
    assert (out / "libmdx.so").read_text() == "old"


def test_the_binding_is_compiled_with_warnings(built, monkeypatch):
    mod, _, out = built
    seen = []
    inner = mod.subprocess.run
    monkeypatch.setattr(mod.subprocess, "run", lambda cmd, **kw: (seen.append(cmd), inner(cmd, **kw))[1])
    mod.build()
    bind = [c for c in seen if any("mdx_bind.cpp" in x for x in c)]
    assert len(bind) == 1 and "-w" not in bind[0] and "-Wall" in bind[0]
