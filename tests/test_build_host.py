"""Building the extension module beside the kernel library (CPU only, nothing is compiled)."""
import importlib.util
import os
import types

import pytest

from conftest import PACKAGE_ROOT


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """csrc/build.py with its outputs in a folder of the test and a recorder in the place of the compilers."""
    spec = importlib.util.spec_from_file_location("csrc_build", os.path.join(PACKAGE_ROOT, "csrc", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for name in ("OBJDIR", "OUTPUT", "HOST_OUTPUT"):
        monkeypatch.setattr(module, name, str(tmp_path / name))
    module.ran, module.fails = [], {}

    def run(cmd, **kwargs):
        tool = os.path.basename(cmd[0])
        module.ran.append((tool, cmd))
        if isinstance(module.fails.get(tool), Exception):
            raise module.fails[tool]
        if tool not in module.fails:
            with open(cmd[cmd.index("-o") + 1], "w") as f:
                f.write("x")
        return types.SimpleNamespace(returncode=int(tool in module.fails), stderr=module.fails.get(tool, ""), stdout="")

    monkeypatch.setattr(module.subprocess, "run", run)
    monkeypatch.delenv("CXX", raising=False)
    return module


@pytest.mark.parametrize("failure", ["Python.h: No such file or directory", FileNotFoundError("g++")])
def test_the_kernel_library_does_not_need_the_extension_module(builder, failure, capsys):
    builder.fails["g++"] = failure
    assert builder.build() == builder.OUTPUT and os.path.exists(builder.OUTPUT)
    assert [t for t, _ in builder.ran].count("g++") == 1 and not os.path.exists(builder.HOST_OUTPUT)
    assert "_host_tensors" in capsys.readouterr().err
    with pytest.raises((RuntimeError, OSError)):
        builder.build_host()


def test_a_kernel_that_does_not_compile_ends_the_build(builder):
    builder.fails["nvcc"] = "error"
    with pytest.raises(RuntimeError, match="nvcc"):
        builder.build()


def test_the_extension_module_is_built_again_for_another_torch(builder, monkeypatch):
    """Whatever the installed files' times: an older torch may be installed after a newer one."""
    import torch
    builds = lambda: [t for t, _ in builder.ran].count("g++")  # noqa: E731
    for k in (1, 1):
        builder.build()
        assert builds() == k and os.path.exists(builder.HOST_OUTPUT)
    monkeypatch.setattr(torch, "__version__", "2.0.0")
    builder.build()
    builder.build()
    assert builds() == 2
    assert any("2.0.0" in x for x in builder.ran[-1][1] if x.startswith("-DICTC"))


def test_an_extension_module_for_another_torch_is_not_used(monkeypatch):
    import torch
    from ictc_o3.backends.cuda import _native
    assert _native.host_tensors().torch_version == torch.__version__
    monkeypatch.setattr(torch, "__version__", "2.0.0")
    with pytest.raises(_native.NativeError, match="another torch"):
        _native.host_tensors()
