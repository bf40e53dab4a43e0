"""The build of the library and of the Python module beside it; needs nvcc, no GPU. Everything is
built in a temporary folder."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path):
    """build.py with a small library of its own and the real module's source."""
    spec = importlib.util.spec_from_file_location("library_build", os.path.join(ROOT, "apex-tune-results_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    source = tmp_path / "small.cu"
    source.write_text("__global__ void kernel() {}\nextern \"C\" int answer() { return 42; }\n")
    b.SOURCES, b.HEADERS = [str(source)], {str(source): []}
    b.OBJ, b.OUT = str(tmp_path / "obj"), str(tmp_path / "libsmall.so")
    b.CALLS_OUT = str(tmp_path / "_calls.so")
    return b


def absent(name):
    return None


@pytest.mark.parametrize("what", ["compiler fails", "no compiler", "no torch"])
def test_the_library_needs_no_torch_and_no_cxx(build, monkeypatch, what):
    if what == "no torch":
        monkeypatch.setattr(build.importlib.util, "find_spec", absent)
    else:
        monkeypatch.setenv("CXX", "false" if what == "compiler fails" else "/nowhere/c++")
    with open(build.CALLS_OUT, "w") as f:
        f.write("of other sources")
    os.utime(build.CALLS_OUT, (0, 0))
    with pytest.warns(UserWarning, match="_calls.so"):
        assert build.build() == build.OUT
    assert os.path.exists(build.OUT) and not os.path.exists(build.CALLS_OUT)
    with pytest.raises(RuntimeError, match="_calls.so"):
        build.build(strict=True)


def test_a_library_that_does_not_compile_is_an_error(build):
    with open(build.SOURCES[0], "a") as f:
        f.write("this is no C++\n")
    with pytest.raises(RuntimeError, match="libapex_attn.so"):
        build.build()


def test_the_module_takes_its_abi_from_torch(build, monkeypatch):
    import torch
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}" in build.calls_command("x.so")
    monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: False)
    assert "-D_GLIBCXX_USE_CXX11_ABI=0" in build.calls_command("x.so")


def test_the_module_is_built_again_for_another_torch_or_compiler(build, monkeypatch):
    built = []
    real = build.subprocess.run

    def run(cmd, **kw):
        if "--version" in cmd:
            return real(cmd, **kw)
        built.append(cmd)
        open(build.CALLS_OUT + ".tmp", "w").close()
        return real(["true"], **kw)

    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_calls()
    build.build_calls()
    assert len(built) == 1
    for name, value in (("calls_key", "torch 1.2.3 cpython-399"), ("cxx", "cc")):
        monkeypatch.setattr(build, name, lambda value=value: value)
        before = len(built)
        build.build_calls()
        build.build_calls()
        assert len(built) == before + 1, name


def test_a_module_of_another_torch_is_left_out(monkeypatch):
    import apex_attn.paged as paged
    module = paged._import_calls()
    if not module:
        pytest.skip("_calls is not built")
    import torch
    assert module.built_for.startswith(f"torch {torch.__version__} ")
    monkeypatch.setattr(module, "built_for", "torch 1.2.3 cpython-399")
    with pytest.warns(UserWarning, match="torch 1.2.3"):
        assert paged._import_calls() is False
    monkeypatch.delattr(module, "built_for")
    with pytest.warns(UserWarning, match="unknown"):
        assert paged._import_calls() is False


def test_the_built_module_is_the_one_for_this_torch(build):
    import apex_attn.paged as paged
    module = paged._import_calls()
    if not module:
        pytest.skip("_calls is not built")
    assert module.built_for == build.calls_key()
