"""Build freshness (llm-inference_b200/build.py): the library is reused only
when the hash of its sources, headers, flags and nvcc version matches the one
recorded at link time. CPU only (nothing is compiled here unless the library
is missing or stale)."""
import os

from _util import load_build_module


def test_hash_recorded_and_reused():
    b = load_build_module()
    b.build(quiet=True)
    assert os.path.exists(b.LIB) and os.path.exists(b.STAMP)
    assert b.built_hash() == b.source_hash()
    assert not b.needs_build()


def test_hash_covers_flags_and_is_path_independent(monkeypatch):
    b = load_build_module()
    h0 = b.source_hash()
    assert h0 == b.source_hash()                 # deterministic
    monkeypatch.setattr(b, "NVCC_FLAGS", b.NVCC_FLAGS + ["-DB2_SOMETHING_ELSE"])
    assert b.source_hash() != h0                 # a flag change forces a rebuild
    monkeypatch.undo()
    # checkout paths are hashed relative to the repository root
    assert all(b.REPO_ROOT not in f.replace(b.REPO_ROOT, ".") for f in b.NVCC_FLAGS)


def test_stale_stamp_means_rebuild(monkeypatch):
    b = load_build_module()
    monkeypatch.setattr(b, "built_hash", lambda: "0" * 64)
    assert b.needs_build()


def test_the_library_does_not_wait_for_the_python_module(monkeypatch, tmp_path, capsys):
    """Without Python's headers or g++ the C library is built and the message says what is not."""
    b = load_build_module()
    src = tmp_path / "one.cu"
    src.write_text('extern "C" int one() { return 1; }\n')
    for name, path in (("LIB", "lib.so"), ("STAMP", "lib.so.sha256"), ("NATIVE", "_native.so"),
                       ("NATIVE_STAMP", "_native.so.sha256"), ("BUILD", "obj")):
        monkeypatch.setattr(b, name, str(tmp_path / path))
    monkeypatch.setattr(b, "sources", lambda: [str(src)])
    monkeypatch.setattr(b, "_python_include", lambda: str(tmp_path / "nowhere"))
    assert b.build() == b.LIB and os.path.exists(b.LIB) and b.built_hash() == b.source_hash()
    assert not os.path.exists(b.NATIVE) and b.needs_build()
    out = capsys.readouterr().out
    assert "compiled" in out and "Python.h" in out
    which = b.shutil.which
    monkeypatch.setattr(b.shutil, "which", lambda c: None if c == "g++" else which(c))
    b.build()
    out = capsys.readouterr().out
    assert "reused" in out and "no g++" in out
    # with both, the module alone is compiled
    monkeypatch.undo()
    c = load_build_module()
    for name, path in (("LIB", "lib.so"), ("STAMP", "lib.so.sha256"), ("NATIVE", "_native.so"),
                       ("NATIVE_STAMP", "_native.so.sha256"), ("BUILD", "obj")):
        monkeypatch.setattr(c, name, str(tmp_path / path))
    monkeypatch.setattr(c, "sources", lambda: [str(src)])
    c.build()
    assert "reused" in capsys.readouterr().out and os.path.exists(c.NATIVE) and not c.needs_build()


def test_another_interpreter_builds_its_module_only(monkeypatch):
    b = load_build_module()
    lib, native = b.source_hash(), b.native_hash()
    get = b.sysconfig.get_config_var
    monkeypatch.setattr(b.sysconfig, "get_config_var", lambda k: "cpython-399" if k == "SOABI" else get(k))
    assert b.source_hash() == lib and b.native_hash() != native
    monkeypatch.undo()
    monkeypatch.setattr(b, "CXX_FLAGS", b.CXX_FLAGS + ["-DB2_SOMETHING_ELSE"])
    assert b.source_hash() == lib and b.native_hash() != native
    assert b.NATIVE.endswith(b.sysconfig.get_config_var("EXT_SUFFIX"))
