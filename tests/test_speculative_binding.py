"""The package without its compiled binding: only the calls that go through it fail. No GPU needed."""

from __future__ import annotations

import importlib.util
import os
import sysconfig

import pytest

from mini_inference_b200 import _lib, build


def load_lib(folder):
    """_lib.py as it would be imported from `folder`, which holds libpkv.so."""
    (folder / "_lib.py").write_text((_lib.LIB_PATH.parent / "_lib.py").read_text())
    os.symlink(_lib.LIB_PATH, folder / _lib.LIB_PATH.name)
    spec = importlib.util.spec_from_file_location("pkv_lib_without_binding", folder / "_lib.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_other_operators_do_without_it(tmp_path):
    mod = load_lib(tmp_path)
    assert mod.lib.pkv_version() == _lib.lib.pkv_version()
    for _ in range(2):  # every call says so
        with pytest.raises(ImportError, match="not built"):
            mod.speculative.tree_attention()


def test_one_that_does_not_load_is_named(tmp_path):
    name = "_speculative" + sysconfig.get_config_var("EXT_SUFFIX")
    (tmp_path / name).write_bytes(b"no shared object")
    mod = load_lib(tmp_path)
    with pytest.raises(ImportError, match="does not load"):
        mod.speculative.rotary_append()


def test_its_file_belongs_to_one_python_and_one_torch():
    assert build.BINDING.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    assert set(vars(_lib.speculative)) <= {"extend_tables", "build_tree_metadata", "rotary_append", "tree_attention", "accept_tree"}
    assert callable(_lib.speculative.accept_tree)
    with pytest.raises(AttributeError):
        _lib.speculative.no_such_call
