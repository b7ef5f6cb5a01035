"""The compiled Python binding belongs to one PyTorch and one interpreter: another
one's is rebuilt, and refused when it is loaded.  No GPU needed."""
import sys

import pytest

from hsd_b200 import _native as N
from hsd_b200 import build as B


def test_binding_knows_what_it_is_built_for():
    import torch
    t = N.ops_target()
    assert torch.__version__ in t and sys.implementation.cache_tag in t
    assert N.ops().built_for == t


def test_another_versions_binding_is_refused(monkeypatch):
    monkeypatch.setattr(N, "_ops", None)
    monkeypatch.setattr(N, "ops_target", lambda: "torch 0.0, cpython-00")
    with pytest.raises(N.HSDNativeError, match="rebuild"):
        N.ops()


def test_another_versions_stamp_means_a_rebuild(monkeypatch, tmp_path):
    out, stamp = tmp_path / "_ops.so", tmp_path / "for.txt"
    out.write_bytes(b"")
    monkeypatch.setattr(B, "OPS", str(out))
    monkeypatch.setattr(B, "OPS_STAMP", str(stamp))
    assert not B._ops_up_to_date()              # no stamp: a build before there were any
    stamp.write_text(N.ops_target())
    assert B._ops_up_to_date()
    stamp.write_text(N.ops_target() + "x")
    assert not B._ops_up_to_date()
    assert B._ops_command("x.so").count("-o") == 1
    assert any(N.ops_target() in a for a in B._ops_command("x.so"))


def test_a_binding_that_does_not_say_is_refused(monkeypatch):
    import importlib.machinery

    class Loader:
        def create_module(self, spec):
            return None

        def exec_module(self, module):
            pass

    monkeypatch.setattr(N, "_ops", None)
    monkeypatch.setattr(N.importlib.util, "spec_from_file_location",
                        lambda name, path: importlib.machinery.ModuleSpec(name, Loader()))
    with pytest.raises(N.HSDNativeError, match="rebuild"):
        N.ops()
