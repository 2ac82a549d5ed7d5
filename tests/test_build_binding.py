"""The build of the torch binding: left out without torch, made again for
another one (no compiler is run)."""
import importlib.util
import os
import sys

import pytest

from vibethinker_webgpu_lora_b200 import build as B
from vibethinker_webgpu_lora_b200 import kernels as K


@pytest.fixture
def ran(monkeypatch, tmp_path):
    """Commands that a build would run; the binding's own files under tmp_path."""
    cmds = []
    monkeypatch.setattr(B, "_run", lambda cmd, verbose: cmds.append(cmd))
    monkeypatch.setattr(B, "OPS", str(tmp_path / "_ops.so"))
    monkeypatch.setattr(B, "OPS_TORCH", str(tmp_path / "_ops.torch"))
    return cmds


def test_the_library_builds_without_torch(ran, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it fails
    assert B.build() == B.LIB
    assert B.build_ops() is None
    assert not any("eg_torch.cpp" in str(c) for c in ran)
    assert "without" in capsys.readouterr().err


def test_the_binding_is_built_again_for_another_torch(ran, monkeypatch):
    assert B.build_ops() == B.OPS and len(ran) == 1  # none yet
    open(B.OPS, "w").close()
    assert B.build_ops() == B.OPS and len(ran) == 1  # as it is
    with open(B.OPS_TORCH, "w") as f:
        f.write("1.0.0 /elsewhere/torch/__init__.py")
    assert B.build_ops() == B.OPS and len(ran) == 2
    assert B.build_ops() == B.OPS and len(ran) == 2


def test_a_build_that_fails_is_tried_again(ran, monkeypatch):
    def fails(cmd, verbose):
        ran.append(cmd)
        raise RuntimeError("no compiler")
    monkeypatch.setattr(B, "_run", fails)
    open(B.OPS, "w").close()
    for i in (1, 2):
        with pytest.raises(RuntimeError):
            B.build_ops()
        assert len(ran) == i


def test_a_missing_binding_says_what_to_do(monkeypatch):
    monkeypatch.setattr(K, "_native", None)
    monkeypatch.setitem(sys.modules, "vibethinker_webgpu_lora_b200._ops", None)
    import vibethinker_webgpu_lora_b200 as E
    monkeypatch.delattr(E, "_ops", raising=False)
    with pytest.raises(ImportError, match="build"):
        K.sample_filtered(None, None, None)


def test_the_binding_is_of_this_python():
    assert os.path.exists(B.OPS) and B.OPS.endswith(importlib.machinery.EXTENSION_SUFFIXES[0])
