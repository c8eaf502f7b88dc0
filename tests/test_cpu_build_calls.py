"""The module of short calls is compiled against PyTorch's headers: another PyTorch (or Python) has it built anew, and one that was built for another is not used."""
import os

import pytest
import torch

from them_bones_b200.csrc import build as B
from them_bones_b200.ops import _lib as L


def test_another_pytorch_has_it_built_anew(monkeypatch):
    B.build_calls()
    ran = []
    monkeypatch.setattr(B.subprocess, "run", lambda *a, **k: ran.append(a) or pytest.fail("compiled"))
    assert B.build_calls() == B.CALLS and not ran              # current: nothing to do
    compiled = []

    class Done:
        returncode, stdout, stderr = 1, "", ""

    monkeypatch.setattr(B.subprocess, "run", lambda *a, **k: compiled.append(a) or Done())
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    with pytest.raises(RuntimeError):                          # the stand-in for the compiler fails: what was there stays, and is not taken for the other's
        B.build_calls()
    assert len(compiled) == 1 and os.path.exists(B.CALLS)
    with pytest.raises(RuntimeError):
        B.build_calls()
    assert len(compiled) == 2


@pytest.mark.skipif(not os.path.exists(L.lib_path()), reason="the library is not built")
def test_one_built_for_another_pytorch_is_not_used(monkeypatch):
    B.build_calls()
    monkeypatch.setattr(L, "_CALLS", None)
    assert L.calls().built_with() == B.calls_for()
    monkeypatch.setattr(L, "_CALLS", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    with pytest.raises(RuntimeError, match="9.9.9"):
        L.calls()
