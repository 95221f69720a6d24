"""The module of autograd functions is built beside the library, loads without a device and is missed loudly."""
import sys

import pytest

from alto_b200 import _lib as L


def test_module_loads_and_is_bound_once():
    module = L.autograd()
    assert module is L.autograd() and callable(module.rms_norm) and callable(module.rms_norm_residual)


def test_a_missing_module_fails_loudly(monkeypatch):
    import alto_b200
    monkeypatch.setattr(L, "_autograd_module", None)
    monkeypatch.delattr(alto_b200, "_autograd", raising=False)
    monkeypatch.setitem(sys.modules, "alto_b200._autograd", None)
    with pytest.raises(RuntimeError, match="python -m alto_b200.build"):
        L.autograd()
