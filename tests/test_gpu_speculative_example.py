"""examples/speculative_layer.py: a layer served with draft trees gives what the
same tokens give one by one, and its cache the same bits."""
import importlib.util
import os

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
def test_speculative_layer(bits):
    path = os.path.join(ROOT, "examples", "speculative_layer.py")
    spec = importlib.util.spec_from_file_location("speculative_layer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(["--bits", str(bits), "--steps", "5"])
