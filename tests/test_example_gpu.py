"""The example that serves and trains adapters by request runs and learns."""
import importlib.util

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_adapters_by_request():
    spec = importlib.util.spec_from_file_location("adapters_by_request", ROOT / "examples" / "adapters_by_request.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.main(40)
    assert losses[-1] < 0.5 * losses[0], losses
