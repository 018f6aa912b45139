"""The host-side checks of an adapter plan."""
from __future__ import annotations

import types

import pytest

from laya_js_b200 import _lib, adapters


@pytest.mark.parametrize("cu,ad,error", [([0.0, 1.5], [0], TypeError), ([0, 2], [0.5], TypeError), ([0, 2 ** 32 + 2], [0], ValueError),
                                         ([0, 2], [2 ** 32], ValueError), ([0, 2], [True], TypeError)])
def test_a_plan_takes_whole_numbers_of_32_bits(monkeypatch, cu, ad, error):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("reached the library"))
    with pytest.raises(error):
        adapters.AdapterPlan(types.SimpleNamespace(_destroyed=True), cu, ad, 1)
