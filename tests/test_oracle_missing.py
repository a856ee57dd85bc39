"""A test that calls the reference's library where it cannot be built is skipped, not failed."""
import unittest

import pytest

from oracle import pyoracle as po


def test_a_missing_reference_skips(monkeypatch, tmp_path):
    monkeypatch.setattr(po, "_libs", {})
    monkeypatch.setattr(po, "REF_SO", str(tmp_path / "absent.so"))
    monkeypatch.setattr(po, "REF_SRC", "")
    assert not po.have_ref()
    for call in (lambda: po._lib("ref"), lambda: po.ref_model_forward([2], 4, 4, 2, 1, 1, {}, None)):
        with pytest.raises(unittest.SkipTest):   # which a test run counts as a skip
            call()
