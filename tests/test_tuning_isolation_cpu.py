"""A DGS_* override that a test sets past monkeypatch ends with the test (tests/conftest.py), in the environment and in the library's
snapshot of it.  The two tests run in this order."""
import os


def test_sets_an_override_and_leaves_it():
    os.environ['DGS_HUB_CHAIN'] = '2048'
    from dgsparse import _capi
    _capi.reload_tuning()
    assert _capi.hub_threshold() == 2048


def test_the_override_is_gone():
    assert 'DGS_HUB_CHAIN' not in os.environ
    from dgsparse import _capi
    assert _capi.hub_threshold() != 2048
