import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, 'dgsparse-lib_amd')):
    if p not in sys.path:
        sys.path.insert(0, p)


collect_ignore_glob = ['_dryrun/*', '_dryrun']  # tests/gpu_dryrun.py's scratch copies (same module names): never collected from here


def pytest_configure(config):
    config.addinivalue_line('markers', 'gpu: needs a real MI355X (run with -m gpu on the GPU box)')
    config.addinivalue_line('markers', 'first_contact: written in rounds 4 / 5 while the GPU pool was closed - never run on hardware: '
                            'tests that force or assert a schedule resting on hardware behaviour no CPU test sees (hub chains, '
                            'in-kernel fold, the device gate) and the other tests added since the last green GPU run (round 3) - '
                            'collected LAST, so that under `-x` a failure there cannot hide the suite that has run green before')


def _has_gpu():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


# Tests that hold a wrong value, kept as they are: name -> the proof (and the test that holds the right one).
HOLDS_A_WRONG_VALUE = {
    'test_storage_tells_the_launches_its_longest_row_and_column': 'sets DGS_HUB_CHAIN=200 and takes a row of 280 for a hub row; the threshold is clamped to '
                                                                 '1024 and above (include/dgsparse_hip.h), so the row is none and keeps its hint (test_gpu_hub_hints.py: the same with 1300 and 1024)',
}


def pytest_collection_modifyitems(config, items):
    for item in items:
        if item.name in HOLDS_A_WRONG_VALUE:
            item.add_marker(pytest.mark.xfail(reason=HOLDS_A_WRONG_VALUE[item.name], strict=True))
    # stable: everything else keeps its file / definition order, the first-contact tests move behind it (the driver runs
    # `pytest -x`: the library's default is protected by the device self-test, the tests that FORCE the gated schedules are not)
    items.sort(key=lambda it: 1 if 'first_contact' in it.keywords else 0)
    if _has_gpu():
        return
    skip = pytest.mark.skip(reason='no GPU in this container')
    for item in items:
        if 'gpu' in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def _dgs_tuning_follows_env(monkeypatch):
    """The library snapshots its DGS_* tuning overrides once per process (no getenv() on the launch path); tests flip them
    through monkeypatch, so every DGS_* change made that way - and the restore at teardown - is followed by a reload."""
    try:
        from dgsparse import _capi
    except Exception:  # CPU-only collection of tests that never import the package
        yield
        return
    before = {k: v for k, v in os.environ.items() if k.startswith('DGS_')}
    setenv, delenv = monkeypatch.setenv, monkeypatch.delenv

    def _setenv(name, value, *a, **k):
        setenv(name, value, *a, **k)
        if name.startswith('DGS_'):
            _capi.reload_tuning()

    def _delenv(name, *a, **k):
        delenv(name, *a, **k)
        if name.startswith('DGS_'):
            _capi.reload_tuning()

    monkeypatch.setenv, monkeypatch.delenv = _setenv, _delenv
    yield
    monkeypatch.undo()
    # (a test that sets them past monkeypatch - the seeded fuzz slice does for each of its cases, and how many it gets through in its time
    # decides what the last one leaves - does not hand them on to the next)
    for k in [k for k in os.environ if k.startswith('DGS_') and k not in before]:
        del os.environ[k]
    os.environ.update(before)
    _capi.reload_tuning()
