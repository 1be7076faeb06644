"""Host logic around the gated linear scans' fault mirror (no GPU needed)."""

from __future__ import annotations

import numpy as np
import pytest

import gru_qat_amd as G
from gru_qat_amd import _lib


@pytest.fixture
def mirrors(monkeypatch):
    """Two devices' words, and the devices that were synchronised."""
    words = {i: np.zeros(1, dtype=np.int32) for i in (0, 3)}
    monkeypatch.setattr(_lib, "_mirrors", {(i, _lib._GATED_SCAN): (None, w) for i, w in words.items()})
    waited = []
    monkeypatch.setattr(_lib.torch.cuda, "synchronize", waited.append)
    monkeypatch.setattr(_lib, "_ws_cache", {})
    return words, waited


class _Dev:
    def __init__(self, index):
        self.index = index


def test_a_fault_is_raised_once(mirrors):
    words, _ = mirrors
    _lib.raise_scan_fault(0, "probe")
    _lib.raise_scan_fault(1, "probe")  # a device without a mirror
    words[3][0] = 18
    _lib.raise_scan_fault(0, "probe")
    with pytest.raises(G.PersistentScanFault, match="probe.*fault value 18"):
        _lib.raise_scan_fault(3, "probe")
    _lib.raise_scan_fault(3, "probe")


def test_check_faults_sees_it(mirrors):
    words, _ = mirrors
    words[3][0] = 2
    G.check_faults(_Dev(0))
    with pytest.raises(G.PersistentScanFault):
        G.check_faults()
    G.check_faults()


def test_workspace_faults_counts_and_clears_it(mirrors):
    words, waited = mirrors
    words[0][0] = words[3][0] = 7
    assert G.workspace_faults(_Dev(3)) == 1 and waited == [3] and words[0][0] == 7
    assert G.workspace_faults() == 1 and waited == [3, 0, 3]
    assert G.workspace_faults() == 0
