"""CPU: the CU mask of the simulator's stream, and what happens where a driver refuses one."""
import warnings

import pytest

from gsc_amd.agents import BatchedTrainer


class Driver:
    """Refuses masks with ``text``, those of ``contiguous`` bits only where told so."""

    def __init__(self, text="hipExtStreamCreateWithCUMask: out of memory", contiguous=False):
        self.text, self.contiguous, self.asked = text, contiguous, []

    def create_cu_masked_stream(self, bits):
        self.asked.append(bits)
        if self.contiguous or bits != list(range(len(bits))):
            raise RuntimeError(self.text)
        return 77


@pytest.fixture(autouse=True)
def _auto_layout(monkeypatch):
    monkeypatch.delenv("GSC_SIM_CU_LAYOUT", raising=False)


def test_refused_small_spread_mask_gives_way_with_a_warning():
    nat = Driver()
    with pytest.warns(UserWarning, match="refuses 32 CUs"):
        assert BatchedTrainer.sim_stream_on(nat, 256, 32, True) == (77, list(range(32)))
    assert [len(b) for b in nat.asked] == [32, 32] and nat.asked[0][4] == 32


def test_accepted_masks_are_used_without_a_warning():
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert BatchedTrainer.sim_stream_on(Driver(), 256, 64, False) == (77, list(range(64)))


@pytest.mark.parametrize("nat,k,spread,layout", [
    (Driver(), 64, True, None),                                # 8 bits a block: the measured mask, which drivers take
    (Driver(), 32, True, "xcd"),                               # chosen by hand
    (Driver("HIP error invalid device in hipGetDevice"), 32, True, None),
    (Driver("gsc_amd native: CU index out of range"), 32, True, None),
    (Driver(contiguous=True), 32, False, None),                # contiguous already
    (Driver(contiguous=True), 32, True, None)])                # and refused as well
def test_other_failures_are_not_hidden(nat, k, spread, layout, monkeypatch):
    if layout:
        monkeypatch.setenv("GSC_SIM_CU_LAYOUT", layout)
    with warnings.catch_warnings(record=True), pytest.raises(RuntimeError):
        BatchedTrainer.sim_stream_on(nat, 256, k, spread)
