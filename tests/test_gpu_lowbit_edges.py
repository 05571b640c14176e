"""The low-bit operators at the ends of their ranges and on their rarer paths, on the GPU against the definitions in 64 bits
(lowbit_ref.py).  Tolerances are those of test_gpu_lowbit.py unless a test derives its own (u = 2^-24)."""
import pytest
import torch

from test_gpu_lowbit import _check_store, _cuda_cache, _filled, eng  # noqa: F401
from whisperdrz_b200.capi import WdzError

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ what is reported
def _misplaced_store(eng):
    c = _cuda_cache(_filled(2, 2, 1))
    rows = torch.zeros(1, 128, device="cuda")
    eng.qcache_store(c, rows, rows, torch.tensor([0], dtype=torch.int32).cuda(), torch.tensor([64], dtype=torch.int32).cuda())


def test_a_store_that_cannot_be_placed_leaves_a_transcription_alone(eng):
    """The decode loop's poll hears of its own kernels only, and what it leaves is told by device_status."""
    _misplaced_store(eng)
    eng.ts_poll()
    eng.decode_status()
    with pytest.raises(WdzError) as err:
        eng.device_status()
    assert "WDZ_EINVAL" in str(err.value)
    eng.device_status()


def test_each_kind_of_report_is_told_and_a_wait_that_ran_out_first(eng):
    """No kernel is made to hang: the words are set as one would leave them (the engine's own, the operators' waits, the
    operators' data)."""
    words = eng.workspace[:24].view(torch.int32).view(3, 2)
    assert (words == 0).all()
    _misplaced_store(eng)
    words[1, 0], words[1, 1] = -7, 2000005
    words[0, 0] = -6
    for name in ("WDZ_ETIMEOUT", "WDZ_ENAN", "WDZ_EINVAL"):
        with pytest.raises(WdzError) as err:
            eng.device_status()
        assert name in str(err.value)
    eng.device_status()
    words[0, 0] = -6
    with pytest.raises(WdzError) as err:
        eng.ts_poll()
    assert "WDZ_ENAN" in str(err.value)
    eng.ts_poll()
    eng.device_status()


# ---------------------------------------------------------------------- store
def test_store_of_a_padded_batch(eng):
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(9, 128, generator=g)
    for device_index in (True, False):
        _check_store(eng, _filled(3, 2, 1), rows[:4], rows[4:8], [2, -1, -1, 0], [5, 0, 0, 9], device_index=device_index)
        _check_store(eng, _filled(3, 2, 1), rows, rows.flip(0), [1, 3, 3, -1, -1], [5, 0, 0, 9, 70], [0, 4, 5, 6, 8, 9], device_index=device_index)
    eng.device_status()
