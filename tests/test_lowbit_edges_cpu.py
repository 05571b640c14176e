"""CPU checks of the low-bit operators' host side: what is refused, what is let through, and what the scheduler asks for."""
import torch

from test_scheduler_cpu import StubEngine, _patch_rules_dev
from whisperdrz_b200.transcriber import Transcriber


def test_scheduler_asks_for_the_decode_loop_s_own_status():
    """A report of the operators on caller-held memory, which device_status would raise, is no failed decode step."""
    class Engine(StubEngine):
        asked = 0

        def device_status(self):
            raise AssertionError("the operators' reports are not the scheduler's")

        def decode_status(self):
            self.asked += 1

    eng = Engine()
    tr = Transcriber(eng, max_new_tokens=10, max_continuations=0)
    _patch_rules_dev(tr)
    assert len(tr.transcribe(torch.randn(16000 * 30)).raw_chunks) == 1
    assert eng.asked > 0
