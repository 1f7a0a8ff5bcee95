"""The statistics of a plan, which reach the host some time after the plan is built: no GPU needed."""
import torch

from torchex_b200 import ScatterData


class _Event:
    asked = 0

    def query(self):
        self.asked += 1
        return True


class _Plan:
    max_cnt, has_empty, settled, no_split = -1, True, False, False


def _waiting(stats=(70, 0, 0, 0)):
    data = ScatterData.__new__(ScatterData)
    data._plan = _Plan()
    data._pending = (torch.tensor(stats, dtype=torch.int32), _Event())
    return data, data._pending[1]


def test_statistics_are_taken_over(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    data, event = _waiting()
    data._poll()
    assert event.asked == 1 and data._pending is None
    assert data._plan.max_cnt == 70 and data._plan.settled and not data._plan.has_empty


def test_no_event_is_asked_while_a_stream_is_captured(monkeypatch):
    """Asking an event is not permitted then, and would end the capture."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    data, event = _waiting()
    data._poll()
    assert event.asked == 0 and data._pending is not None
    assert data._plan.max_cnt == -1 and not data._plan.settled
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    data._poll()
    assert event.asked == 1 and data._plan.max_cnt == 70
