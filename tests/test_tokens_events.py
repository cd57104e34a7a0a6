"""A timed plan's events: the start event in front of the first launch of its entry point, the stop event behind the last.

An event that is recorded on the stream behind a plan comes 4.2 to 4.4 us after the stop event, whatever the plan; one in front of it,
when the stream has work, 5 to 6 before the start event.  Every launch takes 4 us at least: an event that belongs to another
launch is further away by that.
"""

import ctypes
import statistics

import pytest
import torch

from test_tokens import BF16, F16, F32, ops  # noqa: F401
from test_tokens_edges import calls

SLACK = 2.5  # us; the events around one plan were 0.2 us apart from call to call


class Events:
    def __init__(self, lib):
        from nengo_ocl_amd import _lib

        self.lib, self.check, self.made = lib, _lib.check, []

    def record(self, handle):
        event = ctypes.c_void_p()
        self.check(self.lib.nhip_event_create(ctypes.byref(event)))
        self.made.append(event)
        self.check(self.lib.nhip_event_record(event, handle))
        return event

    def between(self, a, b):
        ms = ctypes.c_float()
        self.check(self.lib.nhip_event_elapsed_ms(a, b, ctypes.byref(ms)))
        return 1e3 * ms.value

    def destroy(self):
        for event in self.made:
            self.lib.nhip_event_destroy(event)


def around(queue, plan):
    """us: from an event in front of the plan to its start event, its own time, from its stop event to one behind; and the time
    per call of ten calls in a row."""
    events, load = Events(queue.lib), torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    try:
        rows = []
        plan()
        torch.cuda.synchronize()
        for _ in range(9):
            with torch.cuda.stream(queue.stream):  # (some 200 us: the device is behind the host when the plan comes)
                load.zero_()
            a = events.record(queue.handle)
            plan.enqueue(profiling=True)
            b = events.record(queue.handle)
            queue.finish()
            start, stop = plan._events_to_profile[-1]
            rows.append((events.between(a, start), events.between(start, stop), events.between(stop, b)))
        plan.update_profiling()
        with torch.cuda.stream(queue.stream):
            load.zero_()
        a = events.record(queue.handle)
        for _ in range(10):
            plan.enqueue()
        b = events.record(queue.handle)
        queue.finish()
        before, own, after = zip(*rows)
        return min(before), statistics.median(own), min(after), events.between(a, b) / 10
    finally:
        events.destroy()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", [(BF16, 300, 520, 9001), (F16, 300, 520, 9001), (F32, 300, 130, 310), (BF16, 9000, 1024, 2000),
                                            (F16, 40, 72, 257)])
def test_events_are_those_of_the_first_and_last_launch(queue, ops, dtype, n, d, v):  # noqa: F811
    made = {name: make(**given) for name, (given, make) in calls(ops, queue, 111, dtype, n, d, v).items()}
    one = around(queue, made["norm"])  # a single launch
    for name, plan in made.items():
        before, own, after, outside = around(queue, plan)
        assert before <= one[0] + SLACK, (name, before, one)
        assert after <= one[2] + SLACK, (name, after, one)
        assert own >= 0.5 * outside, (name, own, outside)
