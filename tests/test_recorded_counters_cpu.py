"""Counters of recorded one-launch reductions, two threads recording at once (no GPU: the bookkeeping alone)."""
import threading

import torch


def test_two_recording_threads_get_different_counters(monkeypatch):
    """The first thread to advance the pool is held there until a second one has been through, or cannot get in."""
    from maskplanner_amd import ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    device, second_done = torch.device("cpu"), threading.Event()

    class Pool(list):
        held = False

        def __setitem__(self, i, v):
            super().__setitem__(i, v)
            if not self.held:
                self.held = True
                second_done.wait(1.0)
    monkeypatch.setattr(ops, "_RECORDED_COUNTERS", {device: Pool([torch.zeros(8, dtype=torch.int32), 0, []])})
    taken = []

    def first():
        taken.append(ops._reduce_counter(device))

    def second():
        while not ops._RECORDED_COUNTERS[device].held:
            pass
        taken.append(ops._reduce_counter(device))
        second_done.set()
    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(taken) == 2 and taken[0].data_ptr() != taken[1].data_ptr()
