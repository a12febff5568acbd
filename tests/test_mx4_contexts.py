"""Which context an MXFP4 entry point runs on, with stand-ins for the library's contexts: no GPU."""
import gc
import threading

import pytest

from oxidized_gpt_oss_b200 import abi, mxfp4


class Lib:
    @staticmethod
    def oxg_ctx_set_stream(handle, stream):
        handle.append(stream)
        return abi.OXG_OK


class Context:
    """Remembers its device, the streams that it was put on and whether it was ended."""
    made, ended = [], []

    def __init__(self, device=0):
        self.device, self.lib, self.handle, self.number = device, Lib, [], len(self.made)
        self.made.append(self.number)

    def __del__(self):
        self.ended.append(self.number)


class On:
    """What device_context asks of a tensor."""

    def __init__(self, index):
        self.device = self.index = index

    def get_device(self):
        return self.index


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    Context.made, Context.ended = [], []
    monkeypatch.setattr(abi, "Context", Context)
    monkeypatch.setattr(mxfp4, "_raw_stream", lambda device: (threading.get_ident(), device))
    monkeypatch.setattr(mxfp4.torch.cuda, "current_device", lambda: 0)
    for name, value in (("_default_ctx", None), ("_device_ctx", {}), ("_thread_ctx", {})):
        monkeypatch.setattr(mxfp4, name, value, raising=False)


def in_thread(fn):
    got = []
    t = threading.Thread(target=lambda: got.append(fn()))
    t.start()
    t.join()
    return got[0]


def test_a_threads_context_outlives_it():
    """What a thread captured keeps reporting to its context, and no thread's end frees or waits for anything."""
    number = in_thread(lambda: mxfp4.device_context(On(0), None).number)
    gc.collect()
    assert number in Context.made and not Context.ended


def test_threads_have_a_context_each_and_take_over_those_of_ended_ones():
    gate = threading.Barrier(4)
    seen = []

    def work():
        mine = mxfp4.device_context(On(0), None)
        gate.wait()  # all four are alive
        assert mxfp4.device_context(On(0), None) is mine
        assert mxfp4.device_context(On(1), None) is not mine
        seen.append(mine.number)

    for _ in range(20):
        ts = [threading.Thread(target=work) for _ in range(4)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
    for i in range(0, 80, 4):
        assert len(set(seen[i: i + 4])) == 4
    assert mxfp4.device_context(On(0), None).number not in seen
    assert not Context.ended
