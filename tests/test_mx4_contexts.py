"""Which context an MXFP4 entry point runs on, with stand-ins for the library's contexts: no GPU."""
import gc
import itertools
import threading
import time

import pytest

from oxidized_gpt_oss_b200 import abi, mxfp4


class Lib:
    @staticmethod
    def oxg_ctx_set_stream(handle, stream):
        handle.append(stream)
        return abi.OXG_OK


class Context:
    """Remembers its device, the streams that it was put on and whether it was ended."""
    made, ended, numbers = [], [], itertools.count()

    def __init__(self, device=0):
        self.device, self.lib, self.handle, self.number = device, Lib, [], next(self.numbers)
        time.sleep(0.002)  # others get their turn in the middle
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
    Context.made, Context.ended, Context.numbers = [], [], itertools.count()
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


@pytest.mark.parametrize("first", ["operator", "default", "default in a thread"])
def test_the_main_threads_context_is_the_default_one_in_any_order(first):
    """An error recorded by an operator's call is where device_context(...).sync() and context().sync() look for it, also
    after dequantize_mxfp4, swiglu or a MoE layer has asked for the default context for the first time."""
    if first == "default":
        mxfp4.context()
    elif first == "default in a thread":
        in_thread(mxfp4.context)
    of_call = mxfp4.device_context(On(0), None)
    assert mxfp4.context() is of_call
    assert mxfp4.device_context(On(0), None) is of_call
    other = mxfp4.device_context(On(1), None)
    assert other is not of_call and other.device == 1 and mxfp4.context() is of_call
    assert Context.made == [0, 1]


def test_the_default_context_is_made_once():
    """However many threads ask for it at the same time."""
    gate = threading.Barrier(8)
    got = []

    def work():
        gate.wait()
        got.append(mxfp4.context())

    ts = [threading.Thread(target=work) for _ in range(8)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert all(c is got[0] for c in got) and mxfp4.device_context(On(0), None) is got[0]
