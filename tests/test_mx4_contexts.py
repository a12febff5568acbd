"""Which context an MXFP4 entry point runs on, with stand-ins for the library's contexts: no GPU."""
import gc
import itertools
import threading
import time

import pytest
import torch

from oxidized_gpt_oss_b200 import abi, ffn, mxfp4


class Lib:
    @staticmethod
    def oxg_ctx_set_stream(handle, stream):
        handle.append(stream)
        return abi.OXG_OK

    launched = []

    @classmethod
    def oxg_dequant_mxfp4(cls, handle, *args):
        cls.launched.append(handle)
        return abi.OXG_OK

    @classmethod
    def oxg_swiglu(cls, handle, *args):
        cls.launched.append(handle)
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


class On0(torch.Tensor):
    """Host memory that says it is on a GPU."""
    index, is_cuda = 0, True

    def get_device(self):
        return self.index


class On1(On0):
    index = 1


def tensor(of, *shape, dtype=torch.uint8):
    return torch.zeros(*shape, dtype=dtype).as_subclass(of)


def read_back(of=On0, scales_of=None, **kw):
    return mxfp4.dequantize_mxfp4(tensor(of, 2, 32), tensor(scales_of or of, 2, 2), 2, 64, **kw)


def activate(of=On0, up_of=None, **kw):
    return ffn.swiglu(*(tensor(o, 64, dtype=torch.float32) for o in (of, up_of or of)), **kw)


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    Lib.launched = []
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


@pytest.mark.parametrize("call", [read_back, activate])
def test_another_threads_call_leaves_the_main_threads_context_alone(call):
    """The context that the main thread has just put on its stream is not moved to another thread's before it launches."""
    main = mxfp4.device_context(On(0), None)
    assert main is mxfp4.context()
    streams = list(main.handle)
    in_thread(call)
    assert main.handle == streams
    assert len(Lib.launched) == 1 and Lib.launched[0] is not main.handle
    call()
    assert Lib.launched[1] is main.handle


@pytest.mark.parametrize("call", [read_back, activate])
def test_calls_run_on_their_operands_device(call):
    """On the operands' device whichever is current, and on no other: a context of another, or operands on two, are
    refused before anything is launched."""
    mxfp4.context()
    call(On1)
    assert Lib.launched == [mxfp4.device_context(On(1), None).handle]
    del Lib.launched[:]
    with pytest.raises(ValueError, match="the context is on cuda:0"):
        call(On1, ctx=mxfp4.context())
    for operands in ((On0, On1), (On1, On0)):
        with pytest.raises(ValueError, match="one device"):
            call(*operands)
    assert not Lib.launched
    with pytest.raises(ValueError, match="out"):
        read_back(On0, out=tensor(On1, 128, dtype=torch.int16))
    with pytest.raises(ValueError, match="out"):
        read_back(On0, out=torch.zeros(128, dtype=torch.int16))
    assert not Lib.launched
