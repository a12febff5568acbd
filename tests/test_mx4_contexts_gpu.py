"""What the contexts behind the MXFP4 entry points owe their callers on a GPU: captures, threads that end, errors."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(program):
    r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


FIRST_CALLS_IN_A_CAPTURE = """
import torch
from oxidized_gpt_oss_b200 import ffn, mxfp4
torch.cuda.set_device(0)
blocks = torch.randint(0, 256, (8, 64), dtype=torch.uint8, device="cuda")
scales = torch.randint(120, 130, (8, 4), dtype=torch.uint8, device="cuda")
gate, up = torch.randn(1000, device="cuda"), torch.randn(1000, device="cuda")
x, w = torch.randn(70, 512, device="cuda"), torch.randn(300, 512, device="cuda")
def work():
    q = [mxfp4.quantize_mxfp4(t, tiled=True) for t in (x, w)]
    return [mxfp4.dequantize_mxfp4(blocks, scales, 8, 128), ffn.swiglu(gate, up), mxfp4.mxfp4_matmul(*q[0], *q[1])]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):  # no context exists yet
    out = work()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, work()))
mxfp4.context().sync()
print("done")
"""


def test_a_process_whose_first_calls_are_captured():
    """Making a context allocates nothing, so the capture that makes it stands."""
    _run(FIRST_CALLS_IN_A_CAPTURE)


def test_a_graph_that_outlives_its_context():
    """A product captured with a context that is gone when the graph is replayed: what it finds wrong goes to nobody's
    memory and to nobody's sync, and its rows are as they should be."""
    import torch
    from oxidized_gpt_oss_b200 import abi, mxfp4
    a, w = (mxfp4.quantize_mxfp4(torch.randn(n, 96, device="cuda"), tiled=True) for n in (40, 33))
    w = tuple(t[None] for t in w)
    counts = torch.tensor([40], dtype=torch.int32, device="cuda")
    out = torch.empty(40, 33, device="cuda")
    gone, other = abi.Context(0), abi.Context(0)
    mxfp4.mxfp4_grouped_matmul(*a, counts, *w, out=out, ctx=gone)
    want = mxfp4.mxfp4_grouped_matmul(*a, counts, *w, out_dtype=torch.float32, ctx=other)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mxfp4.mxfp4_grouped_matmul(*a, counts, *w, out=out, ctx=gone)
    gone.close()
    later = abi.Context(0)  # would be given whatever memory a context gives back
    mxfp4.mxfp4_grouped_matmul(*a, counts, *w, ctx=later)
    around = [torch.zeros(1 << 10, dtype=torch.int32, device="cuda") for _ in range(64)]
    counts.fill_(41)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert not any(t.any() for t in around)
    for ctx in (other, later, mxfp4.context()):
        ctx.sync()
    for ctx in (other, later):
        ctx.close()


def test_every_context_has_errors_of_its_own():
    import torch
    from oxidized_gpt_oss_b200 import abi, mxfp4
    a, w = (mxfp4.quantize_mxfp4(torch.randn(n, 96, device="cuda"), tiled=True) for n in (40, 33))
    w = tuple(t[None] for t in w)
    fits, beyond = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (40, 41))
    for _ in range(3):  # a context that ends unread leaves nothing to the next
        ctxs = [abi.Context(0) for _ in range(20)]
        for i, ctx in enumerate(ctxs):
            mxfp4.mxfp4_grouped_matmul(*a, beyond if i % 3 == 0 else fits, *w, ctx=ctx)
        for i, ctx in enumerate(ctxs[:-3]):
            if i % 3 == 0:
                with pytest.raises(abi.OxgError, match="count"):
                    ctx.sync()
            ctx.sync()
        for ctx in ctxs:
            ctx.close()


THREADS_DURING_A_CAPTURE = """
import gc
import threading
import torch
from oxidized_gpt_oss_b200 import mxfp4
torch.cuda.set_device(0)
x = torch.randn(70, 512, device="cuda")
want = mxfp4.quantize_mxfp4(x, tiled=True)
streams = [torch.cuda.Stream() for _ in range(2)]
held = []
for st in streams:
    with torch.cuda.stream(st):
        held.append(torch.empty(1, device="cuda"))  # the allocator has room beside it for the stream's next tensors
got = []
def work(st):
    with torch.cuda.stream(st):
        got.append(mxfp4.quantize_mxfp4(x, tiled=True))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    mine = mxfp4.quantize_mxfp4(x, tiled=True)
    threads = [threading.Thread(target=work, args=(st,)) for st in streams]
    for t in threads: t.start()
    for t in threads: t.join()
    del threads, t
    gc.collect()
g.replay()
torch.cuda.synchronize()
assert len(got) == 2
for q in (mine, *got):
    assert torch.equal(q[0], want[0]) and torch.equal(q[1], want[1])
print("done")
"""


def test_threads_that_begin_and_end_while_another_captures():
    """A capture in the default mode forbids every thread what may synchronise: a thread's first call and its end do not."""
    _run(THREADS_DURING_A_CAPTURE)


def test_a_graph_that_outlives_the_thread_that_captured_it():
    """What it finds wrong is reported by the context that the thread had, whose word is nobody else's."""
    import gc
    import threading
    import torch
    from oxidized_gpt_oss_b200 import abi, mxfp4
    a, w = (mxfp4.quantize_mxfp4(torch.randn(n, 96, device="cuda"), tiled=True) for n in (40, 33))
    w = tuple(t[None] for t in w)
    counts = torch.tensor([40], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    held = {}

    def capture():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            mxfp4.mxfp4_grouped_matmul(*a, counts, *w)
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                mxfp4.mxfp4_grouped_matmul(*a, counts, *w)
        held["graph"], held["ctx"] = g, mxfp4.device_context(counts, None)

    t = threading.Thread(target=capture)
    t.start()
    t.join()
    del t
    gc.collect()
    counts.fill_(41)
    held["graph"].replay()
    torch.cuda.synchronize()
    mxfp4.device_context(counts, None).sync()
    with pytest.raises(abi.OxgError, match="count"):
        held["ctx"].sync()
    held["ctx"].sync()


ERROR_BEFORE_THE_DEFAULT_CONTEXT = """
import torch
from oxidized_gpt_oss_b200 import abi, mxfp4
torch.cuda.set_device(0)
a, w = (mxfp4.quantize_mxfp4(torch.randn(n, 96, device="cuda"), tiled=True) for n in (40, 33))
counts = torch.tensor([41], dtype=torch.int32, device="cuda")
mxfp4.mxfp4_grouped_matmul(*a, counts, *(t[None] for t in w))
mxfp4.dequantize_mxfp4(a[0], torch.zeros(40, 3, dtype=torch.uint8, device="cuda"), 40, 96)
try:
    mxfp4.device_context(counts, None).sync()
except abi.OxgError as e:
    assert e.status == abi.OXG_ERR_SHAPE
    print("done")
"""


def test_an_error_is_not_lost_when_the_default_context_comes_after_it():
    _run(ERROR_BEFORE_THE_DEFAULT_CONTEXT)


def test_threads_that_read_back_while_the_main_thread_multiplies():
    """Two threads quantise and dequantise on streams of their own while the main thread's products run on a third."""
    import threading
    import torch
    from oxidized_gpt_oss_b200 import ffn, mxfp4
    x, w = torch.randn(700, 2048, device="cuda"), mxfp4.quantize_mxfp4(torch.randn(900, 2048, device="cuda"), tiled=True)
    want = mxfp4.mxfp4_matmul(*mxfp4.quantize_mxfp4(x, tiled=True), *w)
    mine = [torch.randn(300, 4096, device="cuda") for _ in range(2)]
    back = [mxfp4.dequantize_mxfp4(*mxfp4.quantize_mxfp4(m), 300, 4096) for m in mine]
    act = [ffn.swiglu(m[:, ::2], m[:, 1::2]) for m in mine]
    torch.cuda.synchronize()
    bad, gate = [], threading.Barrier(3)

    def work(m, b, y):
        with torch.cuda.stream(torch.cuda.Stream()) as _:
            st = torch.cuda.current_stream()
            gate.wait()
            for _ in range(150):
                got, h = mxfp4.dequantize_mxfp4(*mxfp4.quantize_mxfp4(m), 300, 4096), ffn.swiglu(m[:, ::2], m[:, 1::2])
                st.synchronize()
                if not (torch.equal(got, b) and torch.equal(h, y)):
                    bad.append("thread")

    threads = [threading.Thread(target=work, args=a) for a in zip(mine, back, act)]
    for t in threads:
        t.start()
    st = torch.cuda.Stream()
    gate.wait()
    with torch.cuda.stream(st):
        for _ in range(150):
            got = mxfp4.mxfp4_matmul(*mxfp4.quantize_mxfp4(x, tiled=True), *w)
            st.synchronize()
            if not torch.equal(got, want):
                bad.append("main")
    for t in threads:
        t.join()
    assert not bad


def test_dequantize_into_pinned_memory():
    import torch
    from oxidized_gpt_oss_b200 import mxfp4
    b, s = mxfp4.quantize_mxfp4(torch.randn(8, 64, device="cuda"))
    out = torch.empty(8 * 64, dtype=torch.int16, pin_memory=True)
    mxfp4.dequantize_mxfp4(b, s, 8, 64, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out.cuda(), mxfp4.dequantize_mxfp4(b, s, 8, 64))
    with pytest.raises(ValueError, match="pinned"):
        mxfp4.dequantize_mxfp4(b, s, 8, 64, out=torch.empty(8 * 64, dtype=torch.int16))
