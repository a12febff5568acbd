"""MXFP4 operators back to back through the C interface, in buffers that each step overwrites: a kernel may start while the
one before it still runs, and must read what that one wrote, not what stood there before."""
import pytest

from oxidized_gpt_oss_b200 import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n", [(1, 4096, 640), (40, 1024, 384), (300, 512, 2048), (1000, 2880, 1280)])
def test_steps_that_overwrite_the_buffers_of_the_step_before(cuda_ctx, m, k, n):
    import torch
    lib, h = cuda_ctx.lib, cuda_ctx.handle
    cols = n // 2

    def buffer(*shape, dtype=torch.uint8):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    def tiled(rows, width):
        return buffer((width + 127) // 128, rows, 4)

    def call(fn, *args):
        abi.check(getattr(lib, fn)(h, *[a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]), h)

    steps = 24
    gen = torch.Generator(device="cuda").manual_seed(m)
    xs = torch.randn(steps, m, k, generator=gen, device="cuda") * torch.exp2(torch.arange(steps, device="cuda") % 7 - 3)[:, None, None]
    fs = torch.exp2(torch.randint(-4, 5, (steps, m), generator=gen, device="cuda").float())
    weights = torch.randn(2, n, k, generator=gen, device="cuda"), torch.randn(2, 256, cols, generator=gen, device="cuda")
    x, f = buffer(m, k, dtype=torch.float32), buffer(m, dtype=torch.float32)
    wb, rows_, ws = buffer(n, k // 2), buffer(n, k // 32), tiled(n, k)
    vb, vs = buffer(256, cols // 2), tiled(256, cols)
    a, s = buffer(m, k // 2), tiled(m, k)
    y = buffer(m, n, dtype=torch.float32)
    b, t = buffer(m, cols // 2), tiled(m, cols)

    def run(wait):
        outs = []
        for i in range(steps):
            x.copy_(xs[i])
            f.copy_(fs[i])
            out = buffer(m, 256, dtype=torch.float32)
            torch.cuda.synchronize()
            for fn, *args in (("oxg_quantize_mxfp4", weights[0][i % 2], 0, n, k, k, None, 0, 0, wb, rows_),
                              ("oxg_mxfp4_tile_scales", rows_, 1, n, k, ws),
                              ("oxg_quantize_mxfp4", weights[1][i % 2], 0, 256, cols, cols, None, 0, 1, vb, vs),
                              ("oxg_quantize_mxfp4", x, 0, m, k, k, f, 0, 1, a, s),
                              ("oxg_mxfp4_matmul", a, s, m, wb, ws, n, k, None, y, 0, n),
                              ("oxg_swiglu_quantize_mxfp4", y, 0, m, cols, n, 1.702, 7.0, 0, 1, b, t),
                              ("oxg_mxfp4_matmul", b, t, m, vb, vs, 256, cols, None, out, 0, 256),
                              # the next round's, over the same buffers, while the product above may still run
                              ("oxg_quantize_mxfp4", xs[(i + 1) % steps], 0, m, k, k, None, 1, 1, a, s),
                              ("oxg_mxfp4_matmul", a, s, m, wb, ws, n, k, None, y, 0, n)):
                call(fn, *args)
                if wait:
                    torch.cuda.synchronize()
            outs += [out, y.clone()]
        torch.cuda.synchronize()
        return outs

    cuda_ctx.set_stream(torch.cuda.current_stream())
    want = run(True)
    for _ in range(4):
        assert all(torch.equal(p, q) for p, q in zip(run(False), want))
    cuda_ctx.sync()
