"""MXFP4 quantisation and products on the GPU against 64-bit references.

Quantisation has one right answer, so codes and scale bytes are compared as they are.

Products: with S = sum over k of |a b| in exact arithmetic, one MMA adds 64 of the (exact) products to the f32
accumulator, which costs at most one unit in the last place of a running sum that never exceeds S: 2^-23 S for each
of the ceil(k / 64) MMAs. The bias adds half a unit of the result; a bf16 result is rounded by at most half a step,
2^-8 of its magnitude.
"""
import numpy as np
import pytest

import mx4_reference as ref
from oxidized_gpt_oss_b200 import abi

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")


def _torch():
    import torch
    from oxidized_gpt_oss_b200 import ffn, mxfp4
    return torch, mxfp4, ffn


def _same(blocks, scales, codes, bytes_, cols, tiled=False):
    assert np.array_equal(blocks.cpu().numpy().reshape(-1, cols // 2), ref.pack(codes))
    want = ref.tile(bytes_, cols) if tiled else bytes_
    assert np.array_equal(scales.cpu().numpy().reshape(want.shape), want)


def _rows(rng, rows, cols):
    """Rows whose blocks lie far apart, with ties, powers of two, zeros, subnormals and both signs of zero among them."""
    x = rng.standard_normal((rows, cols)) * np.exp(3 * rng.standard_normal((rows, cols // 32)).repeat(32, 1))
    x = x.astype(np.float32)
    flat = x.reshape(-1, 32)
    flat[0] = 0
    flat[0, 1] = -0.0
    ties = np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 7], np.float32)
    flat[-1, :16] = ties / 8
    flat[-1, 16:] = np.nextafter(ties / 8, np.float32(np.inf))
    if len(flat) > 2:
        flat[1] = 2.0 ** rng.integers(-4, 3, 32)
    if len(flat) > 4:
        flat[2] = rng.standard_normal(32) * 1e-39
        flat[3] = 1.5
    return x


@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("rule", ["floor", "noclip"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (7, 2880), (129, 160), (1000, 64)])
def test_quantize_is_the_nearest_code(cuda_ctx, rows, cols, dtype, rule, tiled):
    torch, mxfp4, _ = _torch()
    x = torch.from_numpy(_rows(np.random.default_rng(rows * cols), rows, cols)).cuda().to(getattr(torch, dtype))
    codes, scales = ref.quantize(x.double().cpu().numpy(), rule)
    _same(*mxfp4.quantize_mxfp4(x, scale_rule=rule, tiled=tiled), codes, scales, cols, tiled)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,pitch", [(8, 136), (1, 128), (0, 131), (8, 133)])
def test_quantize_rows_of_a_wider_matrix(cuda_ctx, dtype, offset, pitch):
    torch, mxfp4, _ = _torch()
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((11, pitch)).astype(np.float32)).cuda()
    x = x.to(getattr(torch, dtype))[:, offset: offset + 96]
    f = torch.exp2(torch.arange(-5, 6, device="cuda").float())
    codes, scales = ref.quantize(x.double().cpu().numpy() * f.double().cpu().numpy()[:, None])
    for tiled in (False, True):
        _same(*mxfp4.quantize_mxfp4(x, row_scale=f, tiled=tiled), codes, scales, 96, tiled)


def test_quantize_row_scale_is_an_f32_product(cuda_ctx):
    torch, mxfp4, _ = _torch()
    x = torch.from_numpy(np.random.default_rng(2).standard_normal((64, 256)).astype(np.float32)).cuda()
    f = torch.rand(64, device="cuda") + 0.1
    codes, scales = ref.quantize((x * f[:, None]).double().cpu().numpy())
    _same(*mxfp4.quantize_mxfp4(x, row_scale=f), codes, scales, 256)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_extremes(cuda_ctx, dtype):
    """The type's largest and smallest values quantise; a block with an infinity or a NaN reads back as NaN, its
    neighbours as usual."""
    torch, mxfp4, _ = _torch()
    info = torch.finfo(getattr(torch, dtype))
    x = torch.ones(4, 128, device="cuda", dtype=getattr(torch, dtype))
    x[0, :32] = info.max
    x[0, 32:64] = info.tiny
    x[0, 64:96] = info.smallest_normal * info.eps
    x[1, 5] = float("inf")
    x[1, 70] = float("-inf")
    x[2, 127] = float("nan")
    x[3] = -info.max
    for rule in ("floor", "noclip"):
        codes, scales = ref.quantize(x.double().cpu().numpy(), rule)
        blocks, got = mxfp4.quantize_mxfp4(x, scale_rule=rule)
        _same(blocks, got, codes, scales, 128)
        assert (got.cpu().numpy() == 255).sum() == 3
        back = mxfp4.dequantize_mxfp4(blocks, got, 4, 128).view(torch.bfloat16).view(4, 4, 32)
        bad = ~torch.isfinite(x.view(4, 4, 32)).all(-1)
        assert torch.isnan(back[bad]).all() and torch.isfinite(back[~bad]).all()


def test_quantize_shapes_and_refusals(cuda_ctx):
    torch, mxfp4, _ = _torch()
    x = torch.randn(2, 3, 64, device="cuda")
    b, s = mxfp4.quantize_mxfp4(x)
    assert b.shape == (2, 3, 32) and s.shape == (2, 3, 2)
    b2, s2 = mxfp4.quantize_mxfp4(x.permute(1, 0, 2))  # rows without a common pitch
    assert torch.equal(b2, b.permute(1, 0, 2)) and torch.equal(s2, s.permute(1, 0, 2))
    b1, s1 = mxfp4.quantize_mxfp4(x[0, 0])
    assert torch.equal(b1, b[0, 0]) and torch.equal(s1, s[0, 0])
    b0, s0 = mxfp4.quantize_mxfp4(x[:, :0])
    assert b0.shape == (2, 0, 32) and s0.shape == (2, 0, 2)
    with pytest.raises(ValueError, match="cols must be divisible by 32, got 33"):
        mxfp4.quantize_mxfp4(torch.randn(2, 33, device="cuda"))
    with pytest.raises(ValueError, match="unknown scale rule"):
        mxfp4.quantize_mxfp4(x, scale_rule="up")
    with pytest.raises(ValueError, match="2 dimensions"):
        mxfp4.quantize_mxfp4(x, tiled=True)
    with pytest.raises(ValueError, match="row_scale"):
        mxfp4.quantize_mxfp4(x, row_scale=torch.ones(5, device="cuda"))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        mxfp4.quantize_mxfp4(x.double())


def test_quantize_c_refusals(cuda_ctx):
    torch, _, _ = _torch()
    lib, h = cuda_ctx.lib, cuda_ctx.handle
    x = torch.zeros(4096, device="cuda")
    b, s = torch.full((1024,), 7, dtype=torch.uint8, device="cuda"), torch.full((256,), 7, dtype=torch.uint8, device="cuda")
    px, pb, ps = x.data_ptr(), b.data_ptr(), s.data_ptr()
    for status, args in ((abi.OXG_ERR_INVALID_ARG, (px, 9, 2, 64, 64, None, 0, 0, pb, ps)),
                         (abi.OXG_ERR_INVALID_ARG, (px, 0, 2, 64, 64, None, 2, 0, pb, ps)),
                         (abi.OXG_ERR_INVALID_ARG, (px, 0, 2, 64, 64, None, 0, 2, pb, ps)),
                         (abi.OXG_ERR_SHAPE, (px, 0, 2, 48, 64, None, 0, 0, pb, ps)),
                         (abi.OXG_ERR_SHAPE, (px, 0, 2, 64, 63, None, 0, 0, pb, ps)),
                         (abi.OXG_ERR_SHAPE, (px, 0, 2 ** 60, 64, 64, None, 0, 0, pb, ps)),
                         (abi.OXG_ERR_INVALID_ARG, (None, 0, 2, 64, 64, None, 0, 0, pb, ps)),
                         (abi.OXG_ERR_INVALID_ARG, (px, 0, 2, 64, 64, None, 0, 0, None, ps)),
                         (abi.OXG_ERR_INVALID_ARG, (px, 0, 2, 64, 64, None, 0, 0, pb, None)),
                         (abi.OXG_ERR_INVALID_ARG, (px + 2, 0, 2, 64, 64, None, 0, 0, pb, ps)),
                         (abi.OXG_ERR_INVALID_ARG, (px, 0, 2, 64, 64, None, 0, 0, pb + 2, ps)),
                         (abi.OXG_OK, (None, 0, 0, 64, 64, None, 0, 0, None, None))):
        assert lib.oxg_quantize_mxfp4(h, *args) == status, args
    assert lib.oxg_swiglu_quantize_mxfp4(h, px, 0, 2, 64, 127, 1.702, 7.0, 0, 0, pb, ps) == abi.OXG_ERR_SHAPE
    assert lib.oxg_swiglu_quantize_mxfp4(h, px, 0, 2, 64, 128, 1.702, 0.0, 0, 0, pb, ps) == abi.OXG_ERR_INVALID_ARG
    assert lib.oxg_swiglu_quantize_mxfp4(h, px, 0, 2, 64, 128, 1.702, float("nan"), 0, 0, pb, ps) == abi.OXG_ERR_INVALID_ARG
    assert lib.oxg_mxfp4_tile_scales(h, ps, 1, 2, 48, pb) == abi.OXG_ERR_SHAPE
    assert lib.oxg_mxfp4_tile_scales(h, ps, 1, 2, 64, None) == abi.OXG_ERR_INVALID_ARG
    cuda_ctx.sync()
    assert (b == 7).all() and (s == 7).all()


@pytest.mark.parametrize("rule", ["floor", "noclip"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (64, 2880), (700, 416)])
def test_swiglu_quantize_is_the_exact_values_code(cuda_ctx, rows, cols, dtype, rule):
    torch, _, ffn = _torch()
    x = torch.from_numpy(np.random.default_rng(rows).standard_normal((rows, 2 * cols)).astype(np.float32) * 3).cuda()
    x = x.to(getattr(torch, dtype))
    codes, scales = ref.quantize(ref.swiglu(x.double().cpu().numpy(), ffn.ALPHA, ffn.LIMIT), rule)
    for tiled in (False, True):
        _same(*ffn.swiglu_quantize_mxfp4(x, scale_rule=rule, tiled=tiled), codes, scales, cols, tiled)


def test_swiglu_quantize_at_its_edges(cuda_ctx):
    """Gates so low that the f32 sigmoid is subnormal or zero, products below f32's normal range, up = -1, values at the
    clamps, infinities and NaN; a row pitch off the 16-byte grid."""
    torch, _, ffn = _torch()
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 128)).astype(np.float32)
    x[0, 0::2] = rng.uniform(-63, -45, 64)
    x[1, 0::2] = rng.uniform(-600, -55, 64)
    x[2] *= 1e-30
    x[3, 0::2] *= 1e-38
    x[3, 1::2] = -1 + rng.standard_normal(64) * 1e-6
    x[4, 1::2] = -1
    x[5] = 7.0
    x[6, 0::2], x[6, 1::2] = 1e30, -1e30
    x[7, 0], x[7, 64] = np.inf, -np.inf  # the first is clamped; the second gives -inf * 0
    x[8, 1], x[8, 65] = np.inf, -np.inf  # both clamped
    x[9, 2], x[9, 67] = np.nan, np.nan
    x[10] = 0
    x[11, 0::2] = -1e30
    want = ref.swiglu(x, ffn.ALPHA, ffn.LIMIT)
    wide = torch.zeros(12, 131, device="cuda")
    wide[:, :128] = torch.from_numpy(x)
    for rule in ("floor", "noclip"):
        codes, scales = ref.quantize(want, rule)
        for gate_up in (torch.from_numpy(x).cuda(), wide[:, :128]):
            _same(*ffn.swiglu_quantize_mxfp4(gate_up, scale_rule=rule), codes, scales, 64)
    assert (scales == 255).sum() == 3


def test_swiglu_quantize_with_other_constants(cuda_ctx):
    torch, _, ffn = _torch()
    x = torch.randn(33, 192, device="cuda") * 20
    for alpha, limit in ((1.0, float("inf")), (1.702, 0.5), (0.25, 128.0)):
        codes, scales = ref.quantize(ref.swiglu(x.cpu().numpy(), alpha, limit))
        _same(*ffn.swiglu_quantize_mxfp4(x, alpha, limit), codes, scales, 96)


@pytest.mark.parametrize("shape", [(1, 1), (5, 3), (3, 7, 4), (2, 3, 130, 90), (33, 5)])
def test_tile_scales(cuda_ctx, shape):
    torch, mxfp4, _ = _torch()
    s = np.random.default_rng(3).integers(0, 255, shape, dtype=np.uint8)
    assert np.array_equal(mxfp4.tile_scales(torch.from_numpy(s).cuda()).cpu().numpy(), ref.tile(s, 32 * shape[-1]))


# ---- products ---------------------------------------------------------------------------------------------------------
def _operand(rng, *shape, around=127, spread=3):
    """Random codes and scale rows [..., rows, k]."""
    *lead, k = shape
    blocks = rng.integers(0, 256, (*lead, k // 2), dtype=np.uint8)
    return blocks, rng.integers(around - spread, around + spread + 1, (*lead, k // 32), dtype=np.uint8)


def _cuda(*arrays):
    import torch
    return [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def _check(got, av, bv, bias, dtype):
    """got against av @ bv.T + bias by the module's bound; av, bv float64."""
    y, s = av @ bv.T, np.abs(av) @ np.abs(bv).T
    bound = s * (-(-av.shape[1] // 64)) * 2.0 ** -23
    if bias is not None:
        y = y + bias
        bound = bound + np.abs(y) * 2.0 ** -24
    if dtype == "bfloat16":
        bound = bound + (np.abs(y) + bound) * 2.0 ** -8
    got = got.double().cpu().numpy()
    assert got.shape == y.shape
    err = np.abs(got - y)
    assert np.all(err <= bound + 1e-300), (np.nanmax(err / np.maximum(bound, 1e-300)), np.argwhere(~(err <= bound))[:5])


def _bias(rng, *shape):
    import torch
    t = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16)
    return t.cuda(), t.double().numpy()


SHAPES = [(1, 1, 32), (1, 5, 32), (2, 128, 64), (16, 129, 96), (17, 64, 128), (31, 300, 160), (33, 127, 256), (64, 1000, 288),
          (128, 130, 512), (129, 256, 544), (224, 33, 1024), (225, 77, 1056), (300, 257, 2880), (449, 128, 64), (1000, 640, 2880),
          (8, 5120, 2880), (1, 2880, 4096), (50, 96, 8192), (700, 1, 320), (1037, 2881, 224),
          (40, 38500, 544), (3, 19300, 2400), (100, 60, 8192), (2000, 1300, 1184)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(cuda_ctx, m, n, k, dtype):
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, n, k, around=122)
    bias, bias64 = _bias(rng, n) if (m + n) % 2 else (None, None)
    a, at, b, bt = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k))
    got = mxfp4.mxfp4_matmul(a, at, b, bt, bias=bias, out_dtype=getattr(torch, dtype))
    cuda_ctx.sync()
    _check(got, ref.values(ab, asc), ref.values(bb, bsc), bias64, dtype)


@pytest.mark.parametrize("m,n,k", [(3, 70, 96), (130, 200, 2880), (260, 300, 1024)])
def test_matmul_sums_that_f32_holds_are_exact(cuda_ctx, m, n, k):
    """With every scale 1 the sums are multiples of 1/4 below 2^22, so any order of f32 additions gives them exactly."""
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(k)
    (ab, asc), (bb, bsc) = _operand(rng, m, k, spread=0), _operand(rng, n, k, spread=0)
    a, at, b, bt = _cuda(ab, asc, bb, bsc)  # scale rows: laid out by the call
    got = mxfp4.mxfp4_matmul(a, at, b, bt, out_dtype=torch.float32)
    assert np.array_equal(got.cpu().numpy(), (ref.values(ab, asc) @ ref.values(bb, bsc).T).astype(np.float32))


def test_matmul_scales_far_from_one_and_nan(cuda_ctx):
    """Scales over most of E8M0's range (a's and b's far ends cancel); byte 255 makes its row or column NaN and no other;
    byte 0 is 2^-127."""
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(9)
    m, n, k = 40, 150, 320
    (ab, asc), (bb, bsc) = _operand(rng, m, k, spread=2), _operand(rng, n, k, spread=2)
    rows, cols = rng.integers(-110, 111, m), rng.integers(-8, 9, n)
    asc, bsc = (asc + rows[:, None]).astype(np.uint8), (bsc + cols[:, None]).astype(np.uint8)
    asc[7, 3] = 0
    av, bv = ref.values(ab, asc), ref.values(bb, bsc)
    a, at, b, bt = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k))
    _check(mxfp4.mxfp4_matmul(a, at, b, bt, out_dtype=torch.float32), av, bv, None, "float32")
    asc[5, 9], bsc[149, 0], bsc[3, 4] = 255, 255, 255
    ab[5, 9 * 16: 10 * 16] = 0  # zero codes under a NaN scale are NaN too
    a, at, b, bt = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k))
    got = mxfp4.mxfp4_matmul(a, at, b, bt, out_dtype=torch.float32).cpu().numpy()
    nan = np.zeros((m, n), bool)
    nan[5], nan[:, 149], nan[:, 3] = True, True, True
    assert np.array_equal(np.isnan(got), nan)


@pytest.mark.parametrize("spread", [6, 12, 30])
@pytest.mark.parametrize("m,n,k", [(33, 130, 64), (20, 64, 2880), (300, 256, 1056)])
def test_matmul_scales_spread_in_a_row(cuda_ctx, m, n, k, spread):
    """Blocks of one row up to 2^120 apart: sums that f32 does not hold exactly, within the same bound."""
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(k + spread)
    (ab, asc), (bb, bsc) = _operand(rng, m, k, spread=spread), _operand(rng, n, k, spread=spread)
    a, at, b, bt = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k))
    _check(mxfp4.mxfp4_matmul(a, at, b, bt, out_dtype=torch.float32), ref.values(ab, asc), ref.values(bb, bsc), None, "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("pitch,offset", [(96, 0), (97, 1), (104, 3)])
def test_matmul_writes_its_own_elements_only(cuda_ctx, dtype, pitch, offset):
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(4)
    m, n, k = 35, 91, 160
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, n, k)
    a, at, b, bt = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k))
    whole = torch.full((m + 2, pitch), 77.0, device="cuda", dtype=getattr(torch, dtype))
    out = whole[1: m + 1, offset: offset + n]
    assert mxfp4.mxfp4_matmul(a, at, b, bt, out=out) is out
    _check(out, ref.values(ab, asc), ref.values(bb, bsc), None, dtype)
    whole[1: m + 1, offset: offset + n] = 77.0
    assert (whole == 77.0).all()


COUNTS = [(5, [5]), (40, [0, 40]), (40, [40, 0, 0]), (300, [0, 1, 225, 0, 16, 0, 31]), (700, [224, 224, 1, 251]), (64, [1] * 64),
          (33, [0] * 50 + [2] * 10 + [0] * 40), (513, [100, 0, 400]), (10, [0, 0])]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,counts", COUNTS)
@pytest.mark.parametrize("n,k", [(130, 96), (64, 576)])
def test_grouped_matmul(cuda_ctx, m, counts, n, k, dtype):
    """Ragged and empty groups; rows past the last group keep what they held."""
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(m + n)
    G = len(counts)
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, G, n, k, around=122)
    bias, bias64 = _bias(rng, G, n) if G % 2 else (None, None)
    a, at, b, bt, c = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k), np.array(counts, np.int32))
    out = torch.full((m, n), 55.0, device="cuda", dtype=getattr(torch, dtype))
    mxfp4.mxfp4_grouped_matmul(a, at, c, b, bt, bias=bias, out=out)
    cuda_ctx.sync()
    av, bv, r = ref.values(ab, asc), ref.values(bb, bsc), 0
    for g, cnt in enumerate(counts):
        _check(out[r: r + cnt], av[r: r + cnt], bv[g], None if bias is None else bias64[g], dtype)
        r += cnt
    assert (out[r:] == 55.0).all()


def test_grouped_matmul_at_gpt_oss_widths(cuda_ctx):
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(11)
    counts = rng.multinomial(600, np.full(8, 1 / 8))
    n, k = 5760, 2880
    (ab, asc), (bb, bsc) = _operand(rng, 600, k), _operand(rng, 8, n, k, around=122)
    a, at, b, bt, c = _cuda(ab, asc, bb, bsc, counts.astype(np.int32))
    got = mxfp4.mxfp4_grouped_matmul(a, at, c, b, bt)
    av, r = ref.values(ab, asc), 0
    for g, cnt in enumerate(counts):
        _check(got[r: r + cnt], av[r: r + cnt], ref.values(bb[g], bsc[g]), None, "bfloat16")
        r += cnt


def test_grouped_matmul_of_few_rows_and_many_tiles(cuda_ctx):
    """More tiles than SMs with a handful of rows each: a CTA goes through several tiles of different groups."""
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(14)
    counts = np.array([3, 0, 17, 1, 65, 0, 0, 2, 8, 30])
    m, n, k = int(counts.sum()) + 5, 5764, 2400
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, len(counts), n, k, around=122)
    bias, bias64 = _bias(rng, len(counts), n)
    a, at, b, bt, c = _cuda(ab, ref.tile(asc, k), bb, ref.tile(bsc, k), counts.astype(np.int32))
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m, n), 55.0, device="cuda", dtype=dtype)
        mxfp4.mxfp4_grouped_matmul(a, at, c, b, bt, bias=bias, out=out)
        cuda_ctx.sync()
        av, r = ref.values(ab, asc), 0
        for g, cnt in enumerate(counts):
            _check(out[r: r + cnt], av[r: r + cnt], ref.values(bb[g], bsc[g]), bias64[g], str(dtype)[6:])
            r += cnt
        assert (out[r:] == 55.0).all()


@pytest.mark.parametrize("counts", [[20, 30], [-1, 20], [2 ** 31 - 1, 2 ** 31 - 1], [41, 0]])
def test_grouped_matmul_reports_counts_that_do_not_fit(cuda_ctx, counts):
    """Nothing is read or written past the rows there are, the next sync says so, and the one after is clean."""
    torch, mxfp4, _ = _torch()
    rng = np.random.default_rng(12)
    (ab, asc), (bb, bsc) = _operand(rng, 40, 64), _operand(rng, 2, 33, 64)
    a, at, b, bt, c = _cuda(ab, ref.tile(asc, 64), bb, ref.tile(bsc, 64), np.array(counts, np.int32))
    whole = torch.full((42, 33), 55.0, device="cuda")
    ctx = abi.Context(0)
    mxfp4.mxfp4_grouped_matmul(a, at, c, b, bt, out=whole[1:41], ctx=ctx)
    with pytest.raises(abi.OxgError, match="count") as e:
        ctx.sync()
    assert e.value.status == abi.OXG_ERR_SHAPE
    ctx.sync()
    assert (whole[0] == 55.0).all() and (whole[41] == 55.0).all()
    av, bv = ref.values(ab, asc), ref.values(bb, bsc)
    first = min(max(counts[0], 0), 40)
    last = min(first + max(counts[1], 0), 40)
    _check(whole[1: first + 1], av[:first], bv[0], None, "float32")
    _check(whole[first + 1: last + 1], av[first:last], bv[1], None, "float32")
    assert (whole[last + 1:] == 55.0).all()
    ctx.close()


def test_product_refusals(cuda_ctx):
    torch, mxfp4, _ = _torch()
    a, s = torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), torch.full((1, 4, 4), 127, dtype=torch.uint8, device="cuda")
    for match, call in (("positive multiple of 32", lambda: mxfp4.mxfp4_matmul(a[:, :8].contiguous(), s, a, s)),
                        ("a's scales must be", lambda: mxfp4.mxfp4_matmul(a, s[:, :3], a, s)),
                        ("elements, b of", lambda: mxfp4.mxfp4_matmul(a, s, a[:, :16].contiguous(), s)),
                        ("out_dtype", lambda: mxfp4.mxfp4_matmul(a, s, a, s, out_dtype=torch.float16)),
                        ("out must be", lambda: mxfp4.mxfp4_matmul(a, s, a, s, out=torch.empty(4, 5, device="cuda"))),
                        ("out must be", lambda: mxfp4.mxfp4_matmul(a, s, a, s, out=torch.empty(4, 4, device="cuda").t())),
                        ("bias", lambda: mxfp4.mxfp4_matmul(a, s, a, s, bias=torch.zeros(4, device="cuda"))),
                        ("uint8", lambda: mxfp4.mxfp4_matmul(a.float(), s, a, s)),
                        ("3 dimensions", lambda: mxfp4.mxfp4_grouped_matmul(a, s, torch.zeros(1, dtype=torch.int32, device="cuda"), a, s)),
                        ("counts", lambda: mxfp4.mxfp4_grouped_matmul(a, s, torch.zeros(2, dtype=torch.int32, device="cuda"), a[None], s[None])),
                        ("counts", lambda: mxfp4.mxfp4_grouped_matmul(a, s, torch.zeros(1, device="cuda"), a[None], s[None]))):
        with pytest.raises(ValueError, match=match):
            call()
    lib, h, p = cuda_ctx.lib, cuda_ctx.handle, a.data_ptr()
    sp = s.data_ptr()
    o = torch.full((64,), 3.0, device="cuda")
    q = o.data_ptr()
    for status, args in ((abi.OXG_ERR_SHAPE, (p, sp, -1, p, sp, 4, 64, None, q, 0, 4)), (abi.OXG_ERR_SHAPE, (p, sp, 4, p, sp, 4, 48, None, q, 0, 4)),
                         (abi.OXG_ERR_SHAPE, (p, sp, 4, p, sp, 4, 0, None, q, 0, 4)), (abi.OXG_ERR_SHAPE, (p, sp, 4, p, sp, 4, 64, None, q, 0, 3)),
                         (abi.OXG_ERR_SHAPE, (p, sp, 2 ** 31 - 1, p, sp, 4, 64, None, q, 0, 4)),
                         (abi.OXG_ERR_SHAPE, (p, sp, 4, p, sp, 2 ** 31 - 256, 64, None, q, 0, 2 ** 31)),
                         (abi.OXG_ERR_INVALID_ARG, (p, sp, 4, p, sp, 4, 64, None, q, 2, 4)),
                         (abi.OXG_ERR_INVALID_ARG, (p + 8, sp, 2, p, sp, 4, 32, None, q, 0, 4)),
                         (abi.OXG_ERR_INVALID_ARG, (p, sp + 1, 2, p, sp, 4, 32, None, q, 0, 4)),
                         (abi.OXG_ERR_INVALID_ARG, (p, sp, 4, p, sp, 4, 64, None, q + 2, 0, 4)),
                         (abi.OXG_ERR_INVALID_ARG, (p, sp, 4, p, sp, 4, 64, None, None, 0, 4)),
                         (abi.OXG_OK, (p, sp, 0, p, sp, 4, 64, None, None, 0, 4)), (abi.OXG_OK, (p, sp, 4, p, sp, 0, 64, None, None, 0, 4))):
        assert lib.oxg_mxfp4_matmul(h, *args) == status, args
    assert lib.oxg_mxfp4_grouped_matmul(h, p, sp, 4, None, 1, p, sp, 4, 64, None, q, 0, 4) == abi.OXG_ERR_INVALID_ARG
    assert lib.oxg_mxfp4_grouped_matmul(h, p, sp, 4, p, 1025, p, sp, 4, 64, None, q, 0, 4) == abi.OXG_ERR_SHAPE
    assert lib.oxg_mxfp4_grouped_matmul(h, p, sp, 4, None, 0, p, sp, 4, 64, None, q, 0, 4) == abi.OXG_OK
    cuda_ctx.sync()
    assert (o == 3.0).all()


def test_outputs_past_2_to_31_elements(cuda_ctx):
    torch, mxfp4, _ = _torch()
    m, n, k = 33000, 65600, 32
    rng = np.random.default_rng(13)
    (ab, asc), (bb, bsc) = _operand(rng, m, k, spread=0), _operand(rng, n, k, spread=0)
    a, at, b, bt = _cuda(ab, asc, bb, bsc)
    got = mxfp4.mxfp4_matmul(a, at, b, bt)
    _check(got[-300:, -1000:], ref.values(ab[-300:], asc[-300:]), ref.values(bb[-1000:], bsc[-1000:]), None, "bfloat16")
    _check(got[:200, :500], ref.values(ab[:200], asc[:200]), ref.values(bb[:500], bsc[:500]), None, "bfloat16")


def test_graphs_and_streams(cuda_ctx):
    """Two captured graphs replayed side by side on two streams, with other inputs in their buffers than at capture."""
    torch, mxfp4, ffn = _torch()
    weights = mxfp4.quantize_mxfp4(torch.randn(512, 256, device="cuda"), tiled=True)
    xs = [torch.randn(300, 256, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    counts = torch.tensor([100, 0, 200], dtype=torch.int32, device="cuda")
    experts = torch.randn(3, 192, 256, device="cuda")
    eb, es = mxfp4.quantize_mxfp4(experts)
    es = mxfp4.tile_scales(es)

    def work(x):
        q = mxfp4.quantize_mxfp4(x, tiled=True)
        y = mxfp4.mxfp4_matmul(*q, *weights, out_dtype=torch.float32)
        h = ffn.swiglu_quantize_mxfp4(y, tiled=True)
        return mxfp4.mxfp4_grouped_matmul(*h, counts, eb, es, out_dtype=torch.float32)

    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    torch.cuda.synchronize()
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            work(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(work(x))
        graphs.append(g)
    for x in xs:
        x.copy_(torch.randn_like(x))
    want = [work(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w, o)
    cuda_ctx.sync()


def test_threads_on_streams_of_their_own(cuda_ctx):
    """Two host threads without a context of their own, each on its own stream, calling at once."""
    import threading
    torch, mxfp4, _ = _torch()
    w = mxfp4.quantize_mxfp4(torch.randn(2000, 1024, device="cuda"), tiled=True)
    xs = [torch.randn(m, 1024, device="cuda") for m in (40, 900)]
    want = [mxfp4.mxfp4_matmul(*mxfp4.quantize_mxfp4(x, tiled=True), *w) for x in xs]
    torch.cuda.synchronize()
    bad, gate = [], threading.Barrier(2)

    def work(x, y):
        st = torch.cuda.Stream()
        gate.wait()
        with torch.cuda.stream(st):
            for _ in range(100):
                got = mxfp4.mxfp4_matmul(*mxfp4.quantize_mxfp4(x, tiled=True), *w)
                st.synchronize()
                if not torch.equal(got, y):
                    bad.append(x.shape)
        mxfp4.device_context(x, None).sync()

    threads = [threading.Thread(target=work, args=a) for a in zip(xs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("tokens", [1, 6, 40, 200])
def test_in_turn_with_the_moe_kernels(cuda_ctx, tokens):
    """Products and quantisations between MoE forwards, whose kernels overlap their neighbours' ends as these do: the
    same bits as with a wait after every call."""
    torch, mxfp4, _ = _torch()
    from oxidized_gpt_oss_b200 import synth
    from oxidized_gpt_oss_b200.moe import MoELayer
    layer = MoELayer(synth.moe_layer(seed=8, hidden=576, intermediate=320, n_experts=8, top_k=4))
    layer.reserve(tokens)
    w1 = mxfp4.quantize_mxfp4(torch.randn(576, 1024, device="cuda") / 32, tiled=True)
    w2 = mxfp4.quantize_mxfp4(torch.randn(1024, 576, device="cuda") / 24, tiled=True)

    def rounds(x, wait):
        got = []
        for _ in range(8):
            q = mxfp4.quantize_mxfp4(x, tiled=True)
            wait()
            h = mxfp4.mxfp4_matmul(*q, *w1)
            wait()
            y = layer.forward(h)
            wait()
            q = mxfp4.quantize_mxfp4(y, tiled=True)
            wait()
            x = mxfp4.mxfp4_matmul(*q, *w2)
            wait()
            got += [h, y, x]
        return got

    x = torch.randn(tokens, 1024, device="cuda", dtype=torch.bfloat16)
    want = rounds(x, torch.cuda.synchronize)
    for _ in range(5):
        got = rounds(x, lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    cuda_ctx.sync()
    layer.release()


FIRST_IN_CAPTURE = """
import torch
from oxidized_gpt_oss_b200 import abi, mxfp4
torch.cuda.set_device(0)
mxfp4.context(None)
x, w = torch.randn(70, 512, device="cuda"), torch.randn(300, 512, device="cuda")
one = torch.randn(1, 4096, device="cuda"), torch.randn(300, 4096, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
def work():
    return [mxfp4.mxfp4_matmul(*mxfp4.quantize_mxfp4(a, tiled=True), *mxfp4.quantize_mxfp4(b, tiled=True)) for a, b in ((x, w), one)]
with torch.cuda.graph(g):
    out = work()
g.replay()
torch.cuda.synchronize()
for a, b in zip(out, work()):
    assert torch.equal(a, b)
print("replayed")
"""


def test_first_calls_in_a_capture():
    """A process whose first calls, once it has a context, are captured."""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "replayed" in r.stdout, r.stderr[-2000:]


def test_empty_operands(cuda_ctx):
    torch, mxfp4, ffn = _torch()
    none, w = mxfp4.quantize_mxfp4(torch.empty(0, 64, device="cuda"), tiled=True), mxfp4.quantize_mxfp4(torch.randn(8, 64, device="cuda"), tiled=True)
    assert mxfp4.mxfp4_matmul(*none, *w).shape == (0, 8)
    assert mxfp4.mxfp4_matmul(*w, *none).shape == (8, 0)
    b, s = mxfp4.quantize_mxfp4(torch.empty(0, 5, 64, device="cuda"))
    out = torch.full((8, 5), 3.0, device="cuda")
    assert (mxfp4.mxfp4_grouped_matmul(*w, torch.empty(0, dtype=torch.int32, device="cuda"), b, s, out=out) == 3).all()
    assert ffn.swiglu_quantize_mxfp4(torch.empty(3, 0, device="cuda"))[0].shape == (3, 0)
    cuda_ctx.sync()


def test_moe_block_with_4_bit_activations(cuda_ctx):
    """dispatch -> quantise -> gate/up products -> SwiGLU + quantise -> down products -> combine, the MoE block on 4-bit
    activations, against the same steps in 64 bits from the layer's own routing. A code may differ where the f32 sums
    of the first product lie at a border, so this is held to the size of the result: with 2880-long rows one code is a
    step of at most half its value, and under one in 10^4 lies that close."""
    torch, mxfp4, ffn = _torch()
    from oxidized_gpt_oss_b200 import synth
    from oxidized_gpt_oss_b200.moe import MoELayer
    d = synth.moe_layer(seed=3, hidden=576, intermediate=320, n_experts=8, top_k=4)
    x = torch.from_numpy(synth.activations(3, 100, 576).view(np.int16)).cuda()
    layer = MoELayer(d)
    rows, row_scale, counts = layer.dispatch(x)
    w = {k: torch.from_numpy(d[k]).cuda() for k in ("w1_blocks", "w1_scales", "w2_blocks", "w2_scales")}
    b1, b2 = (torch.from_numpy(d[k].view(np.int16)).cuda().view(torch.bfloat16) for k in ("b1", "b2"))
    s1, s2 = mxfp4.tile_scales(w["w1_scales"]), mxfp4.tile_scales(w["w2_scales"])
    a = mxfp4.quantize_mxfp4(rows, row_scale=row_scale, tiled=True)
    y1 = mxfp4.mxfp4_grouped_matmul(*a, counts, w["w1_blocks"], s1, bias=b1, out_dtype=torch.float32)
    h = ffn.swiglu_quantize_mxfp4(y1, tiled=True)
    y2 = mxfp4.mxfp4_grouped_matmul(*h, counts, w["w2_blocks"], s2, bias=b2, out_dtype=torch.float32)
    got = layer.combine(y2, 100)
    cuda_ctx.sync()
    idx, wts, _ = layer.route(x)
    # 64 bits, token by token slot
    xv = (synth.activations(3, 100, 576).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    idx, wts = idx.cpu().numpy(), wts.double().cpu().numpy()
    codes, sc = ref.quantize(xv)
    xq = ref.values(ref.pack(codes), sc)
    want = np.zeros((100, 576))
    f64 = lambda a: (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)  # noqa: E731
    for e in range(8):
        t, j = np.nonzero(idx == e)
        if not len(t):
            continue
        z = xq[t] @ ref.values(d["w1_blocks"][e], d["w1_scales"][e]).T + f64(d["b1"][e])
        codes, sc = ref.quantize(ref.swiglu(z, d["alpha"], d["limit"]))
        z = ref.values(ref.pack(codes), sc) @ ref.values(d["w2_blocks"][e], d["w2_scales"][e]).T + f64(d["b2"][e])
        np.add.at(want, t, wts[t, j][:, None] * z)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.linalg.norm(err) <= 1e-4 ** 0.5 / 2 * np.linalg.norm(want)
    layer.release()
