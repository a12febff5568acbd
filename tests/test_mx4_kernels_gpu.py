"""Every kernel of the MXFP4 products at the same sizes, whatever the library would choose for them: single CTAs, pairs of
CTAs, and clusters of 2 and of as many CTAs as can split K.

The bound is test_mx4_gpu's: with S = sum over k of |a b|, 2^-23 S for each of the n = ceil(k / 64) MMAs, 2^-24 of the
result for the bias, half a step, 2^-8, for bf16. Where r CTAs split K, each has at most n / r + 4 of the MMAs (K is
split in stages of 4) and a part S_i of S, which costs (n / r + 4) 2^-23 S in all; r - 1 additions of the parts cost
(r - 1) / 2 2^-23 S. Every CTA has a stage, so n > 4 (r - 1), and n / r + (r - 1) / 2 <= n: 4 more than unsplit.
"""
import ctypes

import numpy as np
import pytest

import mx4_reference as ref
from oxidized_gpt_oss_b200 import abi
from test_mx4_gpu import COUNTS, SHAPES, _bias, _cuda, _operand

pytestmark = pytest.mark.gpu
AUTO, FEW, PAIR, SPLIT = -1, 0, 1, 2


def _kernels(k):
    """(kernel, ranks) of all that can do a product of this length."""
    most = min(8, -(-k // 256))
    return [(FEW, 0), (PAIR, 0)] + [(SPLIT, r) for r in sorted({2, most}) if 2 <= r <= most]


def _run(ctx, a, b, n, k, out, kernel=AUTO, ranks=0, counts=None, bias=None):
    """oxgtest_mxfp4_product on torch's current stream; the kernel that ran."""
    import torch
    fn = ctx.lib.oxgtest_mxfp4_product
    P, I = ctypes.c_void_p, ctypes.c_int
    fn.restype, fn.argtypes = I, [P, P, P, I, P, I, P, P, I, I, P, P, I, ctypes.c_size_t, I, I, P]
    ran = (I * 2)()
    ctx.set_stream(torch.cuda.current_stream())
    code = abi.OXG_DTYPE_F32 if out.dtype == torch.float32 else abi.OXG_DTYPE_BF16
    abi.check(fn(ctx.handle, a[0].data_ptr(), a[1].data_ptr(), out.shape[0], None if counts is None else counts.data_ptr(),
                 -1 if counts is None else counts.numel(), b[0].data_ptr(), b[1].data_ptr(), n, k,
                 None if bias is None else bias.data_ptr(), out.data_ptr(), code, out.stride(0), kernel, ranks, ran), ctx.handle)
    assert kernel == AUTO or ran[0] == kernel
    return tuple(ran)


def _within(got, y, s, k, bias, split):
    """got (a tensor) against the sums y, whose magnitudes add up to s, plus bias."""
    bound = s * (-(-k // 64) + (4 if split else 0)) * 2.0 ** -23
    if bias is not None:
        y = y + bias
        bound = bound + np.abs(y) * 2.0 ** -24
    if got.element_size() == 2:
        bound = bound + (np.abs(y) + bound) * 2.0 ** -8
    err = np.abs(got.double().cpu().numpy() - y)
    assert np.all(err <= bound + 1e-300), (split, np.nanmax(err / np.maximum(bound, 1e-300)), np.argwhere(~(err <= bound))[:5])


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_on_every_kernel(cuda_ctx, m, n, k):
    """f32 and bf16, with and without a bias, even and odd n."""
    import torch
    rng = np.random.default_rng(m * 11 + n * 5 + k)
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, n, k, around=122)
    bias, bias64 = _bias(rng, n)
    a, b = _cuda(ab, ref.tile(asc, k)), _cuda(bb, ref.tile(bsc, k))
    av, bv = ref.values(ab, asc), ref.values(bb, bsc)
    y, s = av @ bv.T, np.abs(av) @ np.abs(bv).T
    for kernel, ranks in _kernels(k):
        for dtype in (torch.float32, torch.bfloat16):
            for with_bias in (False, True):
                out = torch.full((m, n), 9.0, device="cuda", dtype=dtype)
                _run(cuda_ctx, a, b, n, k, out, kernel, ranks, bias=bias if with_bias else None)
                cuda_ctx.sync()
                _within(out, y, s, k, bias64 if with_bias else None, kernel == SPLIT)


GROUPED = [*COUNTS, (850, [0, 113, 0, 225, 500, 1]), (8, [0, 3, 0, 0, 4, 0, 1, 0]), (20, [0] * 8), (1500, [1, 1480, 0, 7])]


@pytest.mark.parametrize("m,counts", GROUPED)
@pytest.mark.parametrize("n,k", [(130, 96), (64, 576), (321, 2112)])
def test_grouped_matmul_on_every_kernel(cuda_ctx, m, counts, n, k):
    """Ragged and empty groups, groups of more than one tile and more than one box of rows; rows past the last group keep
    what they held."""
    import torch
    rng = np.random.default_rng(m + n + len(counts))
    G = len(counts)
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, G, n, k, around=122)
    bias, bias64 = _bias(rng, G, n)
    a, b, (c,) = _cuda(ab, ref.tile(asc, k)), _cuda(bb, ref.tile(bsc, k)), _cuda(np.array(counts, np.int32))
    av, bv, held = ref.values(ab, asc), ref.values(bb, bsc), sum(counts)
    group = np.repeat(np.arange(G), counts)
    y, s = np.zeros((held, n)), np.zeros((held, n))
    for g in set(group):
        y[group == g] = av[:held][group == g] @ bv[g].T
        s[group == g] = np.abs(av[:held][group == g]) @ np.abs(bv[g]).T
    for kernel, ranks in _kernels(k):
        for dtype, with_bias in ((torch.float32, True), (torch.bfloat16, False), (torch.bfloat16, True)):
            out = torch.full((m, n), 55.0, device="cuda", dtype=dtype)
            _run(cuda_ctx, a, b, n, k, out, kernel, ranks, counts=c, bias=bias if with_bias else None)
            cuda_ctx.sync()
            _within(out[:held], y, s, k, bias64[group] if with_bias else None, kernel == SPLIT)
            assert (out[held:] == 55.0).all()


@pytest.mark.parametrize("counts", [[200, 300], [-1, 200], [2 ** 31 - 1, 2 ** 31 - 1], [401, 0], [399, 1]])
def test_counts_that_do_not_fit_on_every_kernel(cuda_ctx, counts):
    """Negative ones are taken as 0, the groups end with the rows, and the next sync says so (not for the last, which fit)."""
    import torch
    rng = np.random.default_rng(21)
    m, n, k = 400, 161, 576
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, 2, n, k)
    a, b, (c,) = _cuda(ab, ref.tile(asc, k)), _cuda(bb, ref.tile(bsc, k)), _cuda(np.array(counts, np.int32))
    first = min(max(counts[0], 0), m)
    last = min(first + max(counts[1], 0), m)
    av, bv = ref.values(ab, asc), ref.values(bb, bsc)
    y = np.concatenate([av[:first] @ bv[0].T, av[first:last] @ bv[1].T])
    s = np.concatenate([np.abs(av[:first]) @ np.abs(bv[0]).T, np.abs(av[first:last]) @ np.abs(bv[1]).T])
    for kernel, ranks in _kernels(k):
        whole = torch.full((m + 2, n), 55.0, device="cuda")
        _run(cuda_ctx, a, b, n, k, whole[1: m + 1], kernel, ranks, counts=c)
        if counts != [399, 1]:
            with pytest.raises(abi.OxgError, match="count"):
                cuda_ctx.sync()
        cuda_ctx.sync()
        _within(whole[1: last + 1], y, s, k, None, kernel == SPLIT)
        assert (whole[0] == 55.0).all() and (whole[last + 1:] == 55.0).all()


@pytest.mark.parametrize("spread", [2, 12, 30])
def test_scales_on_every_kernel(cuda_ctx, spread):
    """Blocks far apart within a row, rows far apart, byte 0 (2^-127), and 255, which makes its row or column NaN and no
    other: rows and columns of every tile of either CTA of a pair among them."""
    import torch
    rng = np.random.default_rng(spread)
    m, n, k = 460, 390, 1056
    (ab, asc), (bb, bsc) = _operand(rng, m, k, spread=spread), _operand(rng, n, k, spread=spread)
    asc = (asc + rng.integers(spread - 60, 61 - spread, m)[:, None]).astype(np.uint8)
    asc[7, 3], asc[300, 32] = 0, 0
    av, bv = ref.values(ab, asc), ref.values(bb, bsc)
    y, s = av @ bv.T, np.abs(av) @ np.abs(bv).T
    rows, cols = [5, 130, 229, 459], [3, 127, 128, 255, 256, 389]
    asn, bsn = asc.copy(), bsc.copy()
    for i, r in enumerate(rows):
        asn[r, 8 * i] = 255
    for i, c in enumerate(cols):
        bsn[c, 6 * i + 2] = 255
    nan = np.zeros((m, n), bool)
    nan[rows], nan[:, cols] = True, True
    a, b = _cuda(ab, ref.tile(asc, k)), _cuda(bb, ref.tile(bsc, k))
    an, bn = (a[0], *_cuda(ref.tile(asn, k))), (b[0], *_cuda(ref.tile(bsn, k)))
    out = torch.empty(m, n, device="cuda")
    for kernel, ranks in _kernels(k):
        _run(cuda_ctx, a, b, n, k, out, kernel, ranks)
        cuda_ctx.sync()
        _within(out, y, s, k, None, kernel == SPLIT)
        _run(cuda_ctx, an, bn, n, k, out, kernel, ranks)
        cuda_ctx.sync()
        got = out.cpu().numpy()
        assert np.array_equal(np.isnan(got), nan)
        _within(out[torch.from_numpy(~nan)], y[~nan], s[~nan], k, None, kernel == SPLIT)


@pytest.mark.parametrize("m,n,k", [(35, 91, 544), (230, 260, 544), (450, 515, 1088)])
@pytest.mark.parametrize("extra,offset", [(0, 0), (1, 1), (8, 3), (9, 8)])
def test_own_elements_only_on_every_kernel(cuda_ctx, m, n, k, extra, offset):
    """Outputs inside a wider matrix, at every alignment that its type allows: nothing around them is written."""
    import torch
    rng = np.random.default_rng(n + extra)
    (ab, asc), (bb, bsc) = _operand(rng, m, k), _operand(rng, n, k)
    a, b = _cuda(ab, ref.tile(asc, k)), _cuda(bb, ref.tile(bsc, k))
    av, bv = ref.values(ab, asc), ref.values(bb, bsc)
    y, s = av @ bv.T, np.abs(av) @ np.abs(bv).T
    for kernel, ranks in _kernels(k):
        for dtype in (torch.float32, torch.bfloat16):
            whole = torch.full((m + 2, n + extra + offset), 77.0, device="cuda", dtype=dtype)
            out = whole[1: m + 1, offset: offset + n]
            _run(cuda_ctx, a, b, n, k, out, kernel, ranks)
            cuda_ctx.sync()
            _within(out, y, s, k, None, kernel == SPLIT)
            out.fill_(77.0)
            assert (whole == 77.0).all()


def test_sums_that_f32_holds_are_the_same_on_every_kernel(cuda_ctx):
    """With every scale 1 the sums are multiples of 1/4 below 2^22: exact in any order, so all kernels agree bit for bit."""
    import torch
    rng = np.random.default_rng(31)
    for m, n, k in ((3, 70, 1056), (130, 200, 2880), (700, 600, 2080)):
        (ab, asc), (bb, bsc) = _operand(rng, m, k, spread=0), _operand(rng, n, k, spread=0)
        a, b = _cuda(ab, ref.tile(asc, k)), _cuda(bb, ref.tile(bsc, k))
        want = (ref.values(ab, asc) @ ref.values(bb, bsc).T).astype(np.float32)
        for kernel, ranks in _kernels(k):
            out = torch.empty(m, n, device="cuda")
            _run(cuda_ctx, a, b, n, k, out, kernel, ranks)
            cuda_ctx.sync()
            assert np.array_equal(out.cpu().numpy(), want)


def test_the_library_takes_each_kernel_where_it_is_meant_to(cuda_ctx):
    """Few tiles and a long K are split, many rows go to pairs, few rows over many tiles to single CTAs."""
    import torch
    for (m, n, k), kernel in (((8, 5120, 2880), SPLIT), ((1, 2880, 4096), SPLIT), ((40, 38500, 544), FEW), ((3, 19300, 2400), FEW),
                              ((2000, 1300, 1184), PAIR), ((8192, 5120, 64), PAIR)):
        a = torch.zeros(m, k // 2, dtype=torch.uint8, device="cuda"), torch.zeros((k + 127) // 128, m, 4, dtype=torch.uint8, device="cuda")
        b = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda"), torch.zeros((k + 127) // 128, n, 4, dtype=torch.uint8, device="cuda")
        out = torch.ones(m, n, device="cuda")
        ran = _run(cuda_ctx, a, b, n, k, out)
        assert ran[0] == kernel and (ran[1] > 1) == (kernel == SPLIT), (m, n, k, ran)
        assert not out.any()
    cuda_ctx.sync()


def test_kernels_that_cannot_do_a_shape_are_refused(cuda_ctx):
    import torch
    a = torch.zeros(4, 128, dtype=torch.uint8, device="cuda"), torch.zeros(2, 4, 4, dtype=torch.uint8, device="cuda")
    out = torch.ones(4, 4, device="cuda")
    for kernel, ranks in ((SPLIT, 0), (SPLIT, 1), (SPLIT, 2), (SPLIT, 9)):  # one stage of K: nothing to split
        with pytest.raises(abi.OxgError):
            _run(cuda_ctx, a, a, 4, 256, out, kernel, ranks)
    with pytest.raises(abi.OxgError, match="unknown kernel"):
        _run(cuda_ctx, a, a, 4, 256, out, 3, 0)
    cuda_ctx.sync()
    assert (out == 1).all()
