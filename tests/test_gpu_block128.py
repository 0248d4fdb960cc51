"""Block-128 quantizer and matrix products against plain 64-bit forms, and the MoE layer built from them and the router."""
import os
import subprocess
import sys

import pytest
import torch

import mx8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FLOOR = 2.0 ** -110
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cdiv(a):
    return (a + 127) // 128


def bits(t):
    return t.contiguous().view(torch.uint8)


def quotient(x, amax, dtype):
    """x * 448 / amax rounded to fp32: from 64 bits, or for bf16 input as x * fl(448 / amax).  (A Python number divided by a tensor would be
    reciprocal times number: two roundings.)"""
    if dtype == torch.bfloat16:
        return x * (torch.full_like(amax, 448.0) / amax)
    return (x.double() * 448.0 / amax.double()).float()


def quant_ref(x, square=False):
    """x [M, N] on the CPU -> (bytes, scales) by the definition: the kernel has to give the same bits"""
    dtype = x.dtype
    M, N = x.shape
    full = torch.zeros(cdiv(M) * 128, cdiv(N) * 128)
    full[:M, :N] = x.float()
    if square:
        t = full.view(cdiv(M), 128, cdiv(N), 128)
        amax = t.abs().amax((1, 3)).clamp(min=FLOOR)
        q = quotient(t, amax[:, None, :, None], dtype).view(full.shape)[:M, :N]
        return q.to(torch.float8_e4m3fn), amax / 448.0
    t = full.view(-1, cdiv(N), 128)
    amax = t.abs().amax(2).clamp(min=FLOOR)
    q = quotient(t, amax[:, :, None], dtype).view(full.shape)[:M, :N]
    return q.to(torch.float8_e4m3fn), (amax / 448.0)[:M].t().contiguous()


def check_quant(x, square=False, row_index=None):
    q, sc, qt, sct = mx8.quantize_block128(x, True, True, square=square, row_index=row_index)
    assert mx8.device_status() == 0
    xs = x.cpu()
    if row_index is not None:
        i = row_index.cpu().long()
        ok = (i >= 0) & (i < xs.shape[0])
        xs = torch.where(ok[:, None], xs[torch.where(ok, i, 0)], torch.zeros((), dtype=xs.dtype))
    mats = xs if xs.dim() == 3 else xs[None]
    lead = x.dim() == 3
    for e in range(mats.shape[0]):
        pick = (lambda t: t[e].cpu()) if lead else (lambda t: t.cpu())
        for got, got_sc, ref in ((q, sc, quant_ref(mats[e], square)), (qt, sct, quant_ref(mats[e].t().contiguous(), square))):
            assert torch.equal(pick(got_sc), ref[1])
            assert torch.equal(bits(pick(got)), bits(ref[0]))
            # and against x itself in 64 bits: half a step of 3 bits (2^-4), or of the smallest step 2^-9 of a block, plus the
            # fp32 roundings on the way
            wide = torch.repeat_interleave(torch.repeat_interleave(ref[1].double(), 128, 0), 128, 1)[:got.shape[-2], :got.shape[-1]] if square \
                else torch.repeat_interleave(ref[1].double().t(), 128, 1)[:, :got.shape[-1]]
            want = mats[e].double() if got is q else mats[e].t().double()
            assert ((pick(got).double() * wide - want).abs() <= (2.0 ** -4 + 2.0 ** -21) * want.abs() + 2.0 ** -10 * wide).all()
    # one orientation alone gives the same
    a = mx8.quantize_block128(x, True, False, square=square, row_index=row_index)
    b = mx8.quantize_block128(x, False, True, square=square, row_index=row_index)
    assert a[2] is None and a[3] is None and b[0] is None and b[1] is None
    assert torch.equal(bits(a[0]), bits(q)) and torch.equal(a[1], sc) and torch.equal(bits(b[2]), bits(qt)) and torch.equal(b[3], sct)


def make_x(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    x[..., 0, :] = 0.0                                            # a row of zero blocks
    x.view(-1)[::97] *= 1000.0
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("square", [False, True])
def test_quantize_gives_the_nearest_byte(square, dtype):
    """No byte lies nearer to x * 448 / amax than the one given.  Slack: fp32 input is rounded to fp32 first (2^-24 of the quotient); for
    bf16 that costs nothing, only the 64 bits of this check do (2^-51)."""
    x = make_x(513, 640, seed=31, dtype=dtype)
    q, sc, _, _ = mx8.quantize_block128(x, True, False, square=square)
    t = torch.zeros(640, 640, dtype=torch.float64)
    t[:513] = x.cpu().double()
    t = t.view(5, 128, 5, 128) if square else t.view(640, 1, 5, 128)
    exact = (t * 448.0 / t.abs().amax((1, 3), keepdim=True).clamp(min=FLOOR)).view(640, 640)[:513]
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    table = table[~table.isnan()].unique()
    i = torch.searchsorted(table, exact).clamp(1, len(table) - 1)
    nearest = torch.minimum((exact - table[i - 1]).abs(), (exact - table[i]).abs())
    slack = 2.0 ** -51 if dtype == torch.bfloat16 else 2.0 ** -24
    assert ((q.cpu().double() - exact).abs() <= nearest + slack * exact.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (7, 200), (128, 128), (129, 257), (300, 1000), (513, 64), (1030, 384), (2, 130, 140), (3, 256, 128)])
def test_quantize(shape, dtype):
    x = make_x(*shape, seed=sum(shape), dtype=dtype)
    check_quant(x)
    check_quant(x, square=True)


def test_quantize_strided_offset_and_gathered():
    wide = make_x(300, 700, seed=1)
    for sl in (wide[:, :500], wide[:, 3:260], wide[::2, 4:132]):
        check_quant(sl)
        check_quant(sl, square=True)
    g = torch.Generator().manual_seed(2)
    for rows in (1, 130, 500):
        idx = torch.randint(-1, 301, (rows,), generator=g, dtype=torch.int32)       # -1 and 300 lie outside: zero rows
        if rows > 4:
            idx[3] = idx[2]                                                         # the same row twice
        check_quant(wide[:, :260], row_index=idx.to(DEV))


def test_quantize_tiny_large_and_non_finite():
    x = torch.zeros(130, 256)
    x[0, :128] = 2.0 ** -130                                      # below the floor of amax
    x[1, 128:] = 3.0e38
    x[2, 5] = 2.0 ** -149
    check_quant(x.to(DEV))
    for bad in (float("inf"), float("nan")):
        y = make_x(130, 256, seed=3, dtype=torch.float32)
        y[4, 7] = bad
        q, sc, qt, sct = mx8.quantize_block128(y, True, True)
        deq = q.float() * torch.repeat_interleave(sc.t(), 128, 1)
        deqt = qt.float() * torch.repeat_interleave(sct.t(), 128, 1)[:, :130]
        assert torch.isnan(deq[4, 7]) and torch.isnan(deqt[7, 4])
        if bad != bad:
            assert torch.isnan(deq[4, :128]).all() and torch.isnan(deqt[7, :128]).all()
        assert torch.isfinite(deq[5:]).all() and torch.isfinite(deqt[8:]).all() and torch.isfinite(deq[4, 128:]).all()


# ------------------------------------------------------------------------------------------------ products
def rows64(q, sc):
    return q.cpu().double() * torch.repeat_interleave(sc.cpu().double().t(), 128, 1)[:, :q.shape[1]]


def square64(q, sc):
    return q.cpu().double() * torch.repeat_interleave(torch.repeat_interleave(sc.cpu().double(), 128, 0)[:q.shape[0]], 128, 1)[:, :q.shape[1]]


def check_c(c, a64, b64, what=""):
    """Products of two E4M3 values are exact in fp32; a block of 128 of them added in fp32 in any order, or cut instead of rounded,
    is off by at most 128 * 2^-23 of the sum of magnitudes; the scales' product and the block's scaling add two roundings and every
    further block one (2^-24 each).  The output type adds half a step (bf16: 2^-8)."""
    want, size = a64 @ b64.t(), a64.abs() @ b64.abs().t()
    tol = (128 * 2.0 ** -23 + (cdiv(a64.shape[1]) + 4) * 2.0 ** -24) * size
    if c.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    off = (c.cpu().double() - want).abs()
    assert (off <= tol + 1e-300).all(), f"{what}: {float((off / (tol + 1e-300)).nan_to_num(nan=1e9).max()):.3g} times the bound"


def operands(M, N, K, b, seed=0):
    a = make_x(M, K, seed=seed)
    w = make_x(N, K, seed=seed + 1, dtype=torch.float32) * 0.02
    qa, sa, _, _ = mx8.quantize_block128(a)
    qb, sb, _, _ = mx8.quantize_block128(w, square=(b == "square"))
    return qa, sa, qb, sb, rows64(qa, sa), (square64 if b == "square" else rows64)(qb, sb)


@pytest.mark.parametrize("b", ["square", "rows"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 128, 128), (1, 520, 1040), (3, 300, 100), (16, 256, 512), (17, 129, 272), (32, 1000, 640),
                                   (33, 64, 130), (64, 512, 384), (65, 100, 200), (128, 128, 128), (128, 256, 256), (129, 257, 144), (200, 72, 1000),
                                   (300, 1030, 520), (1000, 640, 1152), (2100, 2304, 200), (70, 300, 2048), (150, 1000, 1100), (64, 128, 600),
                                   (5, 2500, 1030), (40, 20000, 260), (600, 3000, 1024)])
def test_product(shape, b):
    M, N, K = shape
    qa, sa, qb, sb, a64, b64 = operands(M, N, K, b, seed=M + N + K)
    for dtype in (torch.bfloat16, torch.float32):
        c = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        assert mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks=b) is c
        assert mx8.device_status() == 0
        check_c(c, a64, b64, f"{shape} {b} {dtype}")
        again = torch.full_like(c, 7.0)
        mx8.gemm_block128(qa, sa, qb, sb, again, b_blocks=b)
        assert torch.equal(c, again)


def test_product_into_and_from_slices():
    M, N, K = 150, 200, 300
    for m in (M, 5):
        qa, sa, qb, sb, a64, b64 = operands(m, N, K, "square", seed=m)
        big = torch.full((m + 2, N + 9), 3.0, dtype=torch.bfloat16, device=DEV)
        mx8.gemm_block128(qa, sa, qb, sb, big[1:m + 1, 5:N + 5])
        assert mx8.device_status() == 0
        check_c(big[1:m + 1, 5:N + 5], a64, b64)
        edge = big.clone()
        edge[1:m + 1, 5:N + 5] = 3.0
        assert (edge == 3.0).all()
    # rows of A inside a larger buffer, with the larger buffer's scales
    qa, sa, qb, sb, a64, b64 = operands(M, N, K, "rows", seed=8)
    c = torch.empty(40, N, device=DEV)
    mx8.gemm_block128(qa[100:140], sa[:, 100:140], qb, sb, c, b_blocks="rows")
    check_c(c, a64[100:140], b64)


def test_one_row_needs_no_pitch():
    qa, sa, qb, sb, a64, b64 = operands(1, 50, 200, "square", seed=5)
    alone = bits(qa).view(torch.float8_e4m3fn)                     # 200 bytes, contiguous
    c = torch.empty(1, 50, device=DEV)
    mx8.gemm_block128(alone, sa, qb, sb, c)
    check_c(c, a64, b64)


def test_non_finite_blocks_reach_their_rows_only():
    qa, sa, qb, sb, a64, b64 = operands(200, 300, 256, "square", seed=4)
    sa[1, 7] = float("nan")
    c = torch.empty(200, 300, device=DEV)
    mx8.gemm_block128(qa, sa, qb, sb, c)
    assert torch.isnan(c[7]).all()
    keep = torch.arange(200) != 7
    check_c(c[keep.to(DEV)], a64[keep], b64)


@pytest.mark.parametrize("sizes", [[5], [0, 1, 0, 130, 7, 0], [128, 256, 1], [0, 0, 0], [300, 0, 0, 0, 0, 0, 0, 2], [1] * 40, [3] * 256])
def test_grouped_product(sizes):
    G, R, N, K = len(sizes), sum(sizes), 200, 272
    if G > 100:
        N, K = 40, 144
    cap = R + 37
    a = make_x(cap, K, seed=R)
    w = make_x(G, N, K, seed=G, dtype=torch.float32) * 0.02
    qa, sa, _, _ = mx8.quantize_block128(a)
    qb, sb, _, _ = mx8.quantize_block128(w, square=True)
    grp = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        c = torch.full((cap, N), 5.0, dtype=dtype, device=DEV)
        mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=grp)
        assert mx8.device_status() == 0
        a64, at = rows64(qa, sa), 0
        for g, n in enumerate(sizes):
            if n:
                check_c(c[at:at + n], a64[at:at + n], square64(qb[g], sb[g]), f"group {g}")
            at += n
        assert (c[at:] == 5.0).all()


@pytest.mark.parametrize("sizes", [[128], [0, 256, 128, 0], [384, 0, 0, 128, 640], [128] * 9])
@pytest.mark.parametrize("mn", [(64, 40), (200, 300), (129, 520)])
def test_weight_gradient_product(sizes, mn):
    G, R = len(sizes), sum(sizes)
    M, N = mn
    pad = 64                                                       # rows behind the last group take no part
    y, x = make_x(R + pad, M, seed=R, dtype=torch.float32), make_x(R + pad, N, seed=R + 1)
    _, _, qa, sa = mx8.quantize_block128(y, False, True)
    _, _, qb, sb = mx8.quantize_block128(x, False, True)
    grp = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        c = torch.full((G, M, N), float("nan"), dtype=dtype, device=DEV)
        mx8.gemm_block128_wgrad(qa, sa, qb, sb, c, grp)
        assert mx8.device_status() == 0
        a64, b64, at = rows64(qa, sa), rows64(qb, sb), 0
        for g, n in enumerate(sizes):
            if n:
                check_c(c[g], a64[:, at:at + n], b64[:, at:at + n], f"group {g}")
            else:
                assert (c[g] == 0).all()
            at += n


def test_group_sizes_that_do_not_fit_are_cut_and_reported():
    K, N = 256, 64
    qa, sa, _, _ = mx8.quantize_block128(make_x(100, K))
    qb, sb, _, _ = mx8.quantize_block128(make_x(3, N, K), square=True)
    guard = torch.full((140, N), 9.0, device=DEV)
    for sizes in ([50, 60, 10], [-4, 20, 10], [2 ** 31 - 1] * 3):
        mx8.gemm_block128(qa, sa, qb, sb, guard[:100], group_rows=torch.tensor(sizes, dtype=torch.int32, device=DEV))
        with pytest.raises(mx8.Mx8Error):
            mx8.device_status()
        assert (guard[100:] == 9.0).all()
        assert mx8.device_status() == 0
    _, _, qt, st = mx8.quantize_block128(make_x(300, 64), False, True)
    c = torch.empty(2, 64, 64, device=DEV)
    for sizes in ([100, 128], [256, 256], [-128, 128]):
        mx8.gemm_block128_wgrad(qt, st, qt, st, c, torch.tensor(sizes, dtype=torch.int32, device=DEV))
        with pytest.raises(mx8.Mx8Error):
            mx8.device_status()


def test_refusals():
    qa, sa, qb, sb, _, _ = operands(20, 40, 200, "square")
    c = torch.empty(20, 40, dtype=torch.bfloat16, device=DEV)
    g = torch.tensor([20], dtype=torch.int32, device=DEV)
    for bad in (lambda: mx8.gemm_block128(qa, sa, qb, sb, c[:10]), lambda: mx8.gemm_block128(qa, sa, qb, sb, c.half()),
                lambda: mx8.gemm_block128(qa, sa.t(), qb, sb, c), lambda: mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks="rows"),
                lambda: mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks="columns"), lambda: mx8.gemm_block128(qa, sa.double(), qb, sb, c),
                lambda: mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=g), lambda: mx8.gemm_block128(qa.cpu(), sa, qb, sb, c),
                lambda: mx8.gemm_block128(qa, sa.cpu(), qb, sb, c), lambda: mx8.gemm_block128(qa, sa, qb[:, :100], sb, c),
                lambda: mx8.gemm_block128(qa, sa, qb[None], sb[None], c, group_rows=g.long()),
                lambda: mx8.gemm_block128(qa[:0], sa[:, :0], qb, sb, c[:0]),
                lambda: mx8.quantize_block128(torch.zeros(4, 4, dtype=torch.float16, device=DEV)),
                lambda: mx8.quantize_block128(torch.zeros(4, 8, device=DEV).t()), lambda: mx8.quantize_block128(torch.zeros(4, 8, device=DEV), False, False),
                lambda: mx8.quantize_block128(torch.zeros(4, 8, device=DEV), square=True, row_index=g),
                lambda: mx8.quantize_block128(torch.zeros(4, 8, device=DEV), row_index=g.long()),
                lambda: mx8.gemm_block128_wgrad(qa, sa, qa, sa, torch.empty(2, 20, 20, device=DEV), g)):
        with pytest.raises(ValueError):
            bad()
    tight = qa.contiguous()                                        # rows of 200 bytes: no 16-byte boundary
    with pytest.raises(mx8.Mx8Error):
        mx8.gemm_block128(tight, sa, qb, sb, c)


def test_side_stream_and_graphs_at_once():
    qa, sa, qb, sb, a64, b64 = operands(40, 640, 1024, "square", seed=20)
    qc, scc, qd, sd, c64, d64 = operands(600, 640, 1024, "square", seed=21)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for ops, M in (((qa, sa, qb, sb), 40), ((qc, scc, qd, sd), 600)):
        out = torch.zeros(M, 640, device=DEV)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            mx8.gemm_block128(*ops, out)
        graphs.append(gr)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s, gr in zip(streams, graphs):
        with torch.cuda.stream(s):
            for _ in range(3):
                gr.replay()
    torch.cuda.synchronize()
    assert mx8.device_status() == 0
    check_c(outs[0], a64, b64)
    check_c(outs[1], c64, d64)


@pytest.mark.parametrize("b", ["square", "rows"])
@pytest.mark.parametrize("shape", [(300, 1500, 1500), (320, 1000, 1400), (200, 500, 1030), (400, 1100, 4200), (700, 1601, 640)])
def test_product_in_parts(shape, b):
    """small tiles with K in two, four and eight parts, two parts of a long K, and whole"""
    qa, sa, qb, sb, a64, b64 = operands(*shape, b, seed=sum(shape))
    c = torch.full((shape[0], shape[1] + 1), 6.0, dtype=torch.bfloat16, device=DEV)
    mx8.gemm_block128(qa, sa, qb, sb, c[:, 1:], b_blocks=b)
    assert mx8.device_status() == 0
    check_c(c[:, 1:], a64, b64)
    again = torch.empty(shape[0], shape[1], device=DEV)
    mx8.gemm_block128(qa, sa, qb, sb, again, b_blocks=b)
    check_c(again, a64, b64)
    assert (c[:, 0] == 6.0).all()


@pytest.mark.parametrize("b", ["square", "rows"])
def test_product_on_many_large_tiles(b):
    """more K blocks than the rings hold, more tiles than one wave for neither form of the scales"""
    qa, sa, qb, sb, a64, b64 = operands(1500, 1700, 1300, b, seed=40)
    for c in (torch.empty(1500, 1700, device=DEV), torch.empty(1500, 1701, dtype=torch.bfloat16, device=DEV)[:, 1:]):
        mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks=b)
        assert mx8.device_status() == 0
        check_c(c, a64, b64)


@pytest.mark.parametrize("b", ["square", "rows"])
@pytest.mark.parametrize("shape", [(1, 7, 15), (1, 5, 17), (1, 1030, 4111), (1, 130, 9000), (2, 129, 520), (3, 64, 2048), (4, 66, 513), (5, 200, 300), (16, 300, 1000),
                                   (2, 7000, 5000), (9, 3000, 2000), (16, 2500, 900)])
def test_single_tokens(shape, b):
    """few rows, with rubbish behind the ends of A's and B's rows and around C; the last shapes have too many products for vectors"""
    M, N, K = shape
    qa, sa, qb, sb, a64, b64 = operands(M, N, K, b, seed=M + N + K)
    pa, pb = (torch.full((t.shape[0], cdiv(K) * 128 + 16), 0x7F, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for t in (qa, qb))
    pa[:, :K], pb[:, :K] = qa, qb
    for dtype in (torch.bfloat16, torch.float32):
        store = torch.full((M + 2, N + 3), 4.0, dtype=dtype, device=DEV)
        c = store[1:M + 1, 1:N + 1]
        mx8.gemm_block128(pa[:, :K], sa, pb[:, :K], sb, c, b_blocks=b)
        assert mx8.device_status() == 0
        check_c(c, a64, b64, f"{shape} {b} {dtype}")
        c.fill_(4.0)
        assert (store == 4.0).all()


@pytest.mark.parametrize("sizes,cap", [([1], 1), ([0, 0, 1, 0], 2), ([2, 0, 3, 1], 8), ([0] * 40 + [1] + [0] * 30 + [4], 6), ([1] * 8, 8), ([0, 0], 3), ([5, 0, 11], 20)])
def test_single_tokens_of_groups(sizes, cap):
    G, N, K = len(sizes), 70, 600
    qa, sa, _, _ = mx8.quantize_block128(make_x(cap, K, seed=cap))
    qb, sb, _, _ = mx8.quantize_block128(make_x(G, N, K, seed=G, dtype=torch.float32) * 0.02, square=True)
    c = torch.full((cap, N), 5.0, device=DEV)
    mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=torch.tensor(sizes, dtype=torch.int32, device=DEV))
    assert mx8.device_status() == 0
    a64, at = rows64(qa, sa), 0
    for g, n in enumerate(sizes):
        if n:
            check_c(c[at:at + n], a64[at:at + n], square64(qb[g], sb[g]), f"group {g}")
        at += n
    assert (c[at:] == 5.0).all()
    for bad in ([cap + 1] + [0] * (G - 1), [-1] + [0] * (G - 1), [2 ** 31 - 1] * G):
        mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=torch.tensor(bad, dtype=torch.int32, device=DEV))
        with pytest.raises(mx8.Mx8Error):
            mx8.device_status()


@pytest.mark.parametrize("sizes,N,K", [([0, 1, 0, 130, 7, 0], 200, 1100), ([20] * 9, 700, 1100), ([20] * 8, 896, 1040), ([0, 0, 0], 130, 2048), ([64], 100, 4100),
                                       ([1100, 0, 2200], 300, 1300), ([700, 3, 0, 129, 256, 128, 40], 600, 1300), ([0, 127, 64, 65, 0, 1], 1030, 1500),
                                       ([20] * 9, 384, 1500), ([20] * 9, 700, 1500), ([700, 3, 0, 129, 256, 128, 40], 1030, 1300), ([0, 127, 64, 65, 0, 1], 2100, 1500),
                                       ([700, 3, 0, 129, 256, 128, 40], 2100, 272), ([1500, 1300], 1030, 272)])
def test_grouped_product_on_tiles_of_every_kind(sizes, N, K):
    """few tiles, with K in eight, four and two parts; groups of many rows; tiles of one block and of pairs, more of them than one wave"""
    G, cap = len(sizes), sum(sizes) + 37
    qa, sa, _, _ = mx8.quantize_block128(make_x(cap, K, seed=cap))
    qb, sb, _, _ = mx8.quantize_block128(make_x(G, N, K, seed=G, dtype=torch.float32) * 0.02, square=True)
    grp = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    for store in (torch.full((cap, N), 5.0, device=DEV), torch.full((cap, N + 1), 5.0, dtype=torch.bfloat16, device=DEV)):
        c = store[:, :N]
        for _ in range(2):
            mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=grp)
        assert mx8.device_status() == 0
        a64, at = rows64(qa, sa), 0
        for g, n in enumerate(sizes):
            if n:
                check_c(c[at:at + n], a64[at:at + n], square64(qb[g], sb[g]), f"group {g}")
            at += n
        assert (c[at:] == 5.0).all() and (store[:, N:] == 5.0).all()


@pytest.mark.parametrize("sizes", [[1280, 0, 128, 1024], [128] * 9])
def test_weight_gradient_on_large_tiles(sizes):
    test_weight_gradient_product(sizes, (600, 1701))


@pytest.mark.parametrize("sizes,mn", [([4096, 128], (64, 100)), ([0, 2944, 128], (130, 257)), ([1408] * 12, (100, 500)), ([128, 0, 8064], (200, 129))])
def test_weight_gradient_in_parts(sizes, mn):
    """few tiles, groups with fewer blocks than there are parts of K"""
    test_weight_gradient_product(sizes, mn)


def test_small_and_large_tiles_on_two_streams():
    a = operands(3000, 2100, 700, "square", seed=50)
    b = operands(64, 512, 4096, "square", seed=51)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for rep in range(4):
        for st, ops in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                outs.append(mx8.gemm_block128(*ops[:4], torch.empty(ops[0].shape[0], ops[2].shape[0], device=DEV)))
    torch.cuda.synchronize()
    assert mx8.device_status() == 0
    for i, c in enumerate(outs):
        if i < 2:
            check_c(c, *(a, b)[i][4:])
        else:
            assert torch.equal(c, outs[i % 2])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_offsets_beyond_32_bits(m):
    """C that spans more than 2^32 elements is written where it should be and nowhere between"""
    N, K, pitch = 72, 260, 2 ** 32 // m + 7
    qa, sa, qb, sb, a64, b64 = operands(m + 1, N, K, "square", seed=m)
    store = torch.full(((m + 1) * pitch,), 2.0, dtype=torch.bfloat16, device=DEV)
    c = store.as_strided((m + 1, N), (pitch, 1))
    mx8.gemm_block128(qa, sa, qb, sb, c)
    assert mx8.device_status() == 0
    check_c(c, a64, b64)
    c.fill_(2.0)
    assert all(bool((part == 2.0).all()) for part in store.split(2 ** 28))


def test_quantize_beyond_32_bits():
    """input and transposed bytes of more than 2^32 bytes: the last rows get what they get by themselves"""
    N = 2 ** 27 + 24
    x = torch.empty(33, N, dtype=torch.bfloat16, device=DEV)
    for part in x.view(-1).split(2 ** 28):
        part.copy_(torch.arange(part.numel(), device=DEV, dtype=torch.int32) % 509 - 254)
    q, sc, qt, sct = mx8.quantize_block128(x, True, True)
    n0 = 2 ** 27 - 256                                             # columns from a block's start on
    a = mx8.quantize_block128(x[:, n0:].contiguous(), True, True)
    assert torch.equal(bits(q[:, n0:]), bits(a[0])) and torch.equal(sc[n0 // 128:], a[1])
    assert torch.equal(bits(qt[n0:]), bits(a[2])) and torch.equal(sct[:, n0:], a[3])


FRESH = r"""
import sys, threading
sys.path.insert(0, ROOT + "/gpu-experiments_b200")
import torch
import mx8
torch.zeros(1, device="cuda")                    # context only: the library's first calls race, or are captured
g = torch.Generator().manual_seed(1)
xs = [torch.randn(80 + 300 * i, 1200, generator=g).cuda() for i in range(4)]
ws = [torch.randn(700, 1200, generator=g).cuda() for i in range(4)]
ls = [torch.randn(3000, 64, generator=g).cuda() for i in range(4)]
def work(i):
    q, s, _, _ = mx8.quantize_block128(xs[i])
    b, t, _, _ = mx8.quantize_block128(ws[i], square=True)
    c = mx8.gemm_block128(q, s, b, t, torch.zeros(xs[i].shape[0], 700, device="cuda"))
    r = mx8.router_topk(ls[i], 6)
    return [c, *r, mx8.router_topk_bwd(ls[i], r[0], r[1], r[2], r[3], r[5], r[1])]
torch.cuda.synchronize()
got, errors = [None] * 4, []
if MODE == "threads":
    barrier = threading.Barrier(4)
    def worker(i):
        try:
            s = torch.cuda.Stream()
            barrier.wait()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = work(i)
                s.synchronize()
        except Exception as e:
            errors.append(repr(e))
    threads = [threading.Thread(target=worker, args=(i,)) for i in range(4)]
    for t in threads: t.start()
    for t in threads: t.join()
else:
    graphs = [torch.cuda.CUDAGraph() for _ in range(4)]
    for i in range(4):
        with torch.cuda.graph(graphs[i]):
            got[i] = work(i)
    for gr in graphs * 2:
        gr.replay()
torch.cuda.synchronize()
assert not errors, errors
assert mx8.device_status() == 0
for i in range(4):
    for a, b in zip(got[i], work(i)):
        assert torch.equal(a, b)
print("FRESH_OK")
"""


@pytest.mark.parametrize("mode", ["threads", "capture"])
def test_first_calls_in_threads_and_under_capture(mode):
    r = subprocess.run([sys.executable, "-c", f"ROOT, MODE = {ROOT!r}, {mode!r}\n" + FRESH], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "FRESH_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


# ------------------------------------------------------------------------------------------------ together
def test_moe_layer_forward_and_backward_from_the_router_to_the_weight_gradients():
    """One training step of an MoE layer on one rank: router, schedule, gathered quantization, experts' products, SwiGLU, combine,
    weighted sum; then back to the logits and the weights.  Every stage against 64 bits on the inputs it actually had."""
    T, H, I, E, k = 300, 256, 192, 8, 2
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    wr = torch.randn(E, H, generator=g) * H ** -0.5
    w = {n: (torch.randn(E, *s, generator=g) * 0.06).to(DEV) for n, s in (("gate", (I, H)), ("up", (I, H)), ("down", (H, I)))}
    logits = (x.float().cpu() @ wr.t()).to(DEV)
    mask = torch.arange(T, device=DEV) < T - 20
    idx, wt, lse, counts, _, n, loss = mx8.router_topk(logits, k, token_mask=mask)
    cap = (T * k // 256 + E) * 256
    peer_rank, peer_tok, rows, per_expert = mx8.schedule(idx[None].contiguous(), E, cap, 0)
    assert mx8.device_status() == 0
    src = torch.where(peer_rank >= 0, peer_tok // k, -1).to(torch.int32)
    assert int((src >= 0).sum()) == int(counts.sum()) == (T - 20) * k
    qx, sx, qxt, sxt = mx8.quantize_block128(x, True, True, row_index=src)
    quant = {name: mx8.quantize_block128(v, True, True, square=True) for name, v in w.items()}
    new = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    gate = mx8.gemm_block128(qx, sx, *quant["gate"][:2], new(cap, I), group_rows=per_expert)
    up = mx8.gemm_block128(qx, sx, *quant["up"][:2], new(cap, I), group_rows=per_expert)
    hid = mx8.swiglu_bf16(gate, up)
    qh, sh, qht, sht = mx8.quantize_block128(hid, True, True)
    y = mx8.gemm_block128(qh, sh, *quant["down"][:2], new(cap, H), group_rows=per_expert)
    buf = new(T * k, H)
    mx8.combine(y, peer_rank, peer_tok, rows, [buf.data_ptr()], T * k)
    out = mx8.fwd_epilogue(None, buf, wt)
    assert mx8.device_status() == 0
    sizes = per_expert.tolist()

    def grouped(c, qa, sa, qb, sb):
        a64, at = rows64(qa, sa), 0
        for e, m in enumerate(sizes):
            if m:
                check_c(c[at:at + m], a64[at:at + m], square64(qb[e], sb[e]), f"expert {e}")
            at += m

    grouped(gate, qx, sx, *quant["gate"][:2])
    grouped(up, qx, sx, *quant["up"][:2])
    grouped(y, qh, sh, *quant["down"][:2])
    want = (buf.cpu().double().view(T, k, H) * wt.cpu().double()[:, :, None]).sum(1)
    # k products and sums in fp32, then bf16
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * (buf.cpu().double().view(T, k, H).abs() * wt.cpu().double()[:, :, None]).sum(1)).all()
    assert (out[T - 20:] == 0).all()

    # ---- backward
    d_out = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    d_wt = mx8.bwd_topk_weights(d_out, buf, idx)
    d_loss = torch.tensor([0.01], device=DEV)
    d_logits = mx8.router_topk_bwd(logits, idx, wt, lse, counts, n, d_wt, d_loss)
    ref_wt = torch.where(idx.cpu() >= 0, (buf.cpu().double().view(T, k, H) * d_out.cpu().double()[:, None]).sum(2), 0.0)
    assert ((d_wt.cpu().double() - ref_wt).abs() <= 32 * 2.0 ** -24 * (buf.cpu().double().view(T, k, H) * d_out.cpu().double()[:, None]).abs().sum(2)).all()
    p = torch.softmax(logits.cpu().double(), 1)
    i = idx.cpu().long().clamp(min=0)
    ww, dd = wt.cpu().double(), d_wt.cpu().double()
    b = 0.01 * counts.cpu().double() * E / (k * int(n) ** 2)
    ref = torch.zeros(T, E, dtype=torch.float64).scatter_add_(1, i, ww * (dd - (ww * dd).sum(1, keepdim=True))) + p * (b - p @ b[:, None])
    ref = torch.where(mask.cpu()[:, None], ref, 0.0)
    assert ((d_logits.cpu().double() - ref).abs() <= 2.0 ** -16 * ((ww * dd).abs().sum(1, keepdim=True) + b.max())).all()

    d_buf = new(T * k, H)
    mx8.bwd_prologue(d_out, wt, d_buf)
    safe = torch.where(peer_rank >= 0, peer_tok, 0).long()
    d_y = torch.where((peer_rank >= 0)[:, None], d_buf[safe], torch.zeros((), dtype=torch.bfloat16, device=DEV))
    qd, sd, qdt, sdt = mx8.quantize_block128(d_y, True, True)
    d_hid = mx8.gemm_block128(qd, sd, *quant["down"][2:], new(cap, I), group_rows=per_expert)
    grouped(d_hid, qd, sd, *quant["down"][2:])
    d_down = mx8.gemm_block128_wgrad(qdt, sdt, qht, sht, torch.empty(E, H, I, device=DEV), per_expert)
    a64, b64, at = rows64(qdt, sdt), rows64(qht, sht), 0
    for e, m in enumerate(sizes):
        if m:
            check_c(d_down[e], a64[:, at:at + m], b64[:, at:at + m], f"expert {e} weights")
        else:
            assert (d_down[e] == 0).all()
        at += m
    assert mx8.device_status() == 0


@pytest.mark.parametrize("shape,b", [((2, 64, 256), "rows"), ((9, 3000, 2000), "rows"), ((100, 100, 256), "rows"), ((100, 100, 256), "square"), ((100, 100, 2048), "rows"),
                                     ((100, 100, 2048), "square"), ((1500, 1700, 256), "rows"), ((1500, 1700, 256), "square")])
def test_scales_whose_product_alone_is_in_range(shape, b):
    """one scale far above 1 and the other far below: their product is taken first in every form, so that no block's sum overflows or
    loses bits on the way.  Sums of 448 * 448 are exact in fp32 up to the 24 bits of 49 * K, and every block adds two roundings."""
    M, N, K = shape
    a = torch.full((M, 16 * ((K + 15) // 16)), 448.0, device=DEV).to(torch.float8_e4m3fn)[:, :K]
    w = torch.full((N, a.stride(0)), 448.0, device=DEV).to(torch.float8_e4m3fn)[:, :K]
    for sx, sy in ((1e-30, 1e33), (1e33, 1e-30), (1e37, 1e-37), (1e-37, 1e37), (1e-36, 1e2)):
        sa = torch.full((cdiv(K), M), sx, device=DEV)
        sb = torch.full((cdiv(K), N) if b == "rows" else (cdiv(N), cdiv(K)), sy, device=DEV)
        c = torch.empty(M, N, device=DEV)
        mx8.gemm_block128(a, sa, w, sb, c, b_blocks=b)
        want = K * 448.0 ** 2 * float(sa[0, 0].double() * sb[0, 0].double())
        assert ((c.double() / want - 1).abs() <= (2 * cdiv(K) + 1) * 2.0 ** -24).all(), (sx, sy)


def test_scales_whose_product_alone_is_in_range_in_weight_gradients():
    for M, N, R in ((100, 100, 256), (600, 1701, 1280)):
        a, w = (torch.full((rows, R), 448.0, device=DEV).to(torch.float8_e4m3fn) for rows in (M, N))
        grp = torch.tensor([128, 0, R - 128], dtype=torch.int32, device=DEV)
        for sx, sy in ((1e-30, 1e33), (1e33, 1e-30), (1e37, 1e-37)):
            sa, sb = torch.full((R // 128, M), sx, device=DEV), torch.full((R // 128, N), sy, device=DEV)
            c = torch.empty(3, M, N, device=DEV)
            mx8.gemm_block128_wgrad(a, sa, w, sb, c, grp)
            one = 448.0 ** 2 * float(sa[0, 0].double() * sb[0, 0].double())
            assert (c[1] == 0).all()
            for g, rows in ((0, 128), (2, R - 128)):
                assert ((c[g].double() / (rows * one) - 1).abs() <= (rows // 64 + 1) * 2.0 ** -24).all()


def test_sizes_that_do_not_fit_are_named_by_the_status():
    import ctypes
    lib = mx8.load()
    qa, sa, _, _ = mx8.quantize_block128(make_x(100, 256))
    qb, sb, _, _ = mx8.quantize_block128(make_x(3, 64, 256), square=True)
    bad = torch.tensor([50, 60, 10], dtype=torch.int32, device=DEV)
    for _ in range(2):                                             # reported once, then healthy again
        mx8.gemm_block128(qa, sa, qb, sb, torch.empty(100, 64, device=DEV), group_rows=bad)
        with pytest.raises(mx8.Mx8Error, match="group sizes do not fit") as e:
            mx8.device_status()
        assert e.value.word == 17 and "an input on the device did not fit" in str(e.value)
        assert mx8.device_status() == 0
    word = ctypes.c_int(0)
    mx8.gemm_block128(qa[:6], sa[:, :6], qb, sb, torch.empty(6, 64, device=DEV), group_rows=bad)       # single tokens
    assert lib.mx8_device_status(ctypes.byref(word), torch.cuda.current_stream().cuda_stream) == 6 and word.value == 17
    with pytest.raises(mx8.Mx8Error, match="does not fit its capacity") as e:
        mx8.schedule(torch.zeros(1, 300, 1, dtype=torch.int32, device=DEV), 1, 256, 0)
        mx8.device_status()
    assert e.value.word == 16


# ------------------------------------------------------------------------------------------------ C of large tiles
# More 128 x 64 tiles than twice the device's multiprocessors, which large tiles compute: shapes below are checked for it.
def needs_large_tiles(M, N, groups=0):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    small = cdiv(N) * (M // 64 + groups if groups else (M + 63) // 64)
    assert M > 64 and small > 2 * sms
    return M, N


def inside(rows, cols, dtype, before=(1, 3), after=(2, 4)):
    """a slice with guards on its four sides, rows off 16-byte boundaries; and the check that the guards are as they were"""
    store = torch.full((before[0] + rows + after[0], before[1] + cols + after[1]), 6.0, dtype=dtype, device=DEV)
    c = store[before[0]:before[0] + rows, before[1]:before[1] + cols]

    def untouched():
        c.fill_(6.0)
        return bool((store == 6.0).all())
    return c, untouched


@pytest.mark.parametrize("b", ["square", "rows"])
@pytest.mark.parametrize("shape", [(1500, 1700, 700), (1300, 2049, 260), (2050, 1153, 130)])
def test_product_on_large_tiles_stays_inside_a_slice(shape, b):
    M, N = needs_large_tiles(*shape[:2])
    qa, sa, qb, sb, a64, b64 = operands(*shape, b, seed=M)
    for dtype in (torch.bfloat16, torch.float32):
        for before, after in (((1, 3), (2, 4)), ((0, 8), (1, 8 - N % 8)), ((3, 2), (1, 2))):       # odd, 16-byte and 4-byte rows
            c, untouched = inside(M, N, dtype, before, after)
            mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks=b)
            assert mx8.device_status() == 0
            check_c(c, a64, b64, f"{shape} {b} {dtype} {before}")
            assert untouched()


@pytest.mark.parametrize("sizes", [[700, 3, 0, 129, 256, 128, 40], [1500, 1300]])
def test_grouped_product_on_large_tiles_stays_inside_a_slice(sizes):
    G, cap, K = len(sizes), sum(sizes) + 37, 272
    N = needs_large_tiles(cap, 2100, G)[1]
    qa, sa, _, _ = mx8.quantize_block128(make_x(cap, K, seed=cap))
    qb, sb, _, _ = mx8.quantize_block128(make_x(G, N, K, seed=G, dtype=torch.float32) * 0.02, square=True)
    for dtype in (torch.bfloat16, torch.float32):
        c, untouched = inside(cap, N, dtype)
        mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=torch.tensor(sizes, dtype=torch.int32, device=DEV))
        assert mx8.device_status() == 0
        a64, at = rows64(qa, sa), 0
        for g, n in enumerate(sizes):
            if n:
                check_c(c[at:at + n], a64[at:at + n], square64(qb[g], sb[g]), f"group {g}")
            at += n
        assert (c[at:] == 6.0).all() and untouched()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes,mn", [([1280, 0, 128, 1024], (600, 1701)), ([256] * 3, (1030, 1153))])
def test_weight_gradient_on_large_tiles_stays_inside_a_slice(sizes, mn, dtype):
    G, R, (M, N) = len(sizes), sum(sizes), mn
    needs_large_tiles(M * G, N)
    _, _, qa, sa = mx8.quantize_block128(make_x(R, M, seed=R, dtype=torch.float32), False, True)
    _, _, qb, sb = mx8.quantize_block128(make_x(R, N, seed=R + 1), False, True)
    flat, untouched = inside(G * M, N, dtype)
    c = flat.as_strided((G, M, N), (M * flat.stride(0), flat.stride(0), 1))
    mx8.gemm_block128_wgrad(qa, sa, qb, sb, c, torch.tensor(sizes, dtype=torch.int32, device=DEV))
    assert mx8.device_status() == 0
    a64, b64, at = rows64(qa, sa), rows64(qb, sb), 0
    for g, n in enumerate(sizes):
        if n:
            check_c(c[g], a64[:, at:at + n], b64[:, at:at + n], f"group {g}")
        else:
            assert (c[g] == 0).all()
        at += n
    assert untouched()


@pytest.mark.parametrize("b", ["square", "rows"])
def test_non_finite_scales_on_large_tiles_reach_their_rows_only(b):
    M, N = needs_large_tiles(1500, 1700)
    for bad in (float("nan"), float("inf")):
        qa, sa, qb, sb, a64, b64 = operands(M, N, 384, b, seed=4)
        sa[1, 7] = sa[2, 1499] = bad
        rows, cols = torch.arange(M), torch.arange(N)
        if b == "rows":
            sb[0, 1000] = bad
            gone = cols == 1000
        else:
            sb[13, 2] = bad                                        # columns 1664 to 1699
            gone = cols >= 1664
        hit = (rows == 7) | (rows == 1499)
        c = torch.empty(M, N, device=DEV)
        mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks=b)
        assert not torch.isfinite(c[hit.to(DEV)]).any() and not torch.isfinite(c[:, gone.to(DEV)]).any()
        check_c(c[(~hit).to(DEV)][:, (~gone).to(DEV)], a64[~hit], b64[~gone])


@pytest.mark.parametrize("form", ["square", "rows", "grouped"])
def test_large_tiles_beyond_32_bits(form):
    """C that spans more than 2^32 elements: every row where it should be, nothing between"""
    M, N, K = 65 if form != "grouped" else 130, 19100, 260
    needs_large_tiles(M, N, 2 if form == "grouped" else 0)
    pitch = 2 ** 32 // (M - 1) + 7
    b = "rows" if form == "rows" else "square"
    if form == "grouped":
        qa, sa, _, _ = mx8.quantize_block128(make_x(M, K, seed=3))
        qb, sb, _, _ = mx8.quantize_block128(make_x(2, N, K, seed=5, dtype=torch.float32) * 0.02, square=True)
    else:
        qa, sa, qb, sb, a64, b64 = operands(M, N, K, b, seed=M)
    store = torch.full((M * pitch,), 2.0, dtype=torch.bfloat16, device=DEV)
    c = store.as_strided((M, N), (pitch, 1))
    if form == "grouped":
        mx8.gemm_block128(qa, sa, qb, sb, c, group_rows=torch.tensor([40, 90], dtype=torch.int32, device=DEV))
        a64 = rows64(qa, sa)
        check_c(c[:40], a64[:40], square64(qb[0], sb[0]))
        check_c(c[40:], a64[40:], square64(qb[1], sb[1]))
    else:
        mx8.gemm_block128(qa, sa, qb, sb, c, b_blocks=b)
        check_c(c, a64, b64)
    assert mx8.device_status() == 0
    c.fill_(2.0)
    assert all(bool((part == 2.0).all()) for part in store.split(2 ** 28))


def test_weight_gradients_beyond_32_bits():
    """more than 2^32 elements of C over the groups' matrices, most of them between the rows"""
    M, N, G = 300, 2200, 4
    needs_large_tiles(M * G, N)
    pitch = 2 ** 32 // (M * G - 1) + 5
    _, _, qa, sa = mx8.quantize_block128(make_x(128 * G, M, seed=1, dtype=torch.float32), False, True)
    _, _, qb, sb = mx8.quantize_block128(make_x(128 * G, N, seed=2), False, True)
    store = torch.full((M * G * pitch,), 2.0, dtype=torch.bfloat16, device=DEV)
    c = store.as_strided((G, M, N), (M * pitch, pitch, 1))
    mx8.gemm_block128_wgrad(qa, sa, qb, sb, c, torch.full((G,), 128, dtype=torch.int32, device=DEV))
    assert mx8.device_status() == 0
    a64, b64 = rows64(qa, sa), rows64(qb, sb)
    for g in range(G):
        check_c(c[g], a64[:, 128 * g:128 * g + 128], b64[:, 128 * g:128 * g + 128], f"group {g}")
    c.fill_(2.0)
    assert all(bool((part == 2.0).all()) for part in store.split(2 ** 28))
