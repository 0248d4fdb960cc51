"""Router, balance loss, their gradient and the gradient of the routing weights against plain 64-bit forms."""
import pytest
import torch

import mx8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NEG = float("-inf")
# relative error of a softmax value: the difference l - max is rounded (half a step of |l - max| < 32 is 2^-20 absolute in the
# exponent), exp is good to two steps of 2^-23, a sum of 1024 terms in fp32 to 10 * 2^-24 (tree over 32 lanes of 32), one division:
# 2^-20 + 2^-22 + 2^-20.6 + 2^-24 < 2^-18.5 for numerator and denominator together
P_TOL = 2.0 ** -18


def route_ref(logits, k, normalize, mask=None):
    """64-bit forward on the CPU"""
    l = logits.detach().cpu().double()
    T, E = l.shape
    on = (l > NEG).any(1) | torch.isnan(l).any(1)
    if mask is not None:
        on &= mask.cpu()
    order = torch.sort(torch.where(torch.isnan(l), torch.inf, l), dim=1, descending=True, stable=True).indices[:, :k]
    taken = (torch.gather(l, 1, order) != NEG) & on[:, None]
    idx = torch.where(taken, order, -1)
    p = torch.where(on[:, None], torch.softmax(l, 1), 0.0)
    w = torch.where(taken, torch.gather(p, 1, order), 0.0)
    if normalize:
        w = torch.where(taken, w / w.sum(1, keepdim=True), 0.0)
    counts = torch.zeros(E, dtype=torch.int64).scatter_add_(0, idx[taken], torch.ones_like(idx[taken]))
    n = int(on.sum())
    loss = float((counts.double() * p.sum(0)).sum() * E / (k * n * n)) if n else 0.0
    lse = torch.where(on, torch.logsumexp(l, 1), NEG)
    return idx, w, lse, counts, p.sum(0), n, loss


def check_forward(logits, k, normalize, mask=None):
    out = mx8.router_topk(logits, k, normalize=normalize, token_mask=mask)
    assert mx8.device_status() == 0
    idx, w, lse, counts, prob, n, loss = [t.cpu() for t in out]
    ridx, rw, rlse, rcounts, rprob, rn, rloss = route_ref(logits, k, normalize, mask)
    assert idx.dtype == torch.int32 and torch.equal(idx.long(), ridx)
    assert torch.equal(counts.long(), rcounts) and int(n) == rn
    assert torch.allclose(w.double(), rw, rtol=P_TOL, atol=2.0 ** -140)
    live = rlse > NEG
    assert torch.equal(lse == NEG, ~live)
    # the logarithm adds half a step of its own and of the maximum it is added to
    assert ((lse[live].double() - rlse[live]).abs() <= 2.0 ** -18 + 2.0 ** -23 * rlse[live].abs()).all()
    # sums over tokens: fp32 per warp and block (at most 2^13 terms in a row, here far fewer), then 64 bits
    tokens = max(1, logits.shape[0] // 2000 + 40)
    assert torch.allclose(prob.double(), rprob, rtol=P_TOL + tokens * 2.0 ** -24, atol=2.0 ** -120)
    assert abs(float(loss) - rloss) <= (P_TOL + tokens * 2.0 ** -24) * abs(rloss)
    return out


def make_logits(T, E, dtype, seed, ties=False):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(T, E, generator=g)
    if ties:
        l = torch.round(l * 2) / 2
    return l.to(dtype).to(DEV)


SHAPES = [(1, 1, 1), (1, 8, 8), (3, 60, 4), (16, 256, 8), (64, 256, 8), (65, 256, 8), (1000, 257, 6), (5003, 64, 2), (129, 1024, 32),
          (70, 512, 1), (7, 33, 32), (2000, 128, 6), (33, 1000, 5), (300, 4, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    T, E, k = shape
    for normalize in (True, False):
        check_forward(make_logits(T, E, dtype, T + E), k, normalize)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lower_expert(dtype):
    check_forward(make_logits(200, 96, dtype, 1, ties=True), 8, True)
    flat = torch.zeros(9, 256, dtype=dtype, device=DEV)
    flat[3, ::2] = -0.0                                       # both zeros are the same value
    check_forward(flat, 8, True)


@pytest.mark.parametrize("shape", [(70, 512, 8), (33, 1000, 5), (40, 64, 6), (10, 8, 8), (5, 130, 32), (200, 33, 1)])
def test_close_float32_values_are_told_apart(shape):
    """logits of a few last bits' difference, many equal, some experts off: the order is that of the full values, ties to the lower expert"""
    T, E, k = shape
    g = torch.Generator().manual_seed(T)
    l = 1.0 + torch.randint(0, 40, (T, E), generator=g).float() * 2.0 ** -23
    l = torch.where(torch.rand(T, E, generator=g) < 0.1, -l, l)
    l = torch.where(torch.rand(T, E, generator=g) < 0.2, float("-inf"), l)
    idx = mx8.router_topk(l.to(DEV), k)[0].cpu()
    order = torch.sort(l, dim=1, descending=True, stable=True)
    want = torch.where(order.values[:, :k] == float("-inf"), -1, order.indices[:, :k]).to(torch.int32)
    assert torch.equal(idx, want)


def test_masks_switched_off_experts_and_lowest_values():
    l = make_logits(200, 64, torch.float32, 2)
    l[5] = NEG                                                 # nothing left
    l[6, 1:] = NEG                                             # fewer than topk
    l[7, 10:] = torch.finfo(torch.float32).min                 # a mask of the type's lowest value is a value
    l[8] = torch.finfo(torch.float32).min
    l[:, 11] = NEG
    mask = torch.ones(200, dtype=torch.bool, device=DEV)
    mask[150:] = False
    mask[0] = False
    for normalize in (True, False):
        check_forward(l, 12, normalize, mask)
    b = l.to(torch.bfloat16)
    b[7, 10:] = torch.finfo(torch.bfloat16).min
    check_forward(b, 4, True, mask)
    # a batch in which no token takes part
    out = mx8.router_topk(l, 4, token_mask=torch.zeros(200, dtype=torch.bool, device=DEV))
    assert int(out[5]) == 0 and float(out[6]) == 0.0 and int(out[3].abs().sum()) == 0 and float(out[4].abs().sum()) == 0.0
    assert (out[0] == -1).all() and (out[1] == 0).all() and (out[2] == NEG).all()


def test_values_in_masked_tokens_are_not_read_and_live_nan_is_reported():
    l = make_logits(100, 48, torch.float32, 3)
    want = mx8.router_topk(l[:60].contiguous(), 4)
    mask = torch.arange(100, device=DEV) < 60
    l[60:] = float("nan")
    l[70, 3] = float("inf")
    got = mx8.router_topk(l, 4, token_mask=mask)
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a[:60], b)
    assert torch.equal(got[3], want[3]) and torch.isfinite(got[4]).all() and torch.isfinite(got[6]).all()
    # a NaN or an infinity in a live token: first choice, NaN weights, NaN loss, ids inside the range
    for bad in (float("nan"), float("inf")):
        x = make_logits(10, 48, torch.float32, 4)
        x[2, 17] = bad
        idx, w, lse, counts, prob, n, loss = mx8.router_topk(x, 4)
        assert int(idx[2, 0]) == 17 and bool(((idx >= 0) & (idx < 48)).all()) and int(counts.sum()) == 40
        assert torch.isnan(w[2]).all() and torch.isnan(loss).all() and torch.isfinite(w[3]).all()


def test_strided_rows_and_offsets():
    for dtype in (torch.float32, torch.bfloat16):
        wide = make_logits(130, 300, dtype, 5)
        for sl in (wide[:, :256], wide[:, 3:259], wide[:, 1:61], wide[::2, 8:264]):
            got = mx8.router_topk(sl, 6)
            want = mx8.router_topk(sl.contiguous(), 6)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            d = torch.randn(sl.shape[0], 6, device=DEV)
            one = torch.ones(1, device=DEV)
            args = (got[0], got[1], got[2], got[3], got[5], d, one)
            assert torch.equal(mx8.router_topk_bwd(sl, *args), mx8.router_topk_bwd(sl.contiguous(), *args))


def bwd_ref(logits, idx, normalize, counts, n, k, dw, dl):
    """64-bit gradient by automatic differentiation of the forward formula with the choices and counts held"""
    l = logits.detach().cpu().double().requires_grad_(True)
    T, E = l.shape
    on = (l.detach() > NEG).any(1) & (idx >= 0).any(1)
    safe = torch.where(on[:, None], l, torch.zeros_like(l))
    p = torch.softmax(safe, 1) * on[:, None]
    taken = idx >= 0
    w = torch.where(taken, torch.gather(p, 1, idx.clamp(min=0)), 0.0)
    if normalize:
        w = torch.where(taken, w / torch.where(on, w.sum(1), 1.0)[:, None], 0.0)
    total = torch.zeros((), dtype=torch.float64)
    if dw is not None:
        total = total + (w * torch.where(taken, dw.cpu().double(), 0.0)).sum()
    if dl is not None:
        total = total + float(dl) * (counts.double() * p.sum(0)).sum() * E / (k * max(n, 1) ** 2)
    total.backward()
    g = l.grad
    # size of the terms that cancel: the bound of the rounding error
    size = (w.detach().abs() * (dw.cpu().double().nan_to_num().abs() if dw is not None else 0.0)).sum(1, keepdim=True)
    if dl is not None:
        size = size + abs(float(dl)) * counts.double().max() * E / (k * max(n, 1) ** 2)
    return torch.nan_to_num(g), size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, dtype):
    T, E, k = shape
    logits = make_logits(T, E, dtype, 7 * T + E)
    mask = torch.arange(T, device=DEV) < max(1, T - T // 5)
    if E > 4 and T > 3:
        logits[:, 2] = NEG
        logits[1] = NEG
    g = torch.Generator().manual_seed(T)
    dw = torch.randn(T, k, generator=g).to(DEV)
    dl = torch.tensor([3.0], device=DEV)
    for normalize in (True, False):
        idx, w, lse, counts, _, n, _ = mx8.router_topk(logits, k, normalize=normalize, token_mask=mask)
        dw_in = torch.where(idx >= 0, dw, float("nan"))                  # what lies at unfilled choices is not read
        for a, b in ((dw_in, dl), (dw_in, None), (None, dl)):
            got = mx8.router_topk_bwd(logits, idx, w, lse, counts, n, a, b, normalize=normalize)
            assert mx8.device_status() == 0 and got.dtype == dtype and got.shape == (T, E)
            want, size = bwd_ref(logits, idx.cpu().long(), normalize, counts.cpu(), int(n), k, a, b)
            # p, w and the two sums are good to P_TOL of `size`; bf16 rounds the result by half a step of 2^-7
            tol = 4 * P_TOL * size + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0.0) + 2.0 ** -120
            assert ((got.cpu().double() - want).abs() <= tol).all()
            assert (got.cpu()[~mask.cpu()] == 0).all()


def test_backward_against_differences_of_the_forward():
    # S = sum w dw + dl * loss; central differences of the kernel's own forward.  Logits are multiples of 1/4 apart, so a step of 2^-6
    # changes no choice; |third derivative| of softmax terms is below 1 per unit of dw, so the truncation is below 2^-12 / 6 * sum|dw|,
    # and the rounding of S (2^-18 relative) divided by 2 h = 2^-5 below 2^-13 * |S|
    T, E, k, h = 3, 8, 3, 2.0 ** -6
    g = torch.Generator().manual_seed(1)
    base = torch.stack([torch.randperm(E, generator=g) for _ in range(T)]).float() / 4
    dw, dl = torch.randn(T, k, generator=g), 0.7
    for normalize in (True, False):
        def value(l):
            o = mx8.router_topk(l.to(DEV), k, normalize=normalize)
            return float((o[1].cpu().double() * dw.double()).sum() + dl * o[6].cpu().double())
        o = mx8.router_topk(base.to(DEV), k, normalize=normalize)
        got = mx8.router_topk_bwd(base.to(DEV), o[0], o[1], o[2], o[3], o[5], dw.to(DEV), torch.tensor([dl], device=DEV), normalize=normalize).cpu()
        tol = 2.0 ** -12 / 6 * float(dw.abs().sum() + 8 * dl) + 2.0 ** -13 * float(dw.abs().sum() + dl * 4)
        for t in range(T):
            for e in range(E):
                hi, lo = base.clone(), base.clone()
                hi[t, e] += h
                lo[t, e] -= h
                assert abs((value(hi) - value(lo)) / (2 * h) - float(got[t, e])) <= tol


def test_counts_summed_over_ranks_give_the_gradient_of_the_joint_loss():
    T, E, k = 120, 32, 4
    l = make_logits(T, E, torch.float32, 9)
    whole = mx8.router_topk(l, k)
    parts = [mx8.router_topk(x, k) for x in (l[:50].contiguous(), l[50:].contiguous())]
    counts, n = parts[0][3] + parts[1][3], parts[0][5] + parts[1][5]
    assert torch.equal(counts, whole[3]) and int(n) == T
    one = torch.ones(1, device=DEV)
    want = mx8.router_topk_bwd(l, whole[0], whole[1], whole[2], whole[3], whole[5], None, one)
    got = torch.cat([mx8.router_topk_bwd(x.contiguous(), o[0], o[1], o[2], counts, n, None, one) for x, o in zip((l[:50], l[50:]), parts)])
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(1, 1, 8), (3, 8, 128), (61, 8, 2048), (17, 9, 1032), (5, 3, 77), (2, 32, 4096), (130, 2, 7168)])
def test_bwd_topk_weights(shape):
    T, k, H = shape
    g = torch.Generator().manual_seed(T * k + H)
    d = torch.randn(T, H, generator=g).to(torch.bfloat16)
    c = torch.randn(T * k, H, generator=g).to(torch.bfloat16)
    got = mx8.bwd_topk_weights(d.to(DEV), c.to(DEV)).cpu().double()
    terms = c.double().view(T, k, H) * d.double().view(T, 1, H)
    # H products in fp32 with fused adds, at most H/256 + 8 + 7 of them in a chain per thread, lanes and warps
    tol = (H / 128 + 16) * 2.0 ** -24 * terms.abs().sum(2)
    assert ((got - terms.sum(2)).abs() <= tol).all()
    idx = torch.randint(-1, 4, (T, k), generator=g, dtype=torch.int32)
    c2 = c.clone()
    c2[(idx < 0).reshape(-1)] = float("nan")                       # rows that no expert sent
    part = mx8.bwd_topk_weights(d.to(DEV), c2.to(DEV), idx.to(DEV)).cpu().double()
    assert torch.equal(part, torch.where(idx >= 0, got, 0.0))


def test_refusals():
    l = make_logits(8, 16, torch.float32, 0)
    o = mx8.router_topk(l, 2)
    for bad in (lambda: mx8.router_topk(l, 17), lambda: mx8.router_topk(l, 0)):
        with pytest.raises(mx8.Mx8Error):
            bad()
    dw, dl = torch.zeros(8, 2, device=DEV), torch.zeros(1, device=DEV)
    for bad in (lambda: mx8.router_topk(l.half(), 2), lambda: mx8.router_topk(l.t(), 2), lambda: mx8.router_topk(l[:0], 2),
                lambda: mx8.router_topk(l, 2, token_mask=torch.ones(7, dtype=torch.bool, device=DEV)),
                lambda: mx8.router_topk(l, 2, token_mask=torch.ones(8, dtype=torch.int32, device=DEV)),
                lambda: mx8.router_topk(l, 2, token_mask=torch.ones(8, dtype=torch.bool)),
                lambda: mx8.router_topk_bwd(l, o[0], o[1], o[2], o[3], o[5]),
                lambda: mx8.router_topk_bwd(l, o[0], o[1], o[2], o[3], o[5], dw[:4], dl),
                lambda: mx8.router_topk_bwd(l, o[0].long(), o[1], o[2], o[3], o[5], dw, dl),
                lambda: mx8.router_topk_bwd(l, o[0], o[1], o[2], o[3][:8], o[5], dw, dl),
                lambda: mx8.bwd_topk_weights(torch.zeros(3, 8, dtype=torch.bfloat16, device=DEV), torch.zeros(7, 8, dtype=torch.bfloat16, device=DEV)),
                lambda: mx8.bwd_topk_weights(torch.zeros(3, 8, device=DEV), torch.zeros(6, 8, device=DEV))):
        with pytest.raises(ValueError):
            bad()


def test_repeatable_on_a_side_stream_and_in_a_graph():
    l = make_logits(4097, 256, torch.bfloat16, 12)
    want = mx8.router_topk(l, 8)
    dw, dl = torch.randn(4097, 8, device=DEV), torch.ones(1, device=DEV)
    want_d = mx8.router_topk_bwd(l, want[0], want[1], want[2], want[3], want[5], dw, dl)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = mx8.router_topk(l, 8)
        got_d = mx8.router_topk_bwd(l, got[0], got[1], got[2], got[3], got[5], dw, dl)
    s.synchronize()
    for a, b in zip(got + (got_d,), want + (want_d,)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    src = torch.zeros_like(l)
    with torch.cuda.graph(graph):
        out = mx8.router_topk(src, 8)
        out_d = mx8.router_topk_bwd(src, out[0], out[1], out[2], out[3], out[5], dw, dl)
    src.copy_(l)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out + (out_d,), want + (want_d,)):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """logits, and rows of the routing weights' gradient, that span more than 2^32 elements"""
    T, E = 130, 40
    pitch = 2 ** 32 // T + 5
    l = torch.zeros(T * pitch, dtype=torch.bfloat16, device=DEV).as_strided((T, E), (pitch, 1))
    l.copy_(make_logits(T, E, torch.bfloat16, 33))
    dense = l.contiguous()
    want, got = mx8.router_topk(dense, 4), mx8.router_topk(l, 4)
    dw = torch.randn(T, 4, device=DEV)
    for a, b in zip(want + (mx8.router_topk_bwd(dense, want[0], want[1], want[2], want[3], want[5], dw),),
                    got + (mx8.router_topk_bwd(l, got[0], got[1], got[2], got[3], got[5], dw),)):
        assert torch.equal(a, b)
    del l
    T, H, k = 5, 2 ** 17 + 8, 6554                                 # T k H > 2^32
    d = torch.ones(T, H, dtype=torch.bfloat16, device=DEV)
    c = torch.zeros(T * k, H, dtype=torch.bfloat16, device=DEV)
    c[-1, -1] = 3.0
    c[-k, 0] = 5.0
    want = torch.zeros(T, k)
    want[-1, -1], want[-1, 0] = 3.0, 5.0
    assert torch.equal(mx8.bwd_topk_weights(d, c).cpu(), want)


@pytest.mark.parametrize("E", [1, 33, 256, 257, 1000])
def test_balance_loss_of_many_launches_in_a_row(E):
    """the finishing kernel's blocks start at any time beside the forward kernels of a full stream: the loss is that of the returned sums"""
    k = min(E, 5)
    l = make_logits(700, E, torch.float32, E)
    outs = [mx8.router_topk(l + float(i), k) for i in range(200)]
    torch.cuda.synchronize()
    for _, _, _, counts, prob, n, loss in outs:
        want = float((counts.double() * prob.double()).sum()) * E / (k * 700.0 ** 2)
        # prob_sum and the loss are rounded to fp32, half a step each
        assert int(n) == 700 and int(counts.sum()) == 700 * k and abs(float(loss) - want) <= 2.0 ** -23 * want


@pytest.mark.parametrize("H,k", [(8, 1), (264, 3), (1024, 8)])
def test_rows_of_choices_without_an_expert_do_not_reach_the_output(H, k):
    """combine leaves the rows of ids -1 as they were: NaN, infinities or an earlier step's values there change nothing, a NaN of a
    live choice stays one"""
    T, E = 40, 16
    l = make_logits(T, E, torch.float32, H)
    l[3, 1:] = NEG                                                 # one live expert
    mask = torch.arange(T, device=DEV) < 35
    idx, w, _, _, _, _, _ = mx8.router_topk(l, k, token_mask=mask)
    g = torch.Generator().manual_seed(k)
    buf = torch.randn(T * k, H, generator=g).to(torch.bfloat16).to(DEV)
    y = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    dead = (idx < 0).reshape(-1)
    assert int(dead.sum()) == 5 * k + k - 1
    clean = buf.masked_fill(dead[:, None], 0.0)
    for shared in (y, None):
        want = mx8.fwd_epilogue(shared, clean, w)
        for bad in (float("nan"), float("inf"), float("-inf"), 3e38):
            assert torch.equal(mx8.fwd_epilogue(shared, buf.masked_fill(dead[:, None], bad), w), want)
    assert torch.equal(want[35:], torch.zeros_like(want[35:]))
    live = clean.clone()
    live[0, 0] = float("nan")
    out = mx8.fwd_epilogue(None, live, w)
    assert torch.isnan(out[0, 0]) and int(torch.isnan(out).sum()) == 1
    # a finite row times 0 keeps the zero's sign, as before
    one = torch.full((1, 8), -1.0, dtype=torch.bfloat16, device=DEV)
    zero = torch.full((1, 8), -0.0, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(mx8.fwd_epilogue(zero, one, torch.zeros(1, 1, device=DEV)).view(torch.int16), zero.view(torch.int16))


def test_gradients_of_choices_without_an_expert_are_not_summed():
    """the backward's combine leaves the rows of ids -1 as they were; the sum over a token's rows skips them when it has the ids"""
    T, E, H, k = 40, 16, 264, 3
    l = make_logits(T, E, torch.float32, 1)
    l[3, 1:] = NEG
    idx = mx8.router_topk(l, k, token_mask=torch.arange(T, device=DEV) < 35)[0]
    g = torch.Generator().manual_seed(k)
    shared = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    buf = torch.randn(T * k, H, generator=g).to(torch.bfloat16).to(DEV)        # an earlier step's values in the dead rows
    dead = (idx < 0).reshape(-1, 1)
    clean = buf.masked_fill(dead, 0.0)
    want = mx8.bwd_epilogue(shared, clean)
    terms = torch.cat([shared[:, None], clean.view(T, k, H)], 1).double()
    # k + 1 terms added in fp32, then half a step of bf16
    assert ((want.double() - terms.sum(1)).abs() <= 2.0 ** -8 * terms.sum(1).abs() + 2.0 ** -22 * terms.abs().sum(1)).all()
    assert not torch.equal(mx8.bwd_epilogue(shared, buf), want)
    from mx8 import _C
    for held in (buf, buf.masked_fill(dead, float("nan"))):
        assert torch.equal(mx8.bwd_epilogue(shared, held, idx), want)
        assert torch.equal(_C.bwd_epilogue(shared, held, idx), want)
        assert torch.equal(mx8.bwd_epilogue_routed(None, held, k, idx), mx8.bwd_epilogue_routed(None, clean, k))
    for bad in (idx.long(), idx[:5].contiguous(), idx.cpu()):
        with pytest.raises(ValueError):
            mx8.bwd_epilogue(shared, buf, bad)
        with pytest.raises(RuntimeError):
            _C.bwd_epilogue(shared, buf, bad)


def test_calls_of_different_widths_in_threads():
    """host threads through the C ABI, which holds no lock of Python's: all of 513 to 1024 experts share a kernel and its limits"""
    import threading
    lib, failed = mx8.load(), []
    widths = (1024, 520, 1000, 700)
    held = {E: (make_logits(4, E, torch.float32, E), make_logits(4, E, torch.bfloat16, E)) for E in widths}
    barrier = threading.Barrier(len(widths))
    got = {}

    def worker(E):
        s = torch.cuda.Stream()
        out = [torch.empty(4, 8, dtype=torch.int32, device=DEV), torch.empty(4, 8, device=DEV), torch.empty(4, device=DEV),
               torch.empty(E, dtype=torch.int32, device=DEV), torch.empty(E, device=DEV), torch.empty(1, dtype=torch.int32, device=DEV), torch.empty(1, device=DEV)]
        ptrs = [t.data_ptr() for t in out]
        barrier.wait()
        for i in range(20000):
            rc = lib.mx8_router_topk(held[E][i & 1].data_ptr(), 1 - (i & 1), E, 4, E, 8, 1, None, *ptrs, None, 0, s.cuda_stream)
            if rc:
                failed.append((E, i, rc, lib.mx8_last_cuda_error()))
                break
        s.synchronize()
        got[E] = out

    torch.cuda.synchronize()
    threads = [threading.Thread(target=worker, args=(E,)) for E in widths]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for E in widths:
        for a, b in zip(got[E], mx8.router_topk(held[E][1], 8)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [3, 2000])
def test_outputs_can_be_saved_together(T):
    """in calls whose outputs share allocations and in those where they do not; what is saved is what was there"""
    import io
    import itertools
    l = make_logits(T, 64, torch.float32, T)
    out = mx8.router_topk(l, 4)
    for group in list(itertools.combinations(out, 2)) + [out]:
        f = io.BytesIO()
        torch.save(list(group), f)
        f.seek(0)
        for a, b in zip(torch.load(f), group):
            assert a.dtype == b.dtype and torch.equal(a, b)
    # no two of them overlap, and each starts on a 512-byte boundary
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in out)
    assert all(a % 512 == 0 for a, _ in spans) and all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_give_correctly_rounded_values(dtype):
    """exp(0) is 1 and E ones add up exactly, so that a weight is one division, rounded once, and lse the logarithm of an integer (logf: one
    step of 2^-23 of its binade)"""
    for E in [*range(1, 40), *range(41, 1024, 17), 1023, 1024]:
        k = min(E, 1 + E % 32)
        flat = torch.zeros(2, E, dtype=dtype, device=DEV)
        for normalize, n in ((True, k), (False, E)):
            out = mx8.router_topk(flat, k, normalize=normalize)
            assert (out[1].cpu() == torch.full((2, k), 1.0 / n, dtype=torch.float64).float()).all(), (E, k, normalize)
        want = torch.tensor(float(E), dtype=torch.float64).log()
        step = 2.0 ** (float(want.log2().floor()) - 23) if E > 1 else 0.0
        assert ((out[2].cpu().double() - want).abs() <= step).all(), E


@pytest.mark.parametrize("shift", [0.0, 1000.0, -1000.0, 30000.0])
@pytest.mark.parametrize("shape", [(300, 64, 4), (40, 1000, 8), (7, 5, 2), (100, 256, 8)])
def test_backward_of_shifted_logits(shape, shift):
    """the rounding of a large lse does not reach the gradient: it is that of 64 bits, and a token's gradients add up to nothing"""
    T, E, k = shape
    logits = make_logits(T, E, torch.float32, T) + shift                       # the rounded sums are the logits of both sides
    g = torch.Generator().manual_seed(E)
    dw, dl = torch.randn(T, k, generator=g).to(DEV), torch.tensor([3.0], device=DEV)
    for normalize in (True, False):
        idx, w, lse, counts, _, n, _ = mx8.router_topk(logits, k, normalize=normalize)
        got = mx8.router_topk_bwd(logits, idx, w, lse, counts, n, dw, dl, normalize=normalize).cpu().double()
        want, size = bwd_ref(logits, idx.cpu().long(), normalize, counts.cpu(), int(n), k, dw, dl)
        assert ((got - want).abs() <= 4 * P_TOL * size + 2.0 ** -120).all()
        # the sum that is subtracted is off by its E / 32 + 5 additions and two products, every gradient by three roundings, 1 / sum by one,
        # all of 2^-24 and of terms that add up to at most twice `size`
        assert (got.sum(1, keepdim=True).abs() <= (E / 32 + 16) * 2.0 ** -23 * size).all()


def test_mxfp8_layer_of_masked_tokens_needs_no_cleared_buffers():
    """router, schedule, the MXFP8 layer forward and backward and both weighted sums on one rank: with buffers that held NaN or an earlier
    step's values the outputs are those of cleared ones"""
    from oracle import mx8_oracle as O
    T, H, I, k, E = 256, 512, 256, 4, 6
    g = torch.Generator().manual_seed(3)
    l = torch.randn(T, E, generator=g)
    l[5, 1:] = NEG
    idx, w, _, counts, _, n, _ = mx8.router_topk(l.to(DEV), k, token_mask=torch.arange(T, device=DEV) < T - 30)
    assert int(n) == T - 30 and int(counts.sum()) == (T - 30) * k - (k - 1)
    cap = (T * k // 256 + E) * 256
    make = lambda r, c, seed: torch.stack([O.make_input(r, c, seed=seed + e, std=c ** -0.5) for e in range(E)])  # noqa: E731
    ws = [make(I, H, 100), make(I, H, 200), make(H, I, 300)]
    fw = [tuple(t.to(DEV) for t in O.quantize_both(m)[:2]) for m in ws]
    bw = [tuple(t.to(DEV) for t in O.quantize_both(m.transpose(1, 2).contiguous())[:2]) for m in ws]
    x, d_out = O.make_input(T, H, seed=72).to(DEV), O.make_input(T, H, seed=73, std=H ** -0.5).to(DEV)
    pr, pt, nt, tpe = mx8.schedule(idx[None].contiguous(), E, cap, 0)
    assert int((pr >= 0).sum()) == int(counts.sum())

    def step(fill, ids):
        cb, d_xb = (torch.full((T * k, H), fill, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        f = mx8.dispatch_mlp_swiglu_combine_fwd(x, [x.data_ptr()], cb, [cb.data_ptr()], None, *fw[0], None, *fw[1], None, *fw[2], pr, pt, nt, tpe, k)
        out = mx8.fwd_epilogue(None, cb, w)
        d_cb = torch.full_like(cb, fill)
        mx8.bwd_prologue(d_out, w, d_cb)
        mx8.dispatch_mlp_swiglu_combine_bwd(None, d_cb, [d_cb.data_ptr()], d_xb, [d_xb.data_ptr()], None, *bw[0], None, *bw[1], None, *bw[2],
                                            f[0], f[1], None, f[3], f[4], None, f[6], f[7], None, f[9], f[10], x, [x.data_ptr()], *fw[0], *fw[1],
                                            pr, pt, nt, tpe, k)
        res = out, mx8.bwd_epilogue_routed(None, d_xb, k, ids), mx8.bwd_topk_weights(d_out, cb, idx)
        assert mx8.device_status() == 0
        return res
    want = step(0.0, None)
    assert float(want[0].abs().sum()) > 0 and (want[0][T - 30:] == 0).all() and (want[1][T - 30:] == 0).all()
    for fill in (0.0, 3.0, float("nan"), float("inf")):
        for got, ref in zip(step(fill, idx), want):
            assert torch.equal(got, ref)


def test_outputs_are_ordinary_tensors():
    """views of a shared allocation: autograd, in-place changes, copies and other streams treat them as any other"""
    import copy
    l = make_logits(9, 40, torch.float32, 2)
    out = mx8.router_topk(l, 3)
    held = [t.clone() for t in out]
    w = out[1].requires_grad_(True)
    (w * 2).sum().backward()
    assert torch.equal(w.grad, torch.full_like(w, 2.0))
    assert torch.equal(copy.deepcopy(out[3]), held[3])
    out[3].zero_()
    out[4].add_(1.0)
    out[2].record_stream(torch.cuda.Stream())
    for i in (0, 1, 2, 5, 6):
        assert torch.equal(out[i], held[i])
    assert (out[3] == 0).all() and torch.equal(out[4], held[4] + 1.0)
    with pytest.raises(RuntimeError):                              # a saved tensor that was changed is noticed
        v = out[2].requires_grad_(True)
        y = v * v.detach()
        z = (y.exp(), y)
        z[0].mul_(2.0)
        z[0].sum().backward()
