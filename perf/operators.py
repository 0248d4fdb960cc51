"""Measured cases of the router, its gradients and the 8-bit products with one scale per block of 128.

Operators (public names in the mx8 module):
  router_topk / router_topk_bwd   softmax, top-k, per-expert counts and balance loss of a router, and their gradient
  bwd_topk_weights                gradient of the routing weights: one dot product per (token, choice)
  quantize_block128               E4M3 with an fp32 scale per 1 x 128 row block, 128 x 1 column block or 128 x 128 square
  gemm_block128[_wgrad]           the matrix product on those operands: dense, grouped by expert, weight gradient per expert

With `own` false `run` computes the plain form (elementary torch operations in 32 bits or more); with `own` true it makes the calls
a user makes.  Scales of row blocks are stored K-block major: sc[kb][row]; squares as sc[row block][kb].
"""
import os
import sys

import torch

own = False

DEV = "cuda"
BLK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -110          # blocks below it are quantized with the scale of a block whose largest value it is


def _mx8():
    mod = sys.modules.get("mx8")
    if mod is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-experiments_b200"))
        import mx8 as mod
    return mod


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a small batch: 16 tokens through the 256-expert router, where only launches count
        {"name": "route_decode", "op": "route", "T": 16, "E": 256, "k": 8, "dtype": "float32", "norm": True, "pad": 0, "off": 0},
        # the router of the MoE benchmark (32768 tokens, 256 experts, top-8) as a training step runs it, with padded tokens
        {"name": "route_train", "op": "route_step", "T": 32768, "E": 256, "k": 8, "dtype": "bfloat16", "norm": True, "pad": 700, "off": 0},
        # a router of odd width with unnormalised weights and switched-off experts: backward alone
        {"name": "route_bwd_odd", "op": "route_bwd", "T": 5003, "E": 60, "k": 4, "dtype": "float32", "norm": False, "pad": 3, "off": 2},
        # gradient of the routing weights: a small batch, and one rank's share of the benchmark's tokens
        {"name": "weights_grad_small", "op": "weights_grad", "T": 61, "k": 8, "H": 2048},
        {"name": "weights_grad_train", "op": "weights_grad", "T": 8192, "k": 8, "H": 7168},
        # routed rows gathered from the tokens and quantized for the forward and the weight gradient
        {"name": "quantize_dispatch", "op": "quantize", "E": 1, "M": 16391, "N": 7168, "dtype": "bfloat16", "both": True, "square": False, "gather": True},
        # experts' fp32 master weights cut into squares, with the transpose for the data gradient
        {"name": "quantize_weights", "op": "quantize", "E": 4, "M": 2048, "N": 7168, "dtype": "float32", "both": True, "square": True, "gather": False},
        # one token through one projection: bound by reading the weights
        {"name": "linear_token", "op": "gemm", "M": 1, "N": 7168, "K": 2048, "out": "bfloat16", "b": "square"},
        # a prompt of odd length, contraction not a multiple of the block
        {"name": "linear_prompt", "op": "gemm", "M": 1003, "N": 4096, "K": 7120, "out": "bfloat16", "b": "square"},
        # the GEMM benchmark's size
        {"name": "linear_8192", "op": "gemm", "M": 8192, "N": 8192, "K": 8192, "out": "bfloat16", "b": "square"},
        # routed rows of 32 experts (one rank's share), ragged, one expert empty, capacity beyond the last row
        {"name": "experts", "op": "experts", "G": 32, "rows": 9001, "N": 2048, "K": 7168, "out": "bfloat16", "skew": 0.7},
        # weight gradients of 8 experts, both operands with a scale per row and block, fp32 accumulators kept
        {"name": "experts_wgrad", "op": "wgrad", "G": 8, "rows": 16384, "M": 2048, "N": 7168, "out": "float32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "route_step", "route_bwd", "weights_grad", "quantize", "quantize", "gemm", "gemm", "gemm", "experts", "experts", "wgrad"])
    if op.startswith("route"):
        E = _log(rng, 4, 512)
        k = min(E, rng.choice([1, 2, 3, 4, 6, 8]))
        T = _log(rng, 1, 32768)
        return {"op": op, "T": T, "E": E, "k": k, "dtype": rng.choice(["float32", "bfloat16"]), "norm": rng.random() < 0.6,
                "pad": rng.choice([0, T // 7]), "off": rng.choice([0, 0, E // 5])}
    if op == "weights_grad":
        return {"op": op, "T": _log(rng, 1, 8192), "k": rng.choice([1, 2, 4, 6, 8]), "H": 8 * _log(rng, 16, 896)}
    if op == "quantize":
        square = rng.random() < 0.4
        E = rng.choice([1, 1, 3])
        return {"op": op, "E": E, "M": _log(rng, 1, 16384) // E + 1, "N": _log(rng, 64, 7168), "dtype": rng.choice(["bfloat16", "float32"]),
                "both": rng.random() < 0.6, "square": square, "gather": E == 1 and not square and rng.random() < 0.4}
    if op == "gemm":
        return {"op": op, "M": _log(rng, 1, 8192), "N": _log(rng, 64, 8192), "K": _log(rng, 64, 8192), "out": rng.choice(["bfloat16", "float32"]),
                "b": rng.choice(["square", "rows"])}
    if op == "experts":
        return {"op": op, "G": _log(rng, 2, 64), "rows": _log(rng, 1, 12000), "N": 16 * _log(rng, 8, 256), "K": 16 * _log(rng, 8, 448),
                "out": rng.choice(["bfloat16", "float32"]), "skew": rng.choice([0.0, 0.7, 1.5])}
    G = _log(rng, 1, 16)
    return {"op": op, "G": G, "rows": BLK * _log(rng, 1, 96), "M": _log(rng, 64, 2048), "N": _log(rng, 64, 4096), "out": rng.choice(["bfloat16", "float32"])}


# ------------------------------------------------------------------------------------------------ inputs
def _dt(name):
    return getattr(torch, name)


def _pad16(n):
    return (n + 15) // 16 * 16


def _ceil(n):
    return (n + BLK - 1) // BLK


def _rows_quantized(x):
    """E4M3 bytes (row pitch a multiple of 16 bytes) and K-block-major scales of x [R, K]"""
    q, s = _quantize_rows_plain(x)
    buf = torch.zeros(x.shape[0], _pad16(x.shape[1]), dtype=torch.uint8, device=x.device)
    buf[:, :x.shape[1]] = q.view(torch.uint8)
    return buf.view(torch.float8_e4m3fn)[:, :x.shape[1]], s


def _square_quantized(x):
    q, s = _quantize_square_plain(x)
    buf = torch.zeros(*x.shape[:-1], _pad16(x.shape[-1]), dtype=torch.uint8, device=x.device)
    buf[..., :x.shape[-1]] = q.view(torch.uint8)
    return buf.view(torch.float8_e4m3fn)[..., :x.shape[-1]], s


def _group_sizes(G, rows, skew, unit, gen):
    """rows per group, popularity ~ exp(skew * N(0,1)); with more than four groups one of them is empty"""
    pop = torch.exp(skew * torch.randn(G, device=DEV, generator=gen))
    if G > 4:
        pop[G // 2] = 0
    total = rows // unit
    cut = torch.floor(torch.cumsum(pop, 0) / pop.sum() * total + 0.5).long()
    cut[-1] = total
    sizes = torch.diff(cut, prepend=torch.zeros(1, dtype=torch.long, device=DEV)).clamp(min=0) * unit
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rnd = lambda *shape: torch.randn(*shape, device=DEV, generator=gen)  # noqa: E731
    op = case["op"]
    s = {"op": op, "case": case}
    if op.startswith("route"):
        T, E, k = case["T"], case["E"], case["k"]
        # logits ~ N(0,1) with some experts more popular than others
        logits = rnd(T, E) + 0.3 * rnd(1, E)
        if case["off"]:
            logits[:, torch.randperm(E, device=DEV, generator=gen)[:case["off"]]] = float("-inf")
        s["logits"] = logits.to(_dt(case["dtype"]))
        s["mask"] = None
        if case["pad"]:
            mask = torch.ones(T, dtype=torch.bool, device=DEV)
            mask[T - case["pad"]:] = False
            s["mask"] = mask
        s["k"], s["norm"] = k, case["norm"]
        s["d_weights"] = rnd(T, k)
        s["d_loss"] = 0.01 + 0.001 * rnd(1).abs()
        if op == "route_bwd":
            idx, w, lse, counts, _, valid, _ = _route_plain(s["logits"], k, case["norm"], s["mask"])
            s["saved"] = (idx, w, lse, counts, valid)
    elif op == "weights_grad":
        s["d_out"] = (0.01 * rnd(case["T"], case["H"])).to(torch.bfloat16)
        s["combine"] = rnd(case["T"] * case["k"], case["H"]).to(torch.bfloat16)
        s["k"] = case["k"]
    elif op == "quantize":
        E, M, N = case["E"], case["M"], case["N"]
        s["index"] = None
        if case["gather"]:
            # every token is routed to several experts; each fifteenth row is padding
            src = max(1, M // 4)
            idx = torch.randint(0, src, (M,), device=DEV, generator=gen, dtype=torch.int32)
            idx[::15] = -1
            s["index"] = idx
            x = rnd(src, N)
        else:
            x = rnd(E, M, N) if E > 1 else rnd(M, N)
        x = x * (0.02 if case["square"] else 1.0)
        s["x"] = x.to(_dt(case["dtype"]))
    elif op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["a_sc"] = _rows_quantized(rnd(M, K))
        s["b"], s["b_sc"] = (_square_quantized if case["b"] == "square" else _rows_quantized)(0.02 * rnd(N, K))
        s["c"] = torch.zeros(M, N, dtype=_dt(case["out"]), device=DEV)
    elif op == "experts":
        G, N, K = case["G"], case["N"], case["K"]
        sizes = _group_sizes(G, case["rows"], case["skew"], 1, gen)
        cap = case["rows"] + 100          # capacity: rows behind the last group stay as they are
        s["a"], s["a_sc"] = _rows_quantized(rnd(cap, K))
        s["b"], s["b_sc"] = _square_quantized(0.02 * rnd(G, N, K))
        s["group_rows"], s["sizes"] = sizes.to(torch.int32), sizes.tolist()
        s["c"] = torch.zeros(cap, N, dtype=_dt(case["out"]), device=DEV)
    else:
        G, M, N = case["G"], case["M"], case["N"]
        sizes = _group_sizes(G, case["rows"], 0.7, BLK, gen)
        s["a"], s["a_sc"] = _rows_quantized(0.01 * rnd(M, case["rows"]))
        s["b"], s["b_sc"] = _rows_quantized(rnd(N, case["rows"]))
        s["group_rows"], s["sizes"] = sizes.to(torch.int32), sizes.tolist()
        s["c"] = torch.zeros(G, M, N, dtype=_dt(case["out"]), device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _route_plain(logits, k, norm, mask):
    T, E = logits.shape
    l = logits.float()
    valid = (l > float("-inf")).any(1)
    if mask is not None:
        valid = valid & mask
    # stable sort: ties go to the lower expert
    top, idx = torch.sort(l, dim=1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    taken = (top > float("-inf")) & valid[:, None]
    mx = top[:, :1]
    ex = torch.exp(l - mx)
    tot = ex.sum(1, keepdim=True)
    p = torch.where(valid[:, None], ex / tot, 0.0)
    lse = torch.where(valid, (mx + torch.log(tot))[:, 0], float("-inf"))
    w = torch.exp(top - mx)
    w = w / (torch.where(taken, w, 0.0).sum(1, keepdim=True) if norm else tot)
    w = torch.where(taken, w, 0.0)
    idx = torch.where(taken, idx, -1).to(torch.int32)
    counts = (idx.reshape(-1)[:, None].long() == torch.arange(E, device=l.device)).sum(0).to(torch.int32) if T * k * E < 1 << 16 else \
        torch.bincount(idx.reshape(-1).long() + 1, minlength=E + 1)[1:].to(torch.int32)
    prob_sum = p.double().sum(0)
    n = valid.sum().to(torch.int32)
    loss = (counts.double() * prob_sum).sum() * E / (k * n.double().clamp(min=1) ** 2)
    return idx, w, lse, counts, prob_sum.float(), n.reshape(1), loss.float().reshape(1)


def _route_bwd_plain(logits, idx, w, lse, counts, valid, d_w, d_loss, norm):
    T, E = logits.shape
    k = idx.shape[1]
    ok = (lse > float("-inf"))[:, None]
    p = torch.where(ok, torch.exp(logits.float() - lse[:, None]), 0.0)
    taken = idx >= 0
    at = idx.clamp(min=0).long()
    dw = torch.where(taken, d_w, 0.0)
    inner = w * (dw - (w * dw).sum(1, keepdim=True)) if norm else w * dw
    d = torch.zeros(T, E, dtype=torch.float32, device=logits.device).scatter_add_(1, at, torch.where(taken, inner, 0.0))
    if not norm:
        d = d - p * (w * dw).sum(1, keepdim=True)
    n = valid.double().clamp(min=1)
    b = (d_loss.double() * counts.double() * E / (k * n * n)).float()
    d = d + p * (b - (p * b).sum(1, keepdim=True))
    return torch.where(ok, d, 0.0).to(logits.dtype)


def _amax_to_scales(amax):
    amax = amax.clamp(min=AMAX_FLOOR)
    return amax / E4M3_MAX, E4M3_MAX / amax


def _quantize_rows_plain(x):
    """bytes [R, K] and scales [ceil(K / 128), R]"""
    R, K = x.shape
    xb = torch.nn.functional.pad(x.float(), (0, -K % BLK)).view(R, -1, BLK)
    sc, inv = _amax_to_scales(xb.abs().amax(2))
    q = (xb * inv[:, :, None]).view(R, -1)[:, :K].to(torch.float8_e4m3fn)
    return q, sc.t().contiguous()


def _quantize_square_plain(x):
    """bytes [.., M, N] and scales [.., ceil(M / 128), ceil(N / 128)]"""
    M, N = x.shape[-2:]
    xb = torch.nn.functional.pad(x.float(), (0, -N % BLK, 0, -M % BLK))
    xb = xb.view(*x.shape[:-2], _ceil(M), BLK, _ceil(N), BLK)
    sc, inv = _amax_to_scales(xb.abs().amax((-3, -1)))
    q = (xb * inv[..., :, None, :, None]).view(*x.shape[:-2], _ceil(M) * BLK, _ceil(N) * BLK)[..., :M, :N].to(torch.float8_e4m3fn)
    return q, sc


def _quantize_plain(x, index, both, square):
    if index is not None:
        x = torch.where((index >= 0)[:, None], x[index.clamp(min=0).long()], 0.0)
    if square:
        q, sc = _quantize_square_plain(x)
        return (q, sc, q.transpose(-1, -2).contiguous(), sc.transpose(-1, -2).contiguous()) if both else (q, sc)
    lead = x.shape[:-2]
    E, (M, N) = (lead[0] if lead else 1), x.shape[-2:]
    q, sc = _quantize_rows_plain(x.reshape(E * M, N))
    out = (q.view(*lead, M, N), sc.view(-1, E, M).transpose(0, 1).reshape(*lead, -1, M))
    if both:
        qt, st = _quantize_rows_plain(x.transpose(-1, -2).reshape(E * N, M))
        out += (qt.view(*lead, N, M), st.view(-1, E, N).transpose(0, 1).reshape(*lead, -1, N))
    return out


def _wide_rows(q, sc, to):
    """values of row blocks: bytes [R, K], scales [KB, R]"""
    return q.to(to) * torch.repeat_interleave(sc.to(to).t(), BLK, 1)[:, :q.shape[1]]


def _wide_square(q, sc, to):
    N, K = q.shape[-2:]
    return q.to(to) * torch.repeat_interleave(torch.repeat_interleave(sc.to(to), BLK, -2)[..., :N, :], BLK, -1)[..., :K]


def _run_plain(s):
    op = s["op"]
    if op == "route":
        return _route_plain(s["logits"], s["k"], s["norm"], s["mask"])
    if op == "route_step":
        out = _route_plain(s["logits"], s["k"], s["norm"], s["mask"])
        return out + (_route_bwd_plain(s["logits"], out[0], out[1], out[2], out[3], out[5], s["d_weights"], s["d_loss"], s["norm"]),)
    if op == "route_bwd":
        return _route_bwd_plain(s["logits"], *s["saved"], s["d_weights"], s["d_loss"], s["norm"])
    if op == "weights_grad":
        T, H = s["d_out"].shape
        return torch.bmm(s["combine"].float().view(T, s["k"], H), s["d_out"].float().view(T, H, 1)).view(T, s["k"])
    if op == "quantize":
        return _quantize_plain(s["x"], s["index"], s["case"]["both"], s["case"]["square"])
    c = s["c"]
    if op == "gemm":
        a = _wide_rows(s["a"], s["a_sc"], torch.float32)
        b = (_wide_square if s["case"]["b"] == "square" else _wide_rows)(s["b"], s["b_sc"], torch.float32)
        return c.copy_(a @ b.t())
    at = 0
    if op == "experts":
        # one product per expert: a padded batched product would multiply more
        for g, n in enumerate(s["sizes"]):
            if n:
                a = _wide_rows(s["a"][at:at + n], s["a_sc"][:, at:at + n], torch.float32)
                c[at:at + n] = a @ _wide_square(s["b"][g], s["b_sc"][g], torch.float32).t()
            at += n
        return c
    for g, n in enumerate(s["sizes"]):
        a = _wide_rows(s["a"][:, at:at + n], s["a_sc"][at // BLK:(at + n) // BLK], torch.float32)
        c[g] = a @ _wide_rows(s["b"][:, at:at + n], s["b_sc"][at // BLK:(at + n) // BLK], torch.float32).t()
        at += n
    return c


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    mx8 = _mx8()
    op = s["op"]
    if op == "route":
        return mx8.router_topk(s["logits"], s["k"], normalize=s["norm"], token_mask=s["mask"])
    if op == "route_step":
        out = mx8.router_topk(s["logits"], s["k"], normalize=s["norm"], token_mask=s["mask"])
        idx, w, lse, counts, _, valid, _ = out
        return tuple(out) + (mx8.router_topk_bwd(s["logits"], idx, w, lse, counts, valid, s["d_weights"], s["d_loss"], normalize=s["norm"]),)
    if op == "route_bwd":
        return mx8.router_topk_bwd(s["logits"], *s["saved"], s["d_weights"], s["d_loss"], normalize=s["norm"])
    if op == "weights_grad":
        return mx8.bwd_topk_weights(s["d_out"], s["combine"])
    if op == "quantize":
        both = s["case"]["both"]
        out = mx8.quantize_block128(s["x"], True, both, square=s["case"]["square"], row_index=s["index"])
        return out if both else out[:2]
    if op == "gemm":
        return mx8.gemm_block128(s["a"], s["a_sc"], s["b"], s["b_sc"], s["c"], b_blocks=s["case"]["b"])
    if op == "experts":
        return mx8.gemm_block128(s["a"], s["a_sc"], s["b"], s["b_sc"], s["c"], group_rows=s["group_rows"])
    return mx8.gemm_block128_wgrad(s["a"], s["a_sc"], s["b"], s["b_sc"], s["c"], group_rows=s["group_rows"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op.startswith("route"):
        T, E, k = case["T"], case["E"], case["k"]
        b = 4 if case["dtype"] == "float32" else 2
        live = T - case["pad"]
        fwd = live * E * b + T * (8 * k + 4) + 8 * E + 8
        bwd = live * E * b + T * E * b + T * (12 * k + 4) + 4 * E
        return {"bytes": fwd if op == "route" else bwd if op == "route_bwd" else fwd + T * E * b + T * 4 * k,
                "flops": (live * E * 4 if op != "route_bwd" else 0) + (live * E * 5 if op != "route" else 0)}
    if op == "weights_grad":
        T, k, H = case["T"], case["k"], case["H"]
        return {"bytes": 2 * T * (k + 1) * H + 4 * T * k, "flops": 2 * T * k * H}
    if op == "quantize":
        E, M, N = case["E"], case["M"], case["N"]
        b = 4 if case["dtype"] == "float32" else 2
        src = max(1, M // 4) if case["gather"] else M
        one = M * N + (4 * _ceil(M) * _ceil(N) if case["square"] else 4 * M * _ceil(N))
        two = M * N + (4 * _ceil(M) * _ceil(N) if case["square"] else 4 * N * _ceil(M))
        return {"bytes": E * (src * N * b + one + (two if case["both"] else 0)) + (4 * M if case["gather"] else 0), "flops": 3 * E * M * N}
    o = 4 if case["out"] == "float32" else 2
    if op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        sb = 4 * _ceil(K) * (_ceil(N) if case["b"] == "square" else N)
        return {"bytes": M * K + N * K + 4 * M * _ceil(K) + sb + M * N * o, "flops": 2 * M * N * K}
    if op == "experts":
        G, R, N, K = case["G"], case["rows"], case["N"], case["K"]
        live = min(G - (1 if G > 4 else 0), R)          # experts whose weights are read, at most
        return {"bytes": R * K + live * N * K + 4 * R * _ceil(K) + 4 * live * _ceil(N) * _ceil(K) + R * N * o + 4 * G, "flops": 2 * R * N * K}
    G, R, M, N = case["G"], case["rows"], case["M"], case["N"]
    return {"bytes": (M + N) * (R + 4 * (R // BLK)) + G * M * N * o + 4 * G, "flops": 2 * R * M * N}


# ------------------------------------------------------------------------------------------------ 64 bits
def _route_exact(logits, k, norm, mask):
    T, E = logits.shape
    l = logits.double()
    if mask is not None:
        l = l.masked_fill(~mask[:, None], float("-inf"))
    dead = torch.isinf(l).all(1)
    n = T - int(dead.sum())
    lse = torch.logsumexp(l, 1)
    p = torch.softmax(l, 1).masked_fill(dead[:, None], 0.0)
    chosen = torch.zeros(T, E, dtype=torch.bool, device=l.device)
    left, order = l.clone(), []
    for _ in range(k):
        best = left.max(1, keepdim=True).values
        e = torch.where(left == best, torch.arange(E, device=l.device), E).min(1).values
        alive = best[:, 0] > float("-inf")
        order.append(torch.where(alive, e, -1))
        chosen[alive, e[alive]] = True
        left[torch.arange(T, device=l.device), e.clamp(max=E - 1)] = float("-inf")
    idx = torch.stack(order, 1)
    w = torch.where(idx >= 0, torch.gather(p, 1, idx.clamp(min=0)), 0.0)
    if norm:
        w = torch.where(idx >= 0, w / w.sum(1, keepdim=True), 0.0)
    counts = chosen.sum(0)
    loss = (counts * p.sum(0)).sum() * E / (k * max(n, 1) ** 2)
    return p, idx, w, lse, counts, n, loss


def _route_exact_bwd(p, idx, w, counts, n, d_w, d_loss, norm):
    T, E = p.shape
    k = idx.shape[1]
    hit = torch.nn.functional.one_hot(idx + 1, E + 1)[:, :, 1:].double()          # [T, k, E]
    up = torch.einsum("tke,tk->te", hit, d_w.double())                            # gradient at the chosen experts
    if norm:
        g = torch.einsum("tke,tk->te", hit, w)
        d = g * (up - (g * up).sum(1, keepdim=True))
    else:
        d = p * (up - (p * up).sum(1, keepdim=True))
    b = d_loss.double() * counts * E / (k * max(n, 1) ** 2)
    return d + p * (b - p @ b.reshape(-1, 1))


def _exact_scales(amax):
    return amax.clamp(min=AMAX_FLOOR) / E4M3_MAX


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op.startswith("route"):
        p, idx, w, lse, counts, n, loss = _route_exact(s["logits"], s["k"], s["norm"], s["mask"])
        d = None
        if op != "route":
            d = _route_exact_bwd(p, idx, w, counts, n, s["d_weights"], s["d_loss"], s["norm"])
        if op == "route_bwd":
            return d
        out = (None, w, lse, None, p.sum(0), None, loss.reshape(1))
        return out if op == "route" else out + (d,)
    if op == "weights_grad":
        T, H = s["d_out"].shape
        return torch.einsum("tkh,th->tk", s["combine"].double().view(T, s["k"], H), s["d_out"].double())
    if op == "quantize":
        # bytes stand for x / scale rounded to 3 bits: the values before that rounding are what they are near to
        x = s["x"].double()
        if s["index"] is not None:
            x = torch.cat([x, torch.zeros_like(x[:1])])[s["index"].long()]          # -1: the zero row
        M, N = x.shape[-2:]
        lead = x.shape[:-2]
        full = torch.zeros(*lead, _ceil(M) * BLK, _ceil(N) * BLK, dtype=torch.float64, device=x.device)
        full[..., :M, :N] = x
        t = full.view(*lead, _ceil(M), BLK, _ceil(N), BLK).abs()
        e4m3 = lambda v: v.float().to(torch.float8_e4m3fn).double()  # noqa: E731
        if case["square"]:
            sc = _exact_scales(t.amax((-3, -1)))
            q = e4m3((full.view(t.shape) / sc[..., :, None, :, None]).view(full.shape)[..., :M, :N])
            out = (q, sc)
            return out + (q.transpose(-1, -2), sc.transpose(-1, -2)) if case["both"] else out
        sc = _exact_scales(t.amax(-1).view(*lead, _ceil(M) * BLK, _ceil(N)))
        q = e4m3((full.view(*lead, _ceil(M) * BLK, _ceil(N), BLK) / sc[..., None]).view(full.shape)[..., :M, :N])
        out = (q, sc[..., :M, :].transpose(-1, -2))
        if case["both"]:
            st = _exact_scales(t.amax(-3).view(*lead, _ceil(M), _ceil(N) * BLK))
            qt = e4m3((full.view(*lead, _ceil(M), BLK, _ceil(N) * BLK) / st[..., :, None, :]).view(full.shape)[..., :M, :N].transpose(-1, -2))
            out += (qt, st[..., :N])
        return out

    def rows64(q, sc):
        kb = torch.arange(q.shape[1], device=q.device) // BLK
        return q.double() * sc.double()[kb].t()

    def square64(q, sc):
        rb, kb = torch.arange(q.shape[0], device=q.device) // BLK, torch.arange(q.shape[1], device=q.device) // BLK
        return q.double() * sc.double()[rb][:, kb]

    if op == "gemm":
        b = (square64 if case["b"] == "square" else rows64)(s["b"], s["b_sc"])
        return rows64(s["a"], s["a_sc"]) @ b.t()
    c, at = s["c"].double(), 0
    a = rows64(s["a"], s["a_sc"])
    for g, n in enumerate(s["sizes"]):
        if op == "experts":
            c[at:at + n] = a[at:at + n] @ square64(s["b"][g], s["b_sc"][g]).t()
        else:
            c[g] = a[:, at:at + n] @ rows64(s["b"][:, at:at + n], s["b_sc"][at // BLK:(at + n) // BLK]).t()
        at += n
    return c
