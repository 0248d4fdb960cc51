"""Router of the MoE layer: top-k selection with the balance loss, its gradient, and the gradient of the routing weights.

`router_topk` makes the ids that `schedule` reads and the weights that `fwd_epilogue` applies; the backward runs from `fwd_epilogue`'s
gradient through `bwd_topk_weights` to `router_topk_bwd`.
"""
import torch

from . import _lib
from .ops import _stream

_LOGITS = {torch.bfloat16: _lib.T_BF16, torch.float32: _lib.T_F32}


def _logits(logits):
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    if logits.dtype not in _LOGITS:
        raise ValueError(f"logits have dtype {logits.dtype}, expected bfloat16 or float32")
    if logits.dim() != 2 or logits.numel() == 0:
        raise ValueError("logits must be [tokens, experts] and not empty")
    T, E = logits.shape
    if E > 1 and logits.stride(1) != 1:
        raise ValueError("logits must have contiguous rows")
    return T, E, (logits.stride(0) if T > 1 else E)


def _vec(t, name, dtype, shape, device):
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def router_topk(logits, topk, *, normalize=True, token_mask=None):
    """router_topk(logits, topk)
        -> (topk_idx, topk_weights, lse, counts, prob_sum, num_valid, balance_loss)

    logits [T, E], bf16 or float32.  p = softmax(logits) in float32; topk_idx int32 [T, topk] are the largest logits of a token, largest
    first, ties to the lower expert; topk_weights float32 [T, topk] is p there, divided by its sum over the choices when `normalize`.
    token_mask (bool [T]): False for a token that takes no part.  A logit of -inf switches an expert off for its token.  Choices that
    cannot be filled, and all of a token that takes no part, have id -1 (no rank owns it, `schedule` skips it) and weight 0.
    lse [T] float32 is saved for the backward; counts int32 [E]; prob_sum float32 [E]; num_valid int32 [1];
    balance_loss float32 [1] = E / (topk num_valid^2) sum_e counts[e] prob_sum[e]: 1 for an even spread.
    At most 1024 experts and 32 choices."""
    lib = _lib.load()
    T, E, ld = _logits(logits)
    dev = logits.device
    topk = int(topk)
    mp = None
    if token_mask is not None:
        mp = _vec(token_mask, "token_mask", torch.bool, (T,), dev)
    idx = torch.empty(T, max(topk, 0), dtype=torch.int32, device=dev)
    weights = torch.empty(T, max(topk, 0), dtype=torch.float32, device=dev)
    lse = torch.empty(T, dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    prob_sum = torch.empty(E, dtype=torch.float32, device=dev)
    num_valid = torch.empty(1, dtype=torch.int32, device=dev)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        need = lib.mx8_router_topk_workspace_bytes(T, E)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.mx8_router_topk(logits.data_ptr(), _LOGITS[logits.dtype], ld, T, E, topk, int(normalize), mp, idx.data_ptr(),
                                       weights.data_ptr(), lse.data_ptr(), counts.data_ptr(), prob_sum.data_ptr(), num_valid.data_ptr(),
                                       loss.data_ptr(), ws.data_ptr() if need else None, need, _stream()), "router_topk")
    return idx, weights, lse, counts, prob_sum, num_valid, loss


def router_topk_bwd(logits, topk_idx, topk_weights, lse, counts, num_valid, d_topk_weights=None, d_balance_loss=None, *, normalize=True):
    """Gradient of `router_topk` with respect to the logits, [T, E] in their type.

    d_topk_weights float32 [T, topk] (from `bwd_topk_weights`) and d_balance_loss float32 [1]; either may be None.  The counts are
    constants of the loss.  counts and num_valid summed over ranks give the gradient of the loss over all ranks' tokens."""
    lib = _lib.load()
    T, E, ld = _logits(logits)
    dev = logits.device
    if topk_idx.dim() != 2:
        raise ValueError("topk_idx must be [tokens, topk]")
    k = topk_idx.shape[1]
    if d_topk_weights is None and d_balance_loss is None:
        raise ValueError("one of d_topk_weights and d_balance_loss must be given")
    ptrs = [_vec(topk_idx, "topk_idx", torch.int32, (T, k), dev), _vec(topk_weights, "topk_weights", torch.float32, (T, k), dev),
            _vec(lse, "lse", torch.float32, (T,), dev), _vec(counts, "counts", torch.int32, (E,), dev),
            _vec(num_valid, "num_valid", torch.int32, (1,), dev),
            _vec(d_topk_weights, "d_topk_weights", torch.float32, (T, k), dev) if d_topk_weights is not None else None,
            _vec(d_balance_loss, "d_balance_loss", torch.float32, (1,), dev) if d_balance_loss is not None else None]
    d_logits = torch.empty(T, E, dtype=logits.dtype, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.mx8_router_topk_bwd(logits.data_ptr(), _LOGITS[logits.dtype], ld, T, E, k, int(normalize), *ptrs, d_logits.data_ptr(),
                                           _stream()), "router_topk_bwd")
    return d_logits


def bwd_topk_weights(d_output, combine_buffer, topk_idx=None):
    """d_topk_weights[t, j] = sum_h d_output[t, h] * combine_buffer[t * topk + j, h], float32 [T, topk]: the gradient of the weights that
    `fwd_epilogue` applied.  d_output [T, H] and combine_buffer [T * topk, H] bf16; topk_idx (int32 [T, topk]): choices with a negative
    id get 0 and their rows, which the combine did not write, are not read."""
    lib = _lib.load()
    if not isinstance(d_output, torch.Tensor) or not d_output.is_cuda:
        raise ValueError("d_output must be a CUDA tensor")
    dev = d_output.device
    if d_output.dim() != 2 or combine_buffer.dim() != 2 or d_output.numel() == 0 or combine_buffer.numel() == 0 or combine_buffer.shape[0] % d_output.shape[0]:
        raise ValueError("d_output is [T, H], combine_buffer [T * topk, H], neither empty")
    T, H = d_output.shape
    k = combine_buffer.shape[0] // T
    gp = _vec(d_output, "d_output", torch.bfloat16, (T, H), dev)
    cp = _vec(combine_buffer, "combine_buffer", torch.bfloat16, (T * k, H), dev)
    ip = _vec(topk_idx, "topk_idx", torch.int32, (T, k), dev) if topk_idx is not None else None
    out = torch.empty(T, k, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.mx8_moe_bwd_topk_weights(gp, cp, ip, out.data_ptr(), T, H, k, _stream()), "bwd_topk_weights")
    return out
