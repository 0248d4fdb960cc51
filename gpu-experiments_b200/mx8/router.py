"""Router of the MoE layer: top-k selection with the balance loss, its gradient, and the gradient of the routing weights.

`router_topk` makes the ids that `schedule` reads and the weights that `fwd_epilogue` applies; the backward runs from `fwd_epilogue`'s
gradient through `bwd_topk_weights` to `router_topk_bwd`.  Outputs are allocated here; launches go to torch's current stream of the
input's device.  A bad tensor raises ValueError, a size that the library refuses Mx8Error.
"""
from ._lib import host


def router_topk(logits, topk, *, normalize=True, token_mask=None):
    """router_topk(logits, topk)
        -> (topk_idx, topk_weights, lse, counts, prob_sum, num_valid, balance_loss)

    logits [T, E], bf16 or float32.  p = softmax(logits) in float32; topk_idx int32 [T, topk] are the largest logits of a token, largest
    first, ties to the lower expert; topk_weights float32 [T, topk] is p there, divided by its sum over the choices when `normalize`.
    token_mask (bool [T]): False for a token that takes no part.  A logit of -inf switches an expert off for its token.  Choices that
    cannot be filled, and all of a token that takes no part, have id -1 (no rank owns it, `schedule` skips it, `combine` leaves its row as it
    was) and weight 0 (`fwd_epilogue` adds nothing for it).
    lse [T] float32 is saved for the backward; counts int32 [E]; prob_sum float32 [E]; num_valid int32 [1];
    balance_loss float32 [1] = E / (topk num_valid^2) sum_e counts[e] prob_sum[e]: 1 for an even spread.
    At most 1024 experts and 32 choices.  counts and num_valid, prob_sum and balance_loss, and in small calls all outputs of a type share
    a storage (saving one of them saves its storage; `clone` it to keep it alone)."""
    return host().router_topk(logits, topk, normalize, token_mask)


def router_topk_bwd(logits, topk_idx, topk_weights, lse, counts, num_valid, d_topk_weights=None, d_balance_loss=None, *, normalize=True):
    """Gradient of `router_topk` with respect to the logits, [T, E] in their type.

    d_topk_weights float32 [T, topk] (from `bwd_topk_weights`) and d_balance_loss float32 [1]; either may be None.  The counts are
    constants of the loss.  counts and num_valid summed over ranks give the gradient of the loss over all ranks' tokens."""
    return host().router_topk_bwd(logits, topk_idx, topk_weights, lse, counts, num_valid, d_topk_weights, d_balance_loss, normalize)


def bwd_topk_weights(d_output, combine_buffer, topk_idx=None):
    """d_topk_weights[t, j] = sum_h d_output[t, h] * combine_buffer[t * topk + j, h], float32 [T, topk]: the gradient of the weights that
    `fwd_epilogue` applied.  d_output [T, H] and combine_buffer [T * topk, H] bf16; topk_idx (int32 [T, topk]): choices with a negative
    id get 0 and their rows, which the combine did not write, are not read."""
    return host().bwd_topk_weights(d_output, combine_buffer, topk_idx)
