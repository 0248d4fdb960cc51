"""Operators of the block-128 format: E4M3 bytes with one fp32 scale per block of 128.

A row block is 1 x 128 along the contraction, its scales are stored block-major, sc[block][row]; a square is 128 x 128, sc[row block]
[column block].  Activations and gradients use row blocks, weights squares, so that one quantization of a weight serves the forward
and, transposed, the data gradient; weight gradients multiply two transposed row-block operands.  Matrices may have any size; the
bytes of a row start on a 16-byte boundary, so tensors allocated here are slices of rows padded to a multiple of 16.
"""
from ._lib import host


def quantize_block128(x, return_normal=True, return_transposed=False, *, square=False, row_index=None):
    """quantize_block128(x, return_normal, return_transposed) -> (x_fp8, x_sc, x_fp8_t, x_sc_t)

    x [M, N] or [E, M, N], bf16 or float32.  x_fp8 [.., M, N] with scales x_sc [.., ceil(N/128), M] of row blocks along N; x_fp8_t
    [.., N, M] with x_sc_t [.., ceil(M/128), N], the transpose with blocks along M.  square=True: one scale per 128 x 128, x_sc
    [.., ceil(M/128), ceil(N/128)] and x_sc_t its transpose.  Outputs not requested are None.
    row_index (int32 [rows], x 2-D): row r of the output is x[row_index[r]], zeros where the index is outside x: the rows of a routing
    schedule (token = peer_token_idx // topk, -1 for padding) are gathered while they are quantized.
    scale = amax / 448 (amax at least 2^-110), byte = e4m3(x * 448 / amax), the quotient rounded to float32
    (for bfloat16 x times the rounded 448 / amax: another byte only where the quotient lies midway between two); a block with an infinity or NaN dequantizes to NaN.
    """
    return host().quantize_block128(x, return_normal, return_transposed, square, row_index)


def gemm_block128(A, A_sc, B, B_sc, C, *, b_blocks="square", group_rows=None):
    """C = dequant(A) . dequant(B)^T, fp32 sums; returns C.

    A [M, K] E4M3 with row-block scales A_sc [ceil(K/128), M]; B [N, K] with squares B_sc [ceil(N/128), ceil(K/128)], or with row blocks
    B_sc [ceil(K/128), N] and b_blocks="rows"; C [M, N] preallocated, bf16 or float32.  Row pitches of A and B are multiples of 16 bytes
    (what quantize_block128 returns); M, N and K need not be multiples of anything.
    group_rows (int32 [G] on the device): the rows of A belong to G groups back to back, B is [G, N, K] with squares
    [G, ceil(N/128), ceil(K/128)]; group sizes may be any, 0 included; rows of C behind the last group are left as they are.
    """
    return host().gemm_block128(A, A_sc, B, B_sc, C, b_blocks, group_rows)


def gemm_block128_wgrad(A_t, A_t_sc, B_t, B_t_sc, C, group_rows):
    """C[g] = dequant(A_t[:, rows_g]) . dequant(B_t[:, rows_g])^T for every group; returns C.

    A_t [M, R] and B_t [N, R] are transposed outputs of quantize_block128 (scales [ceil(R/128), M] and [ceil(R/128), N]); group_rows int32 [G]
    on the device, multiples of 128, sizes of consecutive ranges of R; C [G, M, N], bf16 or float32.  A group without rows yields
    zeros.  For a single matrix call gemm_block128 with b_blocks="rows"."""
    return host().gemm_block128_wgrad(A_t, A_t_sc, B_t, B_t_sc, C, group_rows)
