"""Operators of the block-128 format: E4M3 bytes with one fp32 scale per block of 128.

A row block is 1 x 128 along the contraction, its scales are stored block-major, sc[block][row]; a square is 128 x 128, sc[row block]
[column block].  Activations and gradients use row blocks, weights squares, so that one quantization of a weight serves the forward
and, transposed, the data gradient; weight gradients multiply two transposed row-block operands.  Matrices may have any size; the
bytes of a row start on a 16-byte boundary, so tensors allocated here are slices of rows padded to a multiple of 16.
"""
import torch

from . import _lib
from .ops import _FP8, _stream

_F32 = (torch.float32,)
_C = {torch.bfloat16: _lib.C_BF16, torch.float32: _lib.C_F32}
_X = {torch.bfloat16: _lib.T_BF16, torch.float32: _lib.T_F32}


def _cdiv(a):
    return (a + 127) // 128


def _matrix(t, name, dtypes, shape, device):
    """pointer and row pitch of a tensor [.., rows, cols] whose columns are contiguous and whose leading dimensions are packed"""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has dtype {t.dtype}, expected one of {tuple(dtypes)}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    st = t.stride()
    rows, cols = shape[-2], shape[-1]
    if st[-1] != 1 and cols > 1:
        raise ValueError(f"{name} must have contiguous rows")
    # the stride of a dimension of size one says nothing
    if rows > 1:
        pitch = st[-2]
    elif len(shape) == 3 and shape[0] > 1:
        pitch = st[-3]
    else:
        pitch = max(cols, st[-2])
    if len(shape) == 3 and shape[0] > 1 and st[-3] != rows * pitch:
        raise ValueError(f"{name}: the matrices must lie back to back")
    return t.data_ptr(), pitch


def _cuda(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.device


def _bytes_out(lead, rows, cols, device):
    """[.., rows, cols] E4M3 whose rows start on 16-byte boundaries"""
    pitch = (cols + 15) // 16 * 16
    t = torch.empty(*lead, rows, pitch, dtype=torch.float8_e4m3fn, device=device)
    return t if pitch == cols else t[..., :cols]


def quantize_block128(x, return_normal=True, return_transposed=False, *, square=False, row_index=None):
    """quantize_block128(x, return_normal, return_transposed) -> (x_fp8, x_sc, x_fp8_t, x_sc_t)

    x [M, N] or [E, M, N], bf16 or float32.  x_fp8 [.., M, N] with scales x_sc [.., ceil(N/128), M] of row blocks along N; x_fp8_t
    [.., N, M] with x_sc_t [.., ceil(M/128), N], the transpose with blocks along M.  square=True: one scale per 128 x 128, x_sc
    [.., ceil(M/128), ceil(N/128)] and x_sc_t its transpose.  Outputs not requested are None.
    row_index (int32 [rows], x 2-D): row r of the output is x[row_index[r]], zeros where the index is outside x: the rows of a routing
    schedule (token = peer_token_idx // topk, -1 for padding) are gathered while they are quantized.
    scale = amax / 448 (amax at least 2^-110), byte = e4m3(x * (448 / amax)); a block with an infinity or NaN dequantizes to NaN.
    """
    lib = _lib.load()
    dev = _cuda(x, "x")
    if x.dim() not in (2, 3) or x.numel() == 0:
        raise ValueError("x must be [M, N] or [E, M, N] and not empty")
    if not (return_normal or return_transposed):
        raise ValueError("at least one of return_normal / return_transposed must be set")
    xp, ldx = _matrix(x, "x", _X, x.shape, dev)
    lead = tuple(x.shape[:-2])
    E = lead[0] if lead else 1
    M, N = x.shape[-2:]
    src, ip = M, None
    if row_index is not None:
        if lead or square:
            raise ValueError("row_index takes a 2-D x and row blocks")
        if row_index.dtype != torch.int32 or row_index.dim() != 1 or not row_index.is_contiguous() or row_index.device != dev or row_index.numel() == 0:
            raise ValueError(f"row_index must be a contiguous int32 vector on {dev}, not empty")
        M, ip = row_index.numel(), row_index.data_ptr()
    q = sc = qt = sct = None
    p = [None, N, None, None, M, None]
    f32 = dict(dtype=torch.float32, device=dev)
    if return_normal:
        q = _bytes_out(lead, M, N, dev)
        sc = torch.empty(*lead, *((_cdiv(M), _cdiv(N)) if square else (_cdiv(N), M)), **f32)
        p[0:3] = q.data_ptr(), (N + 15) // 16 * 16, sc.data_ptr()
    if return_transposed:
        qt = _bytes_out(lead, N, M, dev)
        sct = torch.empty(*lead, *((_cdiv(N), _cdiv(M)) if square else (_cdiv(M), N)), **f32)
        p[3:6] = qt.data_ptr(), (M + 15) // 16 * 16, sct.data_ptr()
    with torch.cuda.device(dev):
        _lib.check(lib.mx8_quantize_block128(xp, _X[x.dtype], E, M, N, ldx, ip, src, *p, int(square), _stream()), "quantize_block128")
    return q, sc, qt, sct


def _scales(t, name, blocks, rows, device):
    """pointer and pitch of row-block scales [blocks, rows]"""
    ptr, pitch = _matrix(t, name, _F32, (blocks, rows), device)
    return ptr, max(pitch, rows)


def _groups(group_rows, device):
    if group_rows.dtype != torch.int32 or group_rows.dim() != 1 or not group_rows.is_contiguous() or group_rows.device != device or group_rows.numel() == 0:
        raise ValueError(f"group_rows must be a contiguous int32 vector on {device}, not empty")
    return group_rows.data_ptr(), group_rows.numel()


def gemm_block128(A, A_sc, B, B_sc, C, *, b_blocks="square", group_rows=None):
    """C = dequant(A) . dequant(B)^T, fp32 sums; returns C.

    A [M, K] E4M3 with row-block scales A_sc [ceil(K/128), M]; B [N, K] with squares B_sc [ceil(N/128), ceil(K/128)], or with row blocks
    B_sc [ceil(K/128), N] and b_blocks="rows"; C [M, N] preallocated, bf16 or float32.  Row pitches of A and B are multiples of 16 bytes
    (what quantize_block128 returns); M, N and K need not be multiples of anything.
    group_rows (int32 [G] on the device): the rows of A belong to G groups back to back, B is [G, N, K] with squares
    [G, ceil(N/128), ceil(K/128)]; group sizes may be any, 0 included; rows of C behind the last group are left as they are.
    """
    lib = _lib.load()
    dev = _cuda(A, "A")
    if b_blocks not in ("square", "rows"):
        raise ValueError('b_blocks is "square" or "rows"')
    if A.dim() != 2 or B.dim() != (2 if group_rows is None else 3):
        raise ValueError("A is [M, K]; B is [N, K], or [G, N, K] with group_rows")
    M, K = A.shape
    N = B.shape[-2]
    if M == 0 or N == 0 or K == 0:
        raise ValueError("empty operand")
    ap, lda = _matrix(A, "A", _FP8, (M, K), dev)
    asp, ldsa = _scales(A_sc, "A_sc", _cdiv(K), M, dev)
    cp, ldc = _matrix(C, "C", _C, (M, N), dev)
    square = b_blocks == "square"
    if group_rows is not None:
        if not square:
            raise ValueError("grouped weights have square blocks")
        gp, G = _groups(group_rows, dev)
        bp, ldb = _matrix(B, "B", _FP8, (G, N, K), dev)
        bs, shape = B_sc, (G, _cdiv(N), _cdiv(K))
    else:
        gp, G = None, 0
        bp, ldb = _matrix(B, "B", _FP8, (N, K), dev)
        bs, shape = B_sc, (_cdiv(N), _cdiv(K))
    if square:
        bsp, ldsb = _matrix(bs, "B_sc", _F32, shape, dev)
        if not bs.is_contiguous():
            raise ValueError("square scales must be contiguous")
    else:
        bsp, ldsb = _scales(B_sc, "B_sc", _cdiv(K), N, dev)
    with torch.cuda.device(dev):
        _lib.check(lib.mx8_gemm_block128(ap, lda, asp, ldsa, bp, ldb, bsp, ldsb, int(square), cp, ldc, M, N, K, _C[C.dtype], gp, G, _stream()),
                   "gemm_block128")
    return C


def gemm_block128_wgrad(A_t, A_t_sc, B_t, B_t_sc, C, group_rows):
    """C[g] = dequant(A_t[:, rows_g]) . dequant(B_t[:, rows_g])^T for every group; returns C.

    A_t [M, R] and B_t [N, R] are transposed outputs of quantize_block128 (scales [ceil(R/128), M] and [ceil(R/128), N]); group_rows int32 [G]
    on the device, multiples of 128, sizes of consecutive ranges of R; C [G, M, N], bf16 or float32.  A group without rows yields
    zeros.  For a single matrix call gemm_block128 with b_blocks="rows"."""
    lib = _lib.load()
    dev = _cuda(A_t, "A_t")
    if A_t.dim() != 2 or B_t.dim() != 2:
        raise ValueError("A_t is [M, R], B_t is [N, R]")
    M, R = A_t.shape
    N = B_t.shape[0]
    if M == 0 or N == 0 or R == 0:
        raise ValueError("empty operand")
    gp, G = _groups(group_rows, dev)
    ap, lda = _matrix(A_t, "A_t", _FP8, (M, R), dev)
    bp, ldb = _matrix(B_t, "B_t", _FP8, (N, R), dev)
    asp, ldsa = _scales(A_t_sc, "A_t_sc", _cdiv(R), M, dev)
    bsp, ldsb = _scales(B_t_sc, "B_t_sc", _cdiv(R), N, dev)
    cp, ldc = _matrix(C, "C", _C, (G, M, N), dev)
    with torch.cuda.device(dev):
        _lib.check(lib.mx8_gemm_block128_wgrad(ap, lda, asp, ldsa, bp, ldb, bsp, ldsb, cp, ldc, M, N, R, _C[C.dtype], gp, G, _stream()),
                   "gemm_block128_wgrad")
    return C
