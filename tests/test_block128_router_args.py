"""Refusals of the router and block-128 entry points: every bad argument is turned down before a device is touched."""
import ctypes

import pytest
import torch

import mx8
from mx8 import _lib

P = ctypes.c_void_p(4096)         # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4098)


@pytest.fixture(scope="module")
def lib():
    return mx8.load()


def test_router_topk_arguments(lib):
    def call(logits=P, dtype=1, ld=8, tokens=4, experts=8, topk=2, idx=P, lse=P, ws=P, ws_bytes=1 << 20):
        return lib.mx8_router_topk(logits, dtype, ld, tokens, experts, topk, 1, None, idx, P, lse, P, P, P, P, ws, ws_bytes, None)

    assert call(logits=None) == _lib.ERR_ARG and call(lse=None) == _lib.ERR_ARG and call(dtype=2) == _lib.ERR_ARG
    for bad in ({"tokens": 0}, {"experts": 0}, {"topk": 0}, {"topk": 9}, {"ld": 7}, {"tokens": -3}):
        assert call(**bad) == _lib.ERR_SIZE, bad
        assert b"topk" in lib.mx8_last_cuda_error()
    assert call(experts=1025, ld=1025) == _lib.ERR_LIMIT
    assert call(experts=64, ld=64, topk=33) == _lib.ERR_LIMIT
    assert call(tokens=1 << 30, topk=2) == _lib.ERR_LIMIT
    assert call(logits=ODD) == _lib.ERR_ALIGN and call(idx=ODD) == _lib.ERR_ALIGN


def test_router_topk_bwd_arguments(lib):
    def call(logits=P, dtype=0, ld=8, topk=2, counts=P, dw=P, dl=P, out=P):
        return lib.mx8_router_topk_bwd(logits, dtype, ld, 4, 8, topk, 1, P, P, P, counts, P, dw, dl, out, None)

    assert call(out=None) == _lib.ERR_ARG and call(counts=None) == _lib.ERR_ARG and call(dtype=-1) == _lib.ERR_ARG
    assert call(dw=None, dl=None) == _lib.ERR_ARG
    assert call(topk=9) == _lib.ERR_SIZE and call(ld=3) == _lib.ERR_SIZE
    assert call(dw=ODD) == _lib.ERR_ALIGN and call(dtype=1, out=ODD) == _lib.ERR_ALIGN


def test_bwd_topk_weights_arguments(lib):
    f = lib.mx8_moe_bwd_topk_weights
    assert f(None, P, None, P, 1, 8, 1, None) == _lib.ERR_ARG
    assert f(P, P, None, P, 0, 8, 1, None) == _lib.ERR_SIZE
    assert f(P, P, None, P, 1, 8, 524281, None) == _lib.ERR_LIMIT
    assert f(P, P, ODD, P, 1, 8, 1, None) == _lib.ERR_ALIGN
    assert f(P, P, None, P, 1, 2 ** 31 - 8, 1, None) == _lib.ERR_LIMIT


def test_quantize_block128_arguments(lib):
    def call(x=P, dtype=0, E=1, M=8, N=8, ldx=8, index=None, src=0, q=P, ld=16, sc=P, qt=None, ld_t=16, sct=None):
        return lib.mx8_quantize_block128(x, dtype, E, M, N, ldx, index, src, q, ld, sc, qt, ld_t, sct, 0, None)

    assert call(x=None) == _lib.ERR_ARG and call(q=None, sc=None) == _lib.ERR_ARG
    assert call(sc=None) == _lib.ERR_ARG and call(qt=P) == _lib.ERR_ARG and call(dtype=3) == _lib.ERR_ARG
    for bad in ({"M": 0}, {"N": 0}, {"E": 0}, {"ldx": 7}, {"ld": 7}, {"qt": P, "sct": P, "ld_t": 7}, {"index": P, "src": 0},
                {"index": P, "src": 4, "E": 2}):
        assert call(**bad) == _lib.ERR_SIZE, bad
    assert call(x=ODD, dtype=1) == _lib.ERR_ALIGN and call(sc=ODD) == _lib.ERR_ALIGN
    assert call(M=2 ** 31 - 1, N=2 ** 31 - 1, ldx=2 ** 31, ld=2 ** 31) == _lib.ERR_LIMIT
    assert call(N=2 ** 31 - 1, ldx=2 ** 31, ld=2 ** 31) == _lib.ERR_LIMIT


def test_gemm_block128_arguments(lib):
    def call(A=P, lda=128, Asc=P, ldsa=64, B=P, ldb=128, Bsc=P, ldsb=64, sq=1, C=P, ldc=64, M=64, N=64, K=128, cd=0, gr=None, G=0):
        return lib.mx8_gemm_block128(A, lda, Asc, ldsa, B, ldb, Bsc, ldsb, sq, C, ldc, M, N, K, cd, gr, G, None)

    assert call(A=None) == _lib.ERR_ARG and call(C=None) == _lib.ERR_ARG and call(cd=2) == _lib.ERR_ARG
    assert call(G=-1) == _lib.ERR_ARG and call(G=2) == _lib.ERR_ARG and call(G=2, gr=P, sq=0) == _lib.ERR_ARG
    for bad in ({"M": 0}, {"N": 0}, {"K": 0}, {"lda": 120}, {"ldb": 136}, {"lda": 112}, {"ldsa": 63}, {"sq": 0, "ldsb": 63}, {"ldc": 63}):
        assert call(**bad) == _lib.ERR_SIZE, bad
    assert call(G=257, gr=P) == _lib.ERR_LIMIT
    top, wide = 2 ** 31 - 1, 2 ** 31
    for huge in ({"M": top, "ldsa": wide}, {"N": top, "ldc": wide, "ldsb": wide}, {"K": top, "lda": wide, "ldb": wide}, {"G": 200, "gr": P, "N": 1 << 24, "ldc": wide}):
        assert call(**huge) == _lib.ERR_LIMIT, huge
    assert call(A=ODD) == _lib.ERR_ALIGN and call(Bsc=ODD) == _lib.ERR_ALIGN and call(C=ODD, cd=1) == _lib.ERR_ALIGN

    def wgrad(A=P, lda=256, ldsa=64, M=64, N=64, R=256, cd=1, gr=P, G=2):
        return lib.mx8_gemm_block128_wgrad(A, lda, P, ldsa, P, 256, P, 64, P, 64, M, N, R, cd, gr, G, None)

    assert wgrad(A=None) == _lib.ERR_ARG and wgrad(G=0) == _lib.ERR_ARG and wgrad(gr=None) == _lib.ERR_ARG
    assert wgrad(lda=250) == _lib.ERR_SIZE and wgrad(ldsa=10) == _lib.ERR_SIZE
    assert wgrad(G=300) == _lib.ERR_LIMIT


def test_no_device_means_error_not_fallback(lib):
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    none = (_lib.ERR_CUDA, _lib.ERR_UNSUPPORTED)
    assert lib.mx8_router_topk(P, 1, 8, 4, 8, 2, 1, None, P, P, P, P, P, P, P, P, 1 << 20, None) in none
    assert lib.mx8_quantize_block128(P, 0, 1, 8, 8, 8, None, 0, P, 16, P, None, 0, None, 0, None) in none
    assert lib.mx8_gemm_block128(P, 128, P, 64, P, 128, P, 64, 1, P, 64, 64, 64, 128, 0, None, 0, None) in none
    with pytest.raises(ValueError):
        mx8.router_topk(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError):
        mx8.quantize_block128(torch.zeros(4, 8))
    with pytest.raises(ValueError):
        mx8.gemm_block128(torch.zeros(4, 16, dtype=torch.float8_e4m3fn), *[torch.zeros(1)] * 4)
    with pytest.raises(ValueError):
        mx8.bwd_topk_weights(torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(8, 8, dtype=torch.bfloat16))


def test_bwd_epilogue_with_ids_arguments(lib):
    f = lib.mx8_moe_bwd_epilogue_ids
    assert f(None, None, P, P, 1, 8, 1, None) == _lib.ERR_ARG and f(None, P, P, None, 1, 8, 1, None) == _lib.ERR_ARG
    assert f(None, P, P, P, 0, 8, 1, None) == _lib.ERR_ARG and f(None, P, P, P, 1, 12, 1, None) == _lib.ERR_SHAPE
    assert f(None, P, ODD, P, 1, 8, 1, None) == _lib.ERR_ALIGN and f(ODD, P, None, P, 1, 8, 1, None) == _lib.ERR_ALIGN


def test_status_words_of_the_header_have_names(lib):
    import os
    import re
    hdr = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mx8.h")).read()
    words = {int(v) for v in re.findall(r"MX8_DEV_\w+\s*=\s*(\d+)", hdr)}
    assert words == set(_lib.DEV_WORDS) and {16, 17} <= words
    assert b"did not fit" in lib.mx8_strerror(_lib.ERR_DEVICE_TIMEOUT) and b"wait expired" in lib.mx8_strerror(_lib.ERR_DEVICE_TIMEOUT)
