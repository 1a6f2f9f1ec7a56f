"""Argument checks of the vocabulary loss and the multi-adapter projection: all of them come before any
CUDA call, so they run without a GPU on made-up addresses."""
import pytest
import torch

from gemm_b200 import _lib

L = _lib.lib
P = 1 << 20            # an aligned address that nothing reads
BIG = 1 << 40
I, A, TL = _lib.ERR_INVALID_ARG, _lib.ERR_ALIGNMENT, _lib.ERR_TOO_LARGE


def xent(X=P, W=P, labels=P, loss=P, lse=P, T=4, V=100, D=64, ldx=64, ldw=64, scratch=P, nbytes=BIG):
    return L.gemm_b200_gemm_bf16_xent(X, W, labels, loss, lse, T, V, D, ldx, ldw, scratch, nbytes, None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=-1), I), (dict(V=0), I), (dict(D=0), I), (dict(ldx=56), I), (dict(ldw=56), I),
    (dict(X=None), I), (dict(W=None), I), (dict(labels=None), I), (dict(loss=None), I), (dict(lse=None), I),
    (dict(X=P + 2), A), (dict(W=P + 8), A), (dict(ldx=68), A), (dict(ldw=65), A),
    (dict(V=1 << 31), TL), (dict(T=1 << 31), TL),
    (dict(scratch=None), I), (dict(scratch=P + 16), I), (dict(nbytes=16), I),
])
def test_xent_refusals(kw, code):
    assert xent(**kw) == code
    assert _lib.last_error().startswith("gemm_bf16_xent")


def test_xent_of_no_tokens():
    assert xent(T=0, X=None, labels=None, loss=None, lse=None, scratch=None, nbytes=0) == _lib.OK


def xent_grad(X=P, W=P, labels=P, lse=P, gl=P, gls=1, gz=None, gzs=0, dX=P, dW=P, T=4, V=100, D=64, ldx=64, ldw=64, lddx=64, lddw=64,
              scratch=P, nbytes=BIG):
    return L.gemm_b200_gemm_bf16_xent_grad(X, W, labels, lse, gl, gls, gz, gzs, dX, dW, T, V, D, ldx, ldw, lddx, lddw, scratch, nbytes, None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=-1), I), (dict(V=0), I), (dict(D=0), I), (dict(lddx=56), I), (dict(lddw=56), I), (dict(gls=-1), I), (dict(gzs=-1), I),
    (dict(X=None), I), (dict(W=None), I), (dict(labels=None), I), (dict(lse=None), I), (dict(gl=None), I), (dict(dX=None), I), (dict(dW=None), I),
    (dict(D=60), A), (dict(dX=P + 2), A), (dict(dW=P + 8), A), (dict(lddx=68), A), (dict(lddw=68), A), (dict(V=1 << 31), TL),
])
def test_xent_grad_refusals(kw, code):
    assert xent_grad(**kw) == code
    assert _lib.last_error().startswith("gemm_bf16_xent_grad")


def lora(X=P, W=P, A=P, B=P, ids=P, scales=None, Y=P, T=4, N=128, D=64, R=16, n=2, ldx=64, ldw=64, lda=64, sa=16 * 64, ldb=128, sb=16 * 128,
         ldy=128, layout=1, od=0, scratch=P, nbytes=BIG):
    return L.gemm_b200_gemm_bf16_lora(X, W, A, B, ids, scales, Y, T, N, D, R, n, ldx, ldw, lda, sa, ldb, sb, ldy, layout, od, scratch, nbytes, None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=-1), I), (dict(N=0), I), (dict(D=0), I), (dict(R=0), I), (dict(n=0), I), (dict(layout=2), I), (dict(od=2), I),
    (dict(R=129, sa=129 * 64, sb=129 * 128), TL), (dict(ldx=56), I), (dict(ldw=56), I), (dict(lda=56), I), (dict(ldb=120), I), (dict(ldy=120), I),
    (dict(sa=15 * 64), I), (dict(sb=15 * 128), I), (dict(layout=0), I),    # W [D, N] needs ldw >= N
    (dict(N=124), A), (dict(D=60), A), (dict(lda=68, sa=16 * 68), A), (dict(ldb=132, sb=16 * 132), A), (dict(sa=16 * 64 + 4), A), (dict(ldx=68), A),
    (dict(ldw=68), A), (dict(ldy=132), A), (dict(ldy=130, od=1), A), (dict(n=1 << 31), TL),
    (dict(X=None), I), (dict(W=None), I), (dict(A=None), I), (dict(B=None), I), (dict(ids=None), I), (dict(Y=None), I),
    (dict(X=P + 2), A), (dict(W=P + 2), A), (dict(A=P + 2), A), (dict(B=P + 2), A), (dict(Y=P + 2), A),
])
def test_lora_refusals(kw, code):
    assert lora(**kw) == code
    assert _lib.last_error().startswith("gemm_bf16_lora")


def lora_grad(X=P, dY=P, A=P, B=P, ids=P, scales=None, dA=P, dB=P, T=4, N=128, D=64, R=16, n=2, ldx=64, lddy=128, lda=64, sa=16 * 64, ldb=128,
              sb=16 * 128, od=0, scratch=P, nbytes=BIG):
    return L.gemm_b200_gemm_bf16_lora_grad(X, dY, A, B, ids, scales, dA, dB, T, N, D, R, n, ldx, lddy, lda, sa, ldb, sb, od, scratch, nbytes, None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=-1), I), (dict(R=0), I), (dict(n=0), I), (dict(n=65536), TL), (dict(R=200), TL), (dict(lddy=120), I), (dict(lddy=132), A), (dict(od=-1), I),
    (dict(X=None), I), (dict(dY=None), I), (dict(A=None), I), (dict(B=None), I), (dict(ids=None), I), (dict(dA=None), I), (dict(dB=None), I),
    (dict(X=P + 2), A), (dict(dY=P + 2), A), (dict(dA=P + 2), A), (dict(dB=P + 2), A),
])
def test_lora_grad_refusals(kw, code):
    assert lora_grad(**kw) == code
    assert _lib.last_error().startswith("gemm_bf16_lora_grad")


def test_scratch_of_nothing_is_nothing():
    assert L.gemm_b200_gemm_bf16_xent_scratch_bytes(0, 100) == 0
    assert L.gemm_b200_gemm_bf16_xent_scratch_bytes(300, 1000) >= 4 * 300 * 8 + 300 * 4
    assert L.gemm_b200_gemm_bf16_xent_grad_scratch_bytes(0, 100, 64) == 0
    assert L.gemm_b200_gemm_bf16_lora_scratch_bytes(0, 64, 64, 8, 2, 0) == 0
    assert L.gemm_b200_gemm_bf16_lora_grad_scratch_bytes(4, 64, 64, 0, 2, 0) == 0


def test_the_python_operators_refuse_cpu_tensors():
    import gemm_b200 as g
    X, W = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16)
    lab = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        g.gemm_bf16_xent(X, W, lab)
    with pytest.raises(ValueError):
        g.gemm_bf16_xent_grad(X, W, lab, torch.zeros(4), torch.zeros(4))
    Ad, Bd = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 8, 104, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        g.gemm_bf16_lora(X, W, Ad, Bd, torch.zeros(4, dtype=torch.int32), b_is_nk=True)
    with pytest.raises(ValueError):
        g.gemm_bf16_lora_grad(X, torch.zeros(4, 104, dtype=torch.bfloat16), Ad, Bd, torch.zeros(4, dtype=torch.int32))
