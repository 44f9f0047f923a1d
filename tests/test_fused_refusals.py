"""Argument checks of the products around a transformer block. None of these calls gets as far as a device."""
import pytest

import clblast_b200 as cb

S = cb.StatusCode
ROW, NO, YES = 101, 111, 112


def epilogue(dtype=16, c_dtype=None, layout=ROW, ta=NO, tb=YES, m=8, n=16, k=24, lda=24, ldb=24, act=161):
    return cb.GemmEpilogue(layout, ta, tb, m, n, k, 1.0, 0, 0, lda, 0, 0, ldb, None, 0, act, None, 0, 16, 0.0, None, 0, 16, 0, 0, 16,
                           precision=dtype, c_precision=c_dtype)


def test_epilogue_refusals():
    assert epilogue(dtype=64) == S.kNotImplemented
    assert epilogue(dtype=3232) == S.kNotImplemented
    assert epilogue(dtype=16, c_dtype=1016) == S.kNotImplemented
    assert epilogue(dtype=32, c_dtype=16) == S.kNotImplemented
    assert epilogue(dtype=7) == S.kUnexpectedError
    assert epilogue(layout=0) == S.kUnexpectedError
    assert epilogue(ta=0) == S.kUnexpectedError
    assert epilogue(act=160) == S.kUnexpectedError
    assert epilogue(m=0) == S.kInvalidDimension
    assert epilogue(n=2 ** 31) == S.kInvalidDimension
    assert epilogue(k=0) == S.kInvalidDimension
    assert epilogue(lda=23) == S.kInvalidLeadDimA
    assert epilogue() == S.kInvalidMatrixA
    for dtype in (16, 1016, 32):
        assert epilogue(dtype=dtype) == S.kInvalidMatrixA


def test_epilogue_grad_refusals():
    def f(dtype=16, act=161, m=8):
        return cb.GemmEpilogueGrad(ROW, NO, NO, m, 16, 24, 1.0, 0, 0, 24, 0, 0, 16, 0.0, None, 0, 16, act, None, 0, 16, 0, 0, 16, None, 0,
                                   precision=dtype)
    assert f(dtype=64) == S.kNotImplemented
    assert f(act=166) == S.kUnexpectedError
    assert f(m=0) == S.kInvalidDimension
    assert f() == S.kInvalidMatrixA


def test_activation_grad_refusals():
    def f(dtype=16, rows=8, n=16, act=161, dz=0, groups=0, offsets=None, ld=16):
        return cb.ActivationGrad(rows, n, act, 4096, 0, ld, None, 0, 16, dz, 0, 16, None, 0, groups=groups, group_offsets=offsets,
                                 precision=dtype)
    assert f(dtype=64) == S.kNotImplemented
    assert f(act=0) == S.kUnexpectedError
    assert f(rows=0) == S.kInvalidDimension
    assert f(dz=0) == S.kInvalidMatrixC       # neither result
    assert f(groups=3) == S.kInvalidBatchCount
    assert f(offsets=4096) == S.kInvalidBatchCount
    assert f(groups=1025, offsets=4096) == S.kInvalidBatchCount
    assert f(dz=4096, ld=15) == S.kInvalidLeadDimA


def test_grouped_refusals():
    def f(dtype=16, c_dtype=None, trans=YES, groups=3, rows=8, n=16, k=24, ldx=24):
        return cb.GemmGrouped(trans, groups, rows, n, k, 1.0, 0, 0, ldx, 0, 0, 24, 384, 0, None, 0, 16, 161, None, 0, 16, 0.0, None, 0, 16,
                              0, 0, 16, precision=dtype, c_precision=c_dtype)
    assert f(dtype=32) == S.kNotImplemented
    assert f(c_dtype=1016) == S.kNotImplemented
    assert f(trans=1) == S.kUnexpectedError
    assert f(groups=0) == S.kInvalidBatchCount
    assert f(groups=1025) == S.kInvalidBatchCount
    assert f(rows=0) == S.kInvalidDimension
    assert f(ldx=23) == S.kInvalidLeadDimA
    assert f() == S.kInvalidMatrixA
    g = lambda groups: cb.GemmGroupedGrad(NO, groups, 8, 16, 24, 1.0, 0, 0, 24, 0, 0, 16, 384, 0, 0.0, None, 0, 16, 161, None, 0, 16, 0, 0,
                                          16, None, 0, 16, precision=16)
    assert g(0) == S.kInvalidBatchCount and g(2) == S.kInvalidMatrixA
    w = lambda m, dtype=16: cb.GemmGroupedWeight(2, 8, m, 16, 1.0, 0, 0, 24, 0, 0, 16, 0, 0.0, 0, 0, 16, 384, precision=dtype)
    assert w(0) == S.kInvalidDimension and w(25) == S.kInvalidLeadDimA and w(24) == S.kInvalidMatrixA
    assert w(24, 32) == S.kNotImplemented


def test_newton_schulz_refusals():
    def f(dtype=16, layout=ROW, m=8, n=16, batch=1, steps=5, ld=16, **kw):
        return cb.NewtonSchulz(layout, m, n, 1.0, 0, 0, ld, 128, 0, 0, 16, 128, batch, steps=steps, precision=dtype, **kw)
    assert f(dtype=64) == S.kNotImplemented
    assert f(layout=1) == S.kUnexpectedError
    assert f(batch=0) == S.kInvalidBatchCount
    assert f(batch=65536) == S.kInvalidBatchCount
    assert f(m=0) == S.kInvalidDimension
    assert f(steps=0) == S.kInvalidDimension
    assert f(steps=5, coefficients=[(1.0, 0.0, 0.0)] * 4) == S.kInvalidDimension
    assert f(epsilon=-1.0) == S.kInvalidDimension
    assert f(epsilon=float("nan")) == S.kInvalidDimension
    assert f(ld=15) == S.kInvalidLeadDimA
    assert f() == S.kInvalidMatrixA


def test_types_of_tensors():
    import torch
    half, single, offsets = torch.zeros(4, dtype=torch.float16), torch.zeros(4), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):  # B is not half
        cb.GemmEpilogue(ROW, NO, NO, 2, 2, 2, 1.0, 0, 0, 2, single, 0, 2, None, 0, 161, None, 0, 2, 0.0, None, 0, 2, 0, 0, 2, precision=16)
    with pytest.raises(TypeError):  # no precision for raw pointers
        cb.GemmEpilogue(ROW, NO, NO, 2, 2, 2, 1.0, 0, 0, 2, 0, 0, 2, None, 0, 161, None, 0, 2, 0.0, None, 0, 2, 0, 0, 2)
    with pytest.raises(TypeError):  # offsets are 64-bit
        cb.GemmGrouped(YES, 1, 2, 2, 2, 1.0, 0, 0, 2, 0, 0, 2, 4, offsets, None, 0, 2, 161, None, 0, 2, 0.0, None, 0, 2, 0, 0, 2, precision=16)
    with pytest.raises(ValueError):  # host memory
        cb.GemmEpilogue(ROW, NO, NO, 2, 2, 2, 1.0, half, 0, 2, half, 0, 2, None, 0, 161, None, 0, 2, 0.0, None, 0, 2, half, 0, 2)
    # the reference's routines do not know bfloat16
    with pytest.raises(TypeError):
        b = torch.zeros(4, dtype=torch.bfloat16)
        cb.Gemm(ROW, NO, NO, 2, 2, 2, 1.0, b, 0, 2, b, 0, 2, 0.0, b, 0, 2)
