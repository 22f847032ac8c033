"""CPU: the polynomials for 2^x of the training kernels, with the coefficients of the sources and fp32 fused multiply-adds (a product of two fp32 numbers is
exact in 64 bits; its sum is rounded there once more than on the device, by 2^-29 of a step). The bounds are the ones that the sources state."""
import os
import re

import numpy as np

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensor-ffn_b200", "csrc")
F32, F64 = np.float32, np.float64


def coefficients(name, function):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    body = text[text.index(function):]
    body = body[body.index("{"):body.index("\n}\n")]
    at = body.index("y = ")
    return [F32(c) for c in re.findall(r"(\d+\.\d{6,}|(?<=f, )1\.)f[,;)]", re.sub(r"f2\((\S+)f, \S+f\)", r"\1f;", body[at:]))]


def polynomial(c, f):
    y = np.full_like(f, c[0])
    for a in c[1:]:
        y = (y.astype(F64) * f.astype(F64) + F64(a)).astype(F32)
    return y


def errors(name, function, degree):
    c = coefficients(name, function)
    assert len(c) == degree + 1 and abs(c[-1] - 1) < 1e-5 and abs(c[-2] - np.log(2)) < 1e-4, c
    f = np.linspace(-0.5, 0.5, 400001).astype(F32)
    exact = F64(0)
    for a in c:
        exact = exact * f.astype(F64) + F64(a)
    want = np.exp2(f.astype(F64))
    return np.abs(exact / want - 1).max(), (polynomial(c, f) / want - 1)


def test_joins_of_partial_sums():
    """train_loss.cu: exp2_exact"""
    fit, off = errors("train_loss.cu", "exp2_exact(float x)", 6)
    assert 1.5e-8 < fit < 1.7e-8
    assert 7.5e-8 < np.abs(off).max() < 8e-8
    assert abs(off.mean()) < 1e-8  # not to one side


def test_forward_exponentials():
    """train_attn.cuh: exp2_poly"""
    fit, off = errors("train_attn.cuh", "exp2_poly(F2 x)", 4)
    assert 2.5e-6 < fit < 2.75e-6
    assert np.abs(off).max() < 2.9e-6
