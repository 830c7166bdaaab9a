"""Arguments that the int8 products and the sampling refuse, before anything
reaches a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd.grouped import int8_grouped_linear
from kquant_amd.int8 import INT8_MAX_K, int8_dequantize, int8_quantize
from kquant_amd.linear import int8_linear
from kquant_amd.sampling import sample_tokens

BF16 = torch.bfloat16


def i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


@pytest.mark.parametrize("x,error,text", [
    (torch.zeros(4, 8, dtype=torch.float64), TypeError, "bfloat16, float16 or float32"),
    (i8(4, 8), TypeError, "bfloat16, float16 or float32"),
    (torch.zeros(()), ValueError, "feature dimension"),
    (torch.zeros(4, 0), ValueError, "feature dimension"),
])
def test_quantize(x, error, text):
    with pytest.raises(error, match=text):
        int8_quantize(x)


@pytest.mark.parametrize("q,scale,error,text", [
    (torch.zeros(4, 8), torch.zeros(4), TypeError, "int8 codes"),
    (i8(4, 8), torch.zeros(4, dtype=BF16), TypeError, "float32 scales"),
    (i8(4, 8), torch.zeros(3), ValueError, "scale shape"),
])
def test_dequantize(q, scale, error, text):
    with pytest.raises(error, match=text):
        int8_dequantize(q, scale)


LINEAR = [
    (dict(source=torch.zeros(4, 32, dtype=torch.float64)), TypeError, "rows must be int8"),
    (dict(source=i8(4, 32)), ValueError, "need their scales"),
    (dict(source=i8(4, 32), source_scale=torch.zeros(4, dtype=BF16)), TypeError, "scales must be float32"),
    (dict(source=i8(4, 32), source_scale=torch.zeros(5)), ValueError, "scales of the rows"),
    (dict(source_scale=torch.zeros(4)), ValueError, "belong to int8 rows"),
    (dict(w=torch.zeros(24, 32)), TypeError, "weight must be int8"),
    (dict(w=torch.zeros(24, 32, dtype=torch.uint8)), TypeError, "weight must be int8"),
    (dict(w=i8(24, 16)), ValueError, "with K=32"),
    (dict(w=i8(24, 32, 1)), ValueError, "with K=32"),
    (dict(scale=torch.zeros(24, dtype=BF16)), TypeError, "scales must be float32"),
    (dict(scale=torch.zeros(25)), ValueError, "scale shape"),
    (dict(scale=torch.zeros(1)), ValueError, "scale shape"),
    (dict(source=torch.zeros(2, INT8_MAX_K + 1, dtype=BF16), w=i8(24, INT8_MAX_K + 1)), ValueError, "between 1 and"),
    (dict(source=torch.zeros(2, 0), w=i8(24, 0)), ValueError, "between 1 and"),
    (dict(out_dtype=torch.int32), TypeError, "out_dtype"),
    (dict(activation="tanh"), ValueError, "activation"),
    (dict(bias=torch.zeros(24, dtype=torch.float16)), TypeError, "bias must be"),
    (dict(bias=torch.zeros(23)), ValueError, "bias shape"),
    (dict(residual=torch.zeros(4, 24)), TypeError, "residual must have"),
    (dict(residual=torch.zeros(4, 23, dtype=BF16)), ValueError, "residual shape"),
    (dict(source=torch.zeros(4, 32, dtype=BF16, requires_grad=True)), RuntimeError, "carries no gradient"),
    (dict(bias=torch.zeros(24, requires_grad=True)), RuntimeError, "carries no gradient"),
    (dict(scale=torch.zeros(24, requires_grad=True)), RuntimeError, "carries no gradient"),
    (dict(source=i8(4, 32), source_scale=torch.zeros(4, requires_grad=True)), RuntimeError, "carries no gradient"),
]


@pytest.mark.parametrize("change,error,text", LINEAR)
def test_linear(change, error, text):
    args = dict(source=torch.zeros(4, 32, dtype=BF16), w=i8(24, 32), scale=torch.zeros(24)) | change
    keywords = {name: v for name, v in args.items() if name not in ("source", "w", "scale")}
    with pytest.raises(error, match=text):
        int8_linear(args["source"], args["w"], args["scale"], **keywords)


@pytest.mark.parametrize("change,error,text", [
    (dict(x=torch.zeros(4, 32, dtype=torch.float64)), TypeError, "rows must be int8"),
    (dict(x=i8(4, 32)), ValueError, "need their scales"),
    (dict(x=torch.zeros(32, dtype=BF16)), ValueError, r"\[rows, K\]"),
    (dict(offsets=torch.zeros(3)), TypeError, "int64 or int32"),
    (dict(offsets=torch.zeros(2, dtype=torch.int64)), ValueError, "offsets shape"),
    (dict(w=i8(24, 32)), ValueError, r"\[groups, N, K\]"),
    (dict(w=i8(2, 20, 32), scale=torch.zeros(2, 20)), ValueError, "multiple of 8"),
    (dict(w=i8(0, 24, 32), scale=torch.zeros(0, 24), offsets=torch.zeros(1, dtype=torch.int64)), ValueError, "groups=0"),
    (dict(w=i8(4097, 8, 32), scale=torch.zeros(4097, 8), offsets=torch.zeros(4098, dtype=torch.int64)), ValueError,
     "groups=4097"),
    (dict(scale=torch.zeros(2, 23)), ValueError, "scale shape"),
    (dict(out_dtype=torch.int8), TypeError, "out_dtype"),
    (dict(x=torch.zeros(4, 32, dtype=BF16, requires_grad=True)), RuntimeError, "carries no gradient"),
    (dict(scale=torch.zeros(2, 24, requires_grad=True)), RuntimeError, "carries no gradient"),
])
def test_grouped(change, error, text):
    args = dict(x=torch.zeros(4, 32, dtype=BF16), w=i8(2, 24, 32), scale=torch.zeros(2, 24),
                offsets=torch.zeros(3, dtype=torch.int64)) | change
    keywords = {name: v for name, v in args.items() if name not in ("x", "w", "scale", "offsets")}
    with pytest.raises(error, match=text):
        int8_grouped_linear(args["x"], args["w"], args["scale"], args["offsets"], **keywords)


@pytest.mark.parametrize("change,error,text", [
    (dict(logits=torch.zeros(4, 9, dtype=torch.float64)), TypeError, "logits must be"),
    (dict(uniform=torch.zeros(4, dtype=torch.float64)), TypeError, "uniform must be float32"),
    (dict(uniform=torch.zeros(4, 1)), ValueError, "uniform has shape"),
    (dict(logits=torch.zeros(4, 0)), ValueError, "V between"),
    (dict(logits=torch.zeros(1, (1 << 18) + 1), uniform=torch.zeros(1)), ValueError, "V between"),
    (dict(logits=torch.zeros(()), uniform=torch.zeros(())), ValueError, "V between"),
    (dict(temperature=-1.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(temperature=float("inf")), ValueError, "temperature"),
    (dict(temperature=None), TypeError, "temperature"),
    (dict(temperature=torch.tensor(1.0)), TypeError, "for each row"),
    (dict(temperature=torch.ones(4, dtype=BF16)), TypeError, "must be float32"),
    (dict(temperature=torch.ones(3)), ValueError, "temperature has shape"),
    (dict(top_k=1.5), ValueError, "top_k"),
    (dict(top_k=torch.ones(4)), TypeError, "int32 or int64"),
    (dict(top_k=torch.ones(5, dtype=torch.int32)), ValueError, "top_k has shape"),
    (dict(top_p=0.0), ValueError, "top_p"),
    (dict(top_p=1.1), ValueError, "top_p"),
    (dict(top_p=torch.ones(4, dtype=torch.float64)), TypeError, "must be float32"),
    (dict(min_p=-0.1), ValueError, "min_p"),
    (dict(min_p=1.5), ValueError, "min_p"),
    (dict(logits=torch.zeros(4, 9, requires_grad=True), return_logprobs=True), RuntimeError, "carries no gradient"),
])
def test_sample(change, error, text):
    args = dict(logits=torch.zeros(4, 9), uniform=torch.zeros(4)) | change
    keywords = {name: v for name, v in args.items() if name not in ("logits", "uniform")}
    with pytest.raises(error, match=text):
        sample_tokens(args["logits"], args["uniform"], **keywords)


def refused(fn, ok, cases):
    lib = N.library()
    for at, value, status, text in cases:
        args = list(ok)
        args[at] = value
        assert getattr(lib, fn)(*args) == status and text in lib.kq_last_error(), (at, value, lib.kq_last_error())


P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(257)  # never read: validation fails first
INVALID, LIMIT = N.KQ_ERR_INVALID, N.KQ_ERR_LIMIT


def test_quantize_c_entry():
    ok = [N.DT_BF16, P, 64, 10, 64, P, 64, P, None]
    refused("kq_int8_quantize", ok, [
        (0, N.DT_I8, INVALID, b"dtype"), (2, 63, INVALID, b"row strides"), (3, -1, INVALID, b"rows >= 0"),
        (4, 0, INVALID, b"k >= 1"), (6, 63, INVALID, b"row strides"), (1, None, INVALID, b"null"), (5, None, INVALID, b"null"),
        (7, None, INVALID, b"null"), (1, ODD, INVALID, b"aligned"), (7, ctypes.c_void_p(258), INVALID, b"aligned"),
        (3, 1 << 31, LIMIT, b"2^30")])


def test_linear_c_entry():
    ok = [N.DT_I8, P, 64, P, P, P, 10, 24, 64, 0, None, N.DT_BF16, None, 24, N.DT_BF16, P, 24, None, 0, None]
    refused("kq_int8_linear", ok, [
        (0, 9, INVALID, b"input dtype"), (2, 48, INVALID, b"lda >= k"), (2, 72, INVALID, b"multiple of 16"),
        (3, None, INVALID, b"null"), (4, None, INVALID, b"null"), (5, None, INVALID, b"null"), (15, None, INVALID, b"null"),
        (8, 56, INVALID, b"k % 16"), (8, 0, INVALID, b"k % 16"), (9, 5, INVALID, b"activation"), (14, N.DT_I8, INVALID, b"output"),
        (16, 23, INVALID, b"ldc"), (1, ctypes.c_void_p(264), INVALID, b"16-byte"), (4, ctypes.c_void_p(264), INVALID, b"16-byte"),
        (2, (1 << 22) + 16, LIMIT, b"2^22"), (6, 1 << 31, LIMIT, b"2^30")])
    wide = list(ok)
    wide[7] = wide[13] = wide[16] = (1 << 26) + 8
    refused("kq_int8_linear", wide, [(9, 0, LIMIT, b"2^26")])
    long = list(ok)
    long[2] = long[8] = INT8_MAX_K + 16
    refused("kq_int8_linear", long, [(9, 0, LIMIT, b"131056")])
    rows = list(ok)
    rows[0], rows[3] = N.DT_BF16, None
    refused("kq_int8_linear", rows, [(9, 0, INVALID, b"workspace needs")])
    biased = list(ok)
    biased[10] = P
    refused("kq_int8_linear", biased, [(11, N.DT_F16, INVALID, b"bias dtype")])
    added = list(ok)
    added[12] = P
    refused("kq_int8_linear", added, [(13, 23, INVALID, b"ldr >= n")])
    lib = N.library()
    assert lib.kq_int8_linear_workspace_size(N.DT_I8, 100, 24, 64) == 0
    assert lib.kq_int8_linear_workspace_size(N.DT_BF16, 100, 24, 64) >= 100 * 68
    assert lib.kq_int8_linear_workspace_size(N.DT_BF16, -1, 24, 64) == -1


def test_grouped_c_entry():
    ok = [P, 64, P, 10, P, 3, P, P, 32, 64, N.DT_BF16, P, 32, None]
    refused("kq_int8_grouped_linear", ok, [
        (10, 7, INVALID, b"output dtype"), (1, 48, INVALID, b"strides"), (1, 72, INVALID, b"multiples of 16"), (3, -1, INVALID, b"groups"),
        (5, 0, INVALID, b"groups >= 1"), (8, 30, INVALID, b"n % 8"), (9, 56, INVALID, b"k % 16"), (12, 24, INVALID, b"strides"),
        (4, None, INVALID, b"offsets"), (4, ctypes.c_void_p(260), INVALID, b"offsets"), (0, ctypes.c_void_p(264), INVALID, b"16-byte"),
        (11, ctypes.c_void_p(264), INVALID, b"16-byte"), (2, None, INVALID, b"null"), (7, None, INVALID, b"null"),
        (5, 4097, LIMIT, b"4096"), (3, 1 << 31, LIMIT, b"2^30"), (1, 1 << 23, LIMIT, b"2^22")])


def test_sample_c_entry():
    ok = [N.DT_F32, P, 100, 4, 100, P, None, 1.0, None, 0, None, 1.0, None, 0.0, P, None, None, 0, None]
    cases = [(0, N.DT_I8, INVALID, b"dtype"), (2, 99, INVALID, b"row stride"), (3, -1, INVALID, b"rows >= 0"),
             (4, 0, INVALID, b"vocab >= 1"), (1, None, INVALID, b"null"), (5, None, INVALID, b"null"), (14, None, INVALID, b"null"),
             (1, ODD, INVALID, b"aligned"), (6, ODD, INVALID, b"aligned"), (8, ODD, INVALID, b"aligned"), (10, ODD, INVALID, b"aligned"),
             (12, ODD, INVALID, b"aligned"), (14, ctypes.c_void_p(260), INVALID, b"aligned"), (15, ODD, INVALID, b"aligned")]
    refused("kq_sample_tokens", ok, cases)
    wide = list(ok)
    wide[2] = wide[4] = (1 << 18) + 1
    refused("kq_sample_tokens", wide, [(3, 4, LIMIT, b"262144"), (3, (1 << 20) + 1, LIMIT, b"2^20 rows")])
    wide[2] = wide[4] = 50257
    lib = N.library()
    small, large = (lib.kq_sample_tokens_workspace_size(4, 50257, f) for f in (0, 1))
    assert 0 < small < large and lib.kq_sample_tokens_workspace_size(4, 100, 1) == 0
    wide[16], wide[17] = P, small
    refused("kq_sample_tokens", wide, [(9, 5, INVALID, b"workspace needs"), (11, 0.5, INVALID, b"workspace needs"),
                                       (17, small - 1, INVALID, b"workspace needs"), (16, ODD, INVALID, b"aligned")])
