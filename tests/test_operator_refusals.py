"""Arguments that the grouped products, the head loss and the linears'
epilogues refuse, before anything reaches a GPU."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd import grouped
from kquant_amd import loss as loss_module
from kquant_amd.grouped import grouped_linear
from kquant_amd.linear import mxfp4_linear, mxfp8_linear
from kquant_amd.loss import linear_cross_entropy

BF16 = torch.bfloat16


def bf16(*shape):
    return torch.zeros(*shape, dtype=BF16)


@pytest.mark.parametrize("change,error,text", [
    (dict(x=torch.zeros(4, 16)), TypeError, "bfloat16 or both float16"),
    (dict(w=torch.zeros(2, 8, 16, dtype=torch.float16)), TypeError, "both"),
    (dict(offsets=torch.zeros(3)), TypeError, "int64 or int32"),
    (dict(x=bf16(4)), ValueError, r"\[rows, K\]"),
    (dict(w=bf16(8, 16)), ValueError, r"\[groups, N, K\]"),
    (dict(x=bf16(4, 24)), ValueError, "expects K=16"),
    (dict(w=bf16(2, 9, 16)), ValueError, "multiples of 8"),
    (dict(x=bf16(4, 12), w=bf16(2, 8, 12)), ValueError, "multiples of 8"),
    (dict(w=bf16(2, 0, 16)), ValueError, "multiples of 8"),
    (dict(w=bf16(0, 8, 16), offsets=torch.zeros(1, dtype=torch.int64)), ValueError, "groups=0"),
    (dict(w=bf16(4097, 8, 16), offsets=torch.zeros(4098, dtype=torch.int64)), ValueError, "groups=4097"),
    (dict(offsets=torch.zeros(2, dtype=torch.int64)), ValueError, "offsets shape"),
])
def test_grouped_linear(change, error, text):
    args = dict(x=bf16(4, 16), w=bf16(2, 8, 16), offsets=torch.zeros(3, dtype=torch.int64)) | change
    with pytest.raises(error, match=text):
        grouped_linear(args["x"], args["w"], args["offsets"])


def test_grouped_c_entries():
    lib = N.library()
    p = ctypes.c_void_p(256)  # never read: validation fails first
    ok = [N.DT_BF16, p, 64, 10, p, 3, p, 32, 64, p, 32, None]
    for at, value, text in ((0, N.DT_F32, b"bf16 or f16"), (2, 56, b"strides"), (2, 68, b"multiples of 8"), (3, -1, b"groups"),
                            (5, 0, b"groups >= 1"), (7, 30, b"n % 8"), (8, 60, b"k % 8"), (10, 24, b"strides"),
                            (4, None, b"offsets"), (1, ctypes.c_void_p(264), b"16-byte"), (6, ctypes.c_void_p(8), b"16-byte"),
                            (9, ctypes.c_void_p(2), b"16-byte")):
        args = list(ok)
        args[at] = value
        assert lib.kq_grouped_linear(*args) == N.KQ_ERR_INVALID and text in lib.kq_last_error(), (at, lib.kq_last_error())
    for at, value in ((5, 4097), (2, 1 << 23), (3, 1 << 31)):
        args = list(ok)
        args[at] = value
        assert lib.kq_grouped_linear(*args) == N.KQ_ERR_LIMIT
    dx = list(ok)
    dx[2], dx[10] = 24, 64
    assert lib.kq_grouped_linear_dx(*dx) == N.KQ_ERR_INVALID
    dw = [N.DT_BF16, p, 32, p, 24, 10, p, 3, 32, 64, p, None]
    assert lib.kq_grouped_linear_dw(*dw) == N.KQ_ERR_INVALID and b"strides" in lib.kq_last_error()


@pytest.mark.parametrize("change,error,text", [
    (dict(reduction="max"), ValueError, "reduction"),
    (dict(h=torch.zeros(4, 64)), TypeError, "hidden must be bfloat16"),
    (dict(h=torch.zeros(4, 64, dtype=torch.float16)), TypeError, "hidden must be bfloat16"),
    (dict(target=torch.zeros(4, dtype=torch.int32)), TypeError, "int64"),
    (dict(target=torch.zeros(5, dtype=torch.int64)), ValueError, "target shape"),
    (dict(w=torch.zeros(9, 64)), TypeError, "without scales must be bfloat16"),
    (dict(w=bf16(9, 32)), ValueError, "does not match K=64"),
    (dict(w=bf16(0, 64)), ValueError, "does not match"),
    (dict(w=bf16(64)), ValueError, r"\[V, K\]"),
    (dict(h=bf16(4, 60), w=bf16(9, 60)), ValueError, "multiple of 8"),
    (dict(scale=torch.zeros(9, 2, dtype=torch.uint8)), TypeError, "block-scaled head"),
    (dict(w=torch.zeros(9, 64, dtype=torch.uint8), scale=torch.zeros(9, 2)), TypeError, "E8M0"),
    (dict(w=torch.zeros(9, 64, dtype=torch.uint8), scale=torch.zeros(9, 3, dtype=torch.uint8)), ValueError, "scale shape"),
    (dict(w=torch.zeros(9, 48, dtype=torch.uint8), scale=torch.zeros(9, 2, dtype=torch.uint8)), ValueError, "does not match"),
    (dict(h=bf16(4, 32), w=torch.zeros(9, 32, dtype=torch.uint8), scale=torch.zeros(9, 1, dtype=torch.uint8)), ValueError,
     "multiple of 64"),
])
def test_linear_cross_entropy(change, error, text):
    args = dict(h=bf16(4, 64), w=bf16(9, 64), target=torch.zeros(4, dtype=torch.int64), scale=None, reduction="mean") | change
    with pytest.raises(error, match=text):
        linear_cross_entropy(args["h"], args["w"], args["target"], args["scale"], reduction=args["reduction"])


def test_loss_c_entries():
    lib = N.library()
    p = ctypes.c_void_p(256)
    ok = [N.FMT_BF16, p, 64, 10, p, None, 99, 64, p, -100, p, p, p, p, 1 << 30, None]
    for at, value, text in ((0, 7, b"head format"), (2, 56, b"ldh >= k"), (2, 68, b"ldh % 8"), (3, -1, b"tokens=-1"),
                            (6, 0, b"vocab >= 1"), (7, 60, b"k % 8"), (1, ctypes.c_void_p(264), b"16-byte"),
                            (0, N.FMT_MXFP8_E4M3, b"needs its scales")):
        args = list(ok)
        args[at] = value
        assert lib.kq_linear_cross_entropy(*args) == N.KQ_ERR_INVALID and text in lib.kq_last_error(), (at, lib.kq_last_error())
    for at, value in ((3, (1 << 20) + 1), (6, (1 << 24) + 1)):
        args = list(ok)
        args[at] = value
        assert lib.kq_linear_cross_entropy(*args) == N.KQ_ERR_LIMIT
    back = [N.FMT_MXFP8_E4M3, p, 64, 10, p, p, 99, 64, p, -100, p, p, N.LOSS_MEAN, p, 64, p, p, 1 << 30, None]
    assert lib.kq_linear_cross_entropy_backward(*back) == N.KQ_ERR_INVALID and b"only a bf16 head" in lib.kq_last_error()
    back[0], back[5], back[12] = N.FMT_BF16, None, 3
    assert lib.kq_linear_cross_entropy_backward(*back) == N.KQ_ERR_INVALID and b"reduction" in lib.kq_last_error()
    back[12], back[14] = N.LOSS_SUM, 56
    assert lib.kq_linear_cross_entropy_backward(*back) == N.KQ_ERR_INVALID and b"lddh" in lib.kq_last_error()
    size = lib.kq_linear_cross_entropy_workspace_size
    assert size(N.FMT_BF16, -1, 10, 64, 0) == -1 and size(N.FMT_BF16, 10, 0, 64, 0) == -1
    assert size(N.FMT_BF16, 0, 10, 64, 0) > 0 and size(N.FMT_BF16, 0, 10, 64, 1) > 0
    # no [tokens, vocabulary] array forward; at most 1 GiB of it backward
    assert size(N.FMT_BF16, 4096, 131072, 4096, 0) < 4096 * 131072 // 4
    assert size(N.FMT_BF16, 16384, 131072, 64, 1) < (1 << 30) + (1 << 28)


@pytest.mark.parametrize("change,error,text", [
    (dict(activation="tanh"), ValueError, "activation"),
    (dict(bias=torch.zeros(9, dtype=torch.float16)), TypeError, "bias must be"),
    (dict(bias=torch.zeros(8)), ValueError, "bias shape"),
    (dict(residual=torch.zeros(4, 9)), TypeError, "result's type"),
    (dict(residual=bf16(4, 8)), ValueError, "residual shape"),
    (dict(source=torch.zeros(4, 64), activation="relu", out_dtype=BF16), TypeError, "float32 result"),
])
def test_linear_epilogue(change, error, text):
    args = dict(source=bf16(4, 64), bias=None, activation=None, residual=None, out_dtype=None) | change
    source = args.pop("source")
    scale = torch.zeros(9, 2, dtype=torch.uint8)
    with pytest.raises(error, match=text):
        mxfp8_linear(source, torch.zeros(9, 64, dtype=torch.uint8), scale, **args)
    with pytest.raises(error, match=text):
        mxfp4_linear(source, torch.zeros(9, 32, dtype=torch.uint8), scale, **args)


def test_linear_epilogue_c_entry():
    lib = N.library()
    p = ctypes.c_void_p(256)
    ok = [N.FMT_MXFP8_E4M3, N.DT_BF16, p, 64, p, p, 4, 9, 64, 0, p, N.DT_F32, p, 9, N.DT_BF16, p, 9, None, 0, None]
    for at, value, text in ((0, N.FMT_BF16, b"weight format"), (1, N.DT_F16, b"input dtype"), (1, N.DT_F32, b"f32 results"),
                            (9, 5, b"activation 5"), (9, -1, b"activation"), (11, N.DT_F16, b"bias dtype"), (13, 8, b"ldr >= n"),
                            (14, N.DT_F16, b"output dtype"), (10, ctypes.c_void_p(2), b"aligned to their type"),
                            (12, ctypes.c_void_p(1), b"aligned to their type"), (16, 8, b"ldc >= n"), (8, 60, b"k % 64")):
        args = list(ok)
        args[at] = value
        assert lib.kq_mx_linear_epilogue(*args) == N.KQ_ERR_INVALID and text in lib.kq_last_error(), (at, lib.kq_last_error())


def test_loss_scale_alignment():
    lib = N.library()
    p = ctypes.c_void_p(256)
    for fmt in (N.FMT_MXFP8_E4M3, N.FMT_MXFP4_E2M1):
        args = [fmt, p, 128, 10, p, ctypes.c_void_p(258), 99, 128, p, -100, p, p, p, p, 1 << 30, None]
        assert lib.kq_linear_cross_entropy(*args) == N.KQ_ERR_INVALID and b"scales 4" in lib.kq_last_error()


def test_capture_beside_a_living_graph(monkeypatch):
    """A leaf whose accumulator belongs to another stream is refused in a capture, and only there."""
    leaf, other = torch.zeros(3, requires_grad=True), torch.zeros(2, 3, requires_grad=True)
    state = {"stream": 7, "capturing": False}
    monkeypatch.setattr(N, "stream_handle", lambda device: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    N.note_leaves(torch.zeros(3))
    kept = leaf * 1.0, other.reshape(6) * 1.0  # a leaf, and one behind a view
    for t in kept:
        N.note_leaves(t)
    N.check_capture(leaf, other)
    state["stream"] = 8
    N.check_capture(leaf, other)
    state["capturing"] = True
    for t in (leaf, other):
        with pytest.raises(RuntimeError, match="still lives"):
            N.check_capture(torch.zeros(3), t)
        with torch.no_grad():
            N.check_capture(t)
    N.check_capture(leaf * 2, torch.zeros(3))
    del kept, t
    N.check_capture(leaf, other)


@pytest.mark.parametrize("reduction,value", [(N.LOSS_MEAN, 5.0), (N.LOSS_SUM, 3.0)])
def test_reduced_loss_is_no_view(monkeypatch, reduction, value):
    """The scalar may be changed in place (loss /= steps), as a loss accumulated over batches is; the kernels are stood in for."""
    sums = torch.tensor([3.0, 5.0])

    def call(name, *args):
        if name == "kq_linear_cross_entropy":
            ctypes.memmove(args[12], sums.data_ptr(), 8)
        else:
            up, dh = ctypes.cast(args[11], ctypes.POINTER(ctypes.c_float)), args[13]
            seen.append(up[0])
            ctypes.memset(dh, 0, 4 * 64 * 2)

    seen = []
    monkeypatch.setattr(N, "call", call)
    monkeypatch.setattr(N, "stream", lambda device: None)
    monkeypatch.setattr(N, "on_device", lambda device: contextlib.nullcontext())
    h = bf16(4, 64).requires_grad_()
    loss = loss_module._LinearCrossEntropy.apply(h, bf16(9, 64), None, torch.zeros(4, dtype=torch.int64), N.FMT_BF16, -100,
                                                 reduction)
    assert loss.shape == () and loss.item() == value and not loss._is_view()
    loss /= 4
    loss += 1
    loss.backward()
    assert loss.item() == value / 4 + 1 and seen == [0.25] and h.grad.shape == (4, 64)


@pytest.mark.parametrize("which", ["source", "bias", "residual", "skip"])
def test_linear_epilogue_drops_no_gradient(monkeypatch, which):
    """Inputs that require a gradient are refused while autograd records, and only then."""
    reached = RuntimeError("reached the GPU")

    def to_gpu(tensors):
        raise reached

    monkeypatch.setattr(N, "to_gpu", to_gpu)
    source, bias, residual = bf16(4, 64), torch.zeros(64), bf16(4, 64)
    if which == "skip":
        residual = source
    {"source": source, "bias": bias, "residual": residual, "skip": source}[which].requires_grad_()
    for f, q in ((mxfp8_linear, torch.zeros(64, 64, dtype=torch.uint8)), (mxfp4_linear, torch.zeros(64, 32, dtype=torch.uint8))):
        scale = torch.zeros(64, 2, dtype=torch.uint8)
        with pytest.raises(RuntimeError, match="carries no gradient"):
            f(source, q, scale, bias=bias, activation="silu", residual=residual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="reached the GPU"):
            f(source, q, scale, bias=bias, activation="silu", residual=residual)
        with pytest.raises(RuntimeError, match="reached the GPU"):
            f(source.detach(), q, scale, bias=bias.detach(), residual=residual.detach())
        with pytest.raises(RuntimeError, match="reached the GPU"):
            f(source, q, scale)  # the linear without an epilogue takes any source, as it always has


@pytest.mark.parametrize("tokens", [1 << 19, (1 << 19) + 8, 600_001, 1 << 20])
def test_loss_workspace_of_many_tokens(tokens):
    """At most 1 GiB of softmax gradients at once up to the most tokens; K = 8, so that little else counts: the rows
    (16 bytes), dh's planes (32 each, two at most of so few steps), 24 bytes a token."""
    size = N.library().kq_linear_cross_entropy_workspace_size
    for vocab in (131072, 1 << 24):
        assert size(N.FMT_BF16, tokens, vocab, 8, 1) <= (1 << 30) + tokens * (16 + 64 + 24) + 4096


def test_grouped_rows_far_apart(monkeypatch):
    """Rows further apart than the kernels' strides reach are copied, not refused."""
    strides = []
    monkeypatch.setattr(N, "call", lambda name, *args: strides.append(args[2]))
    monkeypatch.setattr(N, "stream", lambda device: None)
    monkeypatch.setattr(N, "on_device", lambda device: contextlib.nullcontext())
    w, offsets = bf16(1, 8, 16), torch.tensor([0, 2])
    for stride in (16, grouped.MAX_STRIDE, grouped.MAX_STRIDE + 8):
        x = torch.empty(stride + 16, dtype=BF16).as_strided((2, 16), (stride, 1))
        grouped._GroupedLinear.apply(x, w, offsets)
    assert strides == [16, grouped.MAX_STRIDE, 16]


def test_capture_of_views_beside_a_living_graph(monkeypatch):
    """Leaves behind several views, in the graph that lives and in the capture."""
    state = {"stream": 7, "capturing": False}
    monkeypatch.setattr(N, "stream_handle", lambda device: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    direct, viewed = torch.zeros(6, 4, requires_grad=True), torch.zeros(6, 4, requires_grad=True)
    kept = direct * 1.0, viewed.view(2, 3, 4).transpose(1, 2).contiguous() * 1.0
    for t in kept:
        N.note_leaves(t)
    state.update(stream=8, capturing=True)
    for leaf in (direct, viewed):
        for t in (leaf, leaf.view(2, 3, 4), leaf.view(2, 3, 4).transpose(1, 2), leaf[1:3]):
            with pytest.raises(RuntimeError, match="still lives"):
                N.check_capture(torch.zeros(3), t)
        N.check_capture(leaf.detach().view(2, 12), torch.zeros(3))
    del kept, t
    N.check_capture(direct.view(2, 12), viewed[1:])


def test_no_row_stride_without_rows():
    """A caller that asks for dw alone has no row stride of dh to give (refused here for the workspace at the latest)."""
    lib = N.library()
    p = ctypes.c_void_p(256)
    back = [N.FMT_BF16, p, 64, 10, p, None, 99, 64, p, -100, p, p, N.LOSS_SUM, None, 0, p, None, 0, None]
    assert lib.kq_linear_cross_entropy_backward(*back) != N.KQ_OK and b"lddh" not in lib.kq_last_error()
    back[13] = p
    assert lib.kq_linear_cross_entropy_backward(*back) == N.KQ_ERR_INVALID and b"lddh" in lib.kq_last_error()


def test_capture_of_a_leaf_that_is_a_view(monkeypatch):
    """A leaf made of part of a tensor that needs no gradient is a leaf of its own."""
    state = {"stream": 7, "capturing": False}
    monkeypatch.setattr(N, "stream_handle", lambda device: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    leaf = torch.zeros(8, 4)[2:6].requires_grad_()
    assert leaf.is_leaf and leaf._base is not None
    kept = leaf * 1.0
    N.note_leaves(kept)
    state.update(stream=8, capturing=True)
    for t in (leaf, leaf.view(2, 8)):
        with pytest.raises(RuntimeError, match="still lives"):
            N.check_capture(t)
    del kept, t
    N.check_capture(leaf)
