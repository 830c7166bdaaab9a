"""Forward-mode derivatives: operators that carry none refuse tensors that have a
tangent, as they refuse those that require a gradient (nothing reaches a GPU)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from kquant_amd.grouped import int8_grouped_linear
from kquant_amd.linear import int8_linear, mxfp4_linear, mxfp8_linear
from kquant_amd.sampling import sample_tokens

BF16 = torch.bfloat16


def i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


def linear(**change):
    args = dict(source=torch.zeros(4, 64, dtype=BF16), weight=i8(24, 64), scale=torch.ones(24)) | change
    return int8_linear(**args)


def grouped(**change):
    args = dict(x=torch.zeros(4, 32, dtype=BF16), weight=i8(2, 24, 32), scale=torch.ones(2, 24),
                offsets=torch.zeros(3, dtype=torch.int64)) | change
    return int8_grouped_linear(**args)


def mx(**change):
    args = dict(source=torch.zeros(4, 64, dtype=BF16), activation="relu") | change
    return mxfp8_linear(weight=torch.zeros(24, 64, dtype=torch.uint8), scale=torch.zeros(24, 2, dtype=torch.uint8), **args)


def mx4(**change):
    args = dict(source=torch.zeros(4, 64, dtype=BF16), activation="relu") | change
    return mxfp4_linear(packed=torch.zeros(24, 32, dtype=torch.uint8), scale=torch.zeros(24, 2, dtype=torch.uint8), **args)


def sample(**change):
    return sample_tokens(uniform=torch.zeros(4), return_logprobs=True, **change)


CASES = [(linear, "source", torch.zeros(4, 64, dtype=BF16)), (linear, "scale", torch.ones(24)),
         (linear, "bias", torch.zeros(24)), (linear, "residual", torch.zeros(4, 24, dtype=BF16)),
         (grouped, "x", torch.zeros(4, 32, dtype=BF16)), (grouped, "scale", torch.ones(2, 24)),
         (mx, "source", torch.zeros(4, 64, dtype=BF16)), (mx, "bias", torch.zeros(24)),
         (mx4, "residual", torch.zeros(4, 24, dtype=BF16)), (sample, "logits", torch.zeros(4, 9))]


@pytest.mark.parametrize("recording", [True, False])
@pytest.mark.parametrize("call,name,value", CASES)
def test_tangents_are_refused(call, name, value, recording):
    """``no_grad`` leaves tangents in force."""
    with forward_ad.dual_level(), torch.set_grad_enabled(recording):
        dual = forward_ad.make_dual(value, torch.ones_like(value))
        with pytest.raises(RuntimeError, match="carries no gradient"):
            call(**{name: dual})


def test_rows_scales_and_jvp_are_refused():
    scale = torch.ones(4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(scale, torch.ones_like(scale))
        with pytest.raises(RuntimeError, match="carries no gradient"):
            linear(source=i8(4, 64), source_scale=dual)
        with pytest.raises(RuntimeError, match="carries no gradient"):
            grouped(x=i8(4, 32), x_scale=dual)
    logits = torch.zeros(4, 9)
    with pytest.raises(RuntimeError, match="carries no gradient"):
        torch.func.jvp(lambda z: sample(logits=z)[1], (logits,), (logits,))
