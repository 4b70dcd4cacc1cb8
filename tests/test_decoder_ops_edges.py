"""Calls of the decoder block's operators (ops/decoder.py) at the edges of what they document: values that
change when they are rounded to 32 bits, ranges of the 16-bit types, limits of a launch, streams.

Oracles and tolerances as in test_decoder_ops.py, whose bounds are per element and worked out beforehand.
"""
import gc
import math

import pytest
import torch

from kube_gpu_stats_amd.ops import decoder
from test_decoder_ops import BF16, F16, F32, NORM_GRADS, close, norm_check, norm_inputs, z

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    yield torch.device("cuda", 0)
    gc.collect()
    torch.cuda.empty_cache()  # other modules measure the GPU's memory


@pytest.fixture
def launches(monkeypatch):
    """The entries that calls on CPU tensors would launch, with their argument blocks."""
    seen = []
    monkeypatch.setattr(decoder, "_on_gpu", lambda t, name: None)
    monkeypatch.setattr(decoder, "_here", lambda t, stream: True)
    monkeypatch.setattr(decoder, "_call", lambda entry, args, index: seen.append((entry, args)))
    return seen


# ------------------------------------------------------- add_norm: scales that are one in 32 bits

NEAR_ONE = [0.7 + 0.2 + 0.1, 1 + 1e-9, 1 - 2.0 ** -25, 1 + 2.0 ** -24]  # the last two: ties, rounded to even
NEXT_TO_ONE = [1 - 2.0 ** -24, 1 + 2.0 ** -23]


@pytest.mark.parametrize("scale", NEAR_ONE + NEXT_TO_ONE)
def test_scale_is_rounded_before_it_decides(launches, scale):
    """dbranch is a tensor of its own exactly where the kernels, which get 32 bits, write one."""
    x, w = z(4, 64), z(64)
    _, _, saved = decoder.add_norm_fwd(x, x, w, scale=scale)
    dr, db, *_ = decoder.add_norm_bwd(x, x, x, x, w, saved, scale=scale)
    entry, args = launches[-1]
    packed = decoder._ADD_NORM.unpack(args)
    assert entry == "kgs_add_norm_bwd"
    assert (packed[-2] == 1.0) == (scale in NEAR_ONE)
    assert (dr is db) == (packed[-2] == 1.0)


@gpu
@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("scale", NEAR_ONE + NEXT_TO_ONE)
def test_gradients_of_scales_next_to_one(dev, scale, t):
    a = norm_inputs(9, 200, t, dev, False, False, seed=3)
    want = norm_check(*a, scale=scale)[3]
    r, b = a[0].clone().requires_grad_(), a[1].clone().requires_grad_()
    torch.autograd.backward(decoder.add_norm(r, b, a[2], scale=scale, eps=1e-5), [a[5], a[6]])
    assert torch.equal(r.grad, want[0]) and torch.equal(b.grad, want[1])
