"""Fused decode and draft steps: weights that are replaced, and draft steps from equal roots."""
import pytest
import torch

from ananta_ocr_b200 import moe, norms
from test_fused_steps_gpu import make, plain_add, plain_moe, plain_norm, start

pytestmark = pytest.mark.gpu


def test_replaced_weights_are_the_ones_that_are_read():
    """A layer's tensors can be written into or be other tensors: the steps read what prefill reads."""
    a, b = start(make()), start(make())
    before = a.decode_step().clone()
    b.decode_step()
    a.tok.copy_(b.tok)
    for name in ("gate", "exp_gu", "exp_d", "sh_gu", "sh_d"):
        new = a.layers[1][name].roll(1, 0) * 0.5
        a.layers[1][name].copy_(new)
        b.layers[1][name] = new
        x, y = a.decode_step(), b.decode_step()
        assert torch.equal(x, y) and not torch.equal(x, before), name
        a.tok.copy_(b.tok)
