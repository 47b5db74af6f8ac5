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


@pytest.mark.parametrize("batch", [1, 2, 5])
def test_draft_steps_are_those_of_the_plain_forms(batch, monkeypatch):
    """As the decode steps' test, with the same roots on both sides: always compared."""
    a, b = start(make(batch)), start(make(batch))
    extra = torch.randint(0, 1000, (batch, 4), generator=torch.Generator().manual_seed(5)).cuda()
    a.decode_step()
    root = a.tok.clone()
    got = a.draft_step(extra)[1].float()
    monkeypatch.setattr(norms, "rms_norm", plain_norm)
    monkeypatch.setattr(norms, "add_rms_norm", plain_add)
    monkeypatch.setattr(moe, "moe_layer", plain_moe)
    b.decode_step()
    b.tok.copy_(root)
    want = b.draft_step(extra)[1].float()
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 0.02 * want.abs().max()
