"""Sampling: forward-mode derivatives."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ananta_ocr_b200 import sampling
from test_sampling_gpu import logits_of

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    """Forward-mode derivatives: dual tensors do not ask for gradients."""
    z, u = (t.cuda() for t in logits_of(3, 10, "fp32", 1))
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError):
            sampling.probs(fwAD.make_dual(z, z))
        with pytest.raises(NotImplementedError):
            sampling.probs(z, temperature=fwAD.make_dual(u, u))
        sampling.probs(z)
