"""Sampling of more rows than a CTA of 512 threads is taken for, whole numbers of 64 bits, forward-mode
derivatives: against the definition as in test_sampling_gpu."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ananta_ocr_b200 import sampling
from test_sampling_gpu import SETTINGS, columns, logits_of, same

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


def test_settings_that_ask_for_gradients_are_refused():
    z, u = (t.cuda() for t in logits_of(3, 10, "fp32", 1))
    s = (u + 0.5).requires_grad_()
    for name in ("temperature", "top_p", "min_p"):
        with pytest.raises(NotImplementedError):
            sampling.probs(z, **{name: s})
        with torch.no_grad():
            assert torch.equal(sampling.probs(z, **{name: s}), sampling.probs(z, **{name: s.detach()}))
        assert sampling.sample(z, u, **{name: s}).shape == (3,)      # tokens have no derivatives


def test_top_k_of_64_bits():
    """Numbers beyond 32 bits are beyond the vocabulary, or below zero: all tokens."""
    z, u = logits_of(6, 5000, "fp32", 4)
    k = [1 << 32, (1 << 32) + 3, (1 << 40) + 17, -(1 << 32) + 5, (1 << 62), 9]
    top_k = torch.tensor(k, dtype=torch.int64, device="cuda")
    same(z.cuda(), u.cuda(), [(0.9, n if 0 < n < 5000 else 0, 0.9, 0.0) for n in k], temperature=0.9, top_k=top_k, top_p=0.9)
