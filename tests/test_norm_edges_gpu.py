"""Residual norms and their gradients: forward-mode derivatives."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ananta_ocr_b200 import norms
from test_norms_gpu import make

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    """Forward-mode derivatives: dual tensors do not ask for gradients."""
    t, _, _ = make(4, 64, "fp32", 1, True)
    with fwAD.dual_level():
        norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6, gate=t["gate"], post_weight=t["post"])
        for name in t:
            d = {**t, name: fwAD.make_dual(t[name], torch.ones_like(t[name]))}
            with pytest.raises(NotImplementedError):
                norms.add_rms_norm(d["y"], d["residual"], d["weight"], 1e-6, gate=d["gate"], post_weight=d["post"])
        for y, w in ((fwAD.make_dual(t["y"], t["y"]), t["weight"]), (t["y"], fwAD.make_dual(t["weight"], t["weight"]))):
            with pytest.raises(NotImplementedError):
                norms.rms_norm(y, w, 1e-6)
        dual = fwAD.make_dual(t["y"], t["y"])
        for ds, dh in ((dual, t["y"]), (None, dual)):
            with pytest.raises(NotImplementedError):
                norms.add_rms_norm_backward(ds, dh, t["y"], t["residual"], t["weight"], 1e-6)
