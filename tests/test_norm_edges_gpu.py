"""Residual norms and their gradients: streams of any size, many rows for each CTA, forward-mode
derivatives.  Tolerances are those of test_norms_gpu."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ananta_ocr_b200 import norms
from test_norms_gpu import check_forward, check_grads, make

pytestmark = pytest.mark.gpu


def grads_of(t, ds, dh, eps, scale=1.0):
    g = norms.add_rms_norm_backward(ds, dh, t["y"], t["residual"], t["weight"], eps, gate=t["gate"], post_weight=t["post"], scale=scale)
    return dict(y=g.y, residual=g.residual, weight=g.weight, gate=g.gate, post=g.post_weight)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hidden", [136, 1280, 1283, 4104, 8192])
@pytest.mark.parametrize("power,eps", [(45, 1e-6), (52, 1e-6), (-50, 0.0)])
def test_gradients_of_streams_of_any_size(power, eps, hidden, dt):
    """Values around 2^45, 2^52 and 2^-50: 1 / rms to the third power is no 32-bit number there."""
    for groups, post in ((0, False), (1, True)):
        t, _, dh = make(5, hidden, dt, groups, post)
        t["y"].mul_(2.0 ** power), t["residual"].mul_(1.0 if post else 2.0 ** power)
        check_grads(t, None, dh, grads_of(t, None, dh, eps), eps, 1.0)
        if post:
            t["residual"].mul_(2.0 ** power)
            check_grads(t, None, dh, grads_of(t, None, dh, eps), eps, 1.0)


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


def test_many_numbers_of_rows():
    """What is kept for a number of rows is bounded, and so is a call's workspace."""
    y = torch.randn(2100, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for rows in range(1, 2100):
        norms.add_rms_norm_backward(None, y[:rows], y[:rows], None, w, 1e-6)
    assert len(norms._SIZES) <= 1024


@pytest.mark.parametrize("hidden,dt,groups,post", [(4104, "bf16", 31, True), (8192, "fp16", 1, False), (2056, "fp32", 100, True)])
def test_forward_of_many_long_rows(hidden, dt, groups, post):
    """Two vectors per thread, and four rows or more for each CTA (at most 740 of them)."""
    rows = 3100
    t, _, _ = make(rows, hidden, dt, groups, post)
    check_forward(t, *norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6, gate=t["gate"], post_weight=t["post"],
                                         scale=0.5), 1e-6, 0.5)


@pytest.mark.parametrize("rows,hidden,dt,groups,post", [
    (24000, 136, "bf16", 1, True),               # 21 rows for each of 1,143 CTAs
    (36000, 136, "fp16", 3600, True),            # chunks of 10 rows, three or four for each CTA
    (24000, 136, "bf16", 0, False),
    (9000, 520, "fp32", 450, True),              # one vector per thread, several warps, chunks of 20 rows
    (3000, 4104, "bf16", 300, True),             # two vectors per thread, chunks of 10 rows, two or three for each CTA
    (3000, 4104, "fp16", 1, True),               # 21 rows for each CTA
    (3000, 4104, "bf16", 0, False),
    (600, 8192, "fp32", 200, True),              # four vectors per thread, chunks of 3 rows
    (9000, 131, "bf16", 900, True),              # rows that are not aligned
])
def test_gradients_of_many_rows_per_cta(rows, hidden, dt, groups, post):
    t, ds, dh = make(rows, hidden, dt, groups, post)
    check_grads(t, ds, dh, grads_of(t, ds, dh, 1e-6, 0.5), 1e-6, 0.5)
