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


@pytest.mark.parametrize("rows,vocab,dt", [(65, 5000, "bf16"), (130, 5000, "fp32"), (70, 60000, "bf16"), (66, 60000, "fp32"),
                                           (100, 60001, "fp16"), (66, 129280, "bf16"), (66, 129280, "fp32")])
def test_many_rows(rows, vocab, dt):
    """256 threads, one to eight CTAs for a row, slices in shared memory or not."""
    settings = [SETTINGS[i % len(SETTINGS)] for i in range(rows)]
    z, u = logits_of(rows, vocab, dt, vocab, spread=2.0)
    same(z.cuda(), u.cuda(), settings, **columns(settings))


@pytest.mark.parametrize("rows", [40, 64])
def test_four_ctas_of_512_threads(rows):
    """16-bit rows of which four CTAs hold one."""
    settings = [SETTINGS[i % len(SETTINGS)] for i in range(rows)]
    z, u = logits_of(rows, 129280, "bf16", rows, spread=2.0)
    same(z.cuda(), u.cuda(), settings, **columns(settings))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_ties_across_slices_of_many_rows(dt):
    g = torch.Generator().manual_seed(3)
    z = torch.randint(0, 4, (72, 40000), generator=g).to(torch.float32 if dt == "fp32" else torch.bfloat16)
    u = torch.rand(72, generator=g)
    settings = [(1.0, 11000, 1.0, 0.0), (1.0, 0, 0.55, 0.0), (1.0, 30001, 0.77, 0.0), (0.5, 1, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 2, 0.6, 0.0)] * 12
    same(z.cuda(), u.cuda(), settings, **columns(settings))


@pytest.mark.parametrize("setting", [(0.8, 30, 0.9, 0.01), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 3000, 1.0, 0.0), (1.0, 0, 0.9, 0.0)])
def test_masks_and_odd_values_of_many_rows(setting):
    """Rows with nothing, one token, masks of -inf or of the type's lowest value, NaN, an infinite logit."""
    V, inf = 20000, float("inf")
    for dt in (torch.float32, torch.bfloat16):
        z, u = logits_of(70, V, "fp32", 5)
        z = z.to(dt)
        z[0] = -inf
        z[1] = -inf
        z[1, 14321] = -7.0
        z[2, 100:] = torch.finfo(dt).min
        z[3, ::3] = float("nan")
        z[4] = float("nan")
        z[5, :19990] = -inf
        z[6, 17] = inf
        z[7, 9000:] = -inf
        t, k, p, m = setting
        same(z.cuda(), u.cuda(), [setting] * 70, temperature=t, top_k=k, top_p=p, min_p=m)
