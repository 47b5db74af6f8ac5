"""The few-token mixture-of-experts layer where calls follow one another, in odd layouts and
with tensors that are trained."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ananta_ocr_b200 import moe
from step_testutil import moe as definition
from test_moe_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,topk", [(1, 32, 4), (9, 32, 4), (70, 12, 3)])
def test_picks_of_an_earlier_call_are_not_used(tokens, experts, topk):
    """Replays in a row on one workspace, each with other picks: every kernel has to wait for those of
    its own call."""
    n = 24
    t, w = make(tokens, 128, 64, experts, 32)
    xs = torch.stack([make(tokens, 128, 64, experts, 32, seed=s)[0]["x"] for s in range(n)])
    want = [moe.moe_layer(x, w, topk, residual=t["residual"]) for x in xs]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = moe.moe_layer(t["x"], w, topk, residual=t["residual"])
    outs, ids = torch.empty_like(xs), torch.empty(n, tokens, topk, dtype=torch.int32, device="cuda")
    for _ in range(3):
        for i in range(n):
            t["x"].copy_(xs[i])
            g.replay()
            outs[i].copy_(r.out)
            ids[i].copy_(r.ids)
        for i in range(n):
            assert torch.equal(outs[i], want[i].out) and torch.equal(ids[i], want[i].ids)
    assert not torch.equal(ids[0], ids[1])


@pytest.mark.parametrize("which", range(5))
def test_weights_that_are_trained_are_refused(which):
    """The flag can be set after the handle was made, and taken back."""
    t, w = make(4, 64, 32, 6, 8)
    want = moe.moe_layer(t["x"], w, 2).out
    w.tensors[which].requires_grad_()
    with pytest.raises(NotImplementedError):
        moe.moe_layer(t["x"], w, 2)
    with torch.no_grad():
        assert torch.equal(moe.moe_layer(t["x"], w, 2).out, want)
    w.tensors[which].requires_grad_(False)
    assert torch.equal(moe.moe_layer(t["x"], w, 2).out, want)


@pytest.mark.parametrize("at", [0, 3, 8])
def test_one_row_of_a_wider_tensor(at):
    """torch leaves the stride of a dimension of one as it is, also in copies."""
    t, w = make(1, 64, 32, 6, 8)
    want = moe.moe_layer(t["x"], w, 2, residual=t["residual"])
    x, res = (torch.zeros(1, 83, dtype=torch.bfloat16, device="cuda")[:, at:at + 64] for _ in range(2))
    x.copy_(t["x"]), res.copy_(t["residual"])
    assert x.stride(0) == 83
    for a, b in ((x, t["residual"]), (t["x"], res), (x, res)):
        got = moe.moe_layer(a, w, 2, residual=b)
        assert torch.equal(got.out, want.out) and torch.equal(got.ids, want.ids)


def test_tangents_are_refused():
    """Forward-mode derivatives: dual tensors do not ask for gradients."""
    t, w = make(4, 64, 32, 6, 8)
    one = torch.ones_like(t["x"])
    with fwAD.dual_level():
        want = moe.moe_layer(t["x"], w, 2, residual=t["residual"]).out
        for x, res in ((fwAD.make_dual(t["x"], one), t["residual"]), (t["x"], fwAD.make_dual(t["residual"], one))):
            with pytest.raises(NotImplementedError):
                moe.moe_layer(x, w, 2, residual=res)
        dual = moe.MoeWeights(fwAD.make_dual(t["gate"], torch.ones_like(t["gate"])), t["gu"], t["down"])
        with pytest.raises(NotImplementedError):
            moe.moe_layer(t["x"], dual, 2)
    assert torch.equal(moe.moe_layer(t["x"], w, 2, residual=t["residual"]).out, want)


@pytest.mark.parametrize("gate", ["same", "fp32"])
@pytest.mark.parametrize("factor,other", [(2.0 ** 70, 0.0), (2.0 ** 70, -0.5), (2.0 ** -80, 0.0)])
def test_scores_of_products_beyond_32_bits(factor, other, gate):
    """2^140 and 2^-160 are numbers of a 64-bit score, and 2^140 - 2^139 is 2^139."""
    t, w = make(3, 64, 32, 6, gate=gate)
    t["gate"].zero_()
    t["gu"][:, :, :2] = 0                         # (of the router alone)
    t["x"][:, 0], t["x"][:, 1] = factor, other * factor
    for e in range(6):
        t["gate"][e, :2] = factor * (e + 1)
    r = moe.moe_layer(t["x"], w, 3, residual=t["residual"])
    assert r.ids.tolist() == [[5, 4, 3]] * 3
    check(t, r, 3)


@pytest.mark.parametrize("tokens", [2, 20])
def test_small_inner_values(tokens):
    """fp16: inner values around 2^-21, where that type has multiples of 2^-24.  Their second number
    holds what the first one leaves to 2^-36 (half a step of 2^-24, kept 2^11 times as large)."""
    t, w = make(tokens, 64, 136, 6, 40, "fp16")
    t["gu"].mul_(2.0 ** -10), t["sgu"].mul_(2.0 ** -10)
    t["down"].mul_(8.0), t["sd"].mul_(8.0)
    r = moe.moe_layer(t["x"], w, 4)
    up = {k: v.double().cpu() for k, v in t.items()}
    out, ids, _, tol = definition(up["x"], up["gate"], up["gu"], up["down"], up["sgu"], up["sd"], 4, False, 1.0, None,
                                  torch.float16, least=2.0 ** -36)
    assert torch.equal(r.ids.cpu(), ids)
    off = (r.out.double().cpu() - out).abs()
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [(256, 64, 104, 64, 16, 0), (16, 64, 248, 64, 16, 72), (256, 64, 152, 64, 16, 72), (16, 64, 296, 64, 16, 72),
                                  (256, 64, 176, 64, 16, 72), (16, 64, 344, 64, 16, 0)])
def test_heights_of_tiles(case, dt):
    """gate_up's tiles of 40, 48, 56, 56, 64 and 64 rows, none of which divides the width."""
    tokens, hidden, ffn, experts, topk, shared = case
    t, w = make(tokens, hidden, ffn, experts, shared, dt)
    check(t, moe.moe_layer(t["x"], w, topk, residual=t["residual"]), topk)


def test_weights_of_other_memory():
    """A tensor's .data can be other memory (a module's `to`): it is read, or refused where it does not fit."""
    t, w = make(4, 64, 32, 6, 8)
    moe.moe_layer(t["x"], w, 2)
    n, nw = make(4, 64, 32, 6, 8, seed=1)
    want = moe.moe_layer(t["x"], nw, 2)
    old = [v.data for v in w.tensors]
    for a, b in zip(w.tensors, nw.tensors):
        a.data = b.data.clone()
    assert torch.equal(moe.moe_layer(t["x"], w, 2).out, want.out)
    for a in w.tensors:
        a.data = a.data.half()
    with pytest.raises(ValueError):
        moe.moe_layer(t["x"], w, 2)
    half = dict(zip(("gate", "gu", "down", "sgu", "sd"), w.tensors), x=t["x"].half(), residual=None)
    check(half, moe.moe_layer(half["x"], w, 2), 2, residual=False)
    for a, b in zip(w.tensors, old):
        a.data = b
    w.tensors[2].data = old[2][:, :56].contiguous()
    for _ in range(2):
        with pytest.raises(ValueError):
            moe.moe_layer(t["x"], w, 2)
    w.tensors[2].data = old[2].cpu()
    with pytest.raises(RuntimeError):
        moe.moe_layer(t["x"], w, 2)
    w.tensors[2].data = old[2]
    check(t, moe.moe_layer(t["x"], w, 2, residual=t["residual"]), 2)


@pytest.mark.parametrize("tokens", [2, 20])
def test_wide_shared_experts(tokens):
    """More weights than are fetched ahead."""
    t, w = make(tokens, 4096, 64, 3, 1032)
    check(t, moe.moe_layer(t["x"], w, 2, residual=t["residual"]), 2)


@pytest.mark.parametrize("tokens", [1, 8, 64])
def test_calls_repeat_themselves(tokens):
    """Whatever the workspace held before: bit for bit."""
    t, w = make(tokens, 1280, 896, 64, 1792)
    want = moe.moe_layer(t["x"], w, 6, residual=t["residual"])
    size = w.workspace_bytes(tokens, 6)
    for byte in (0xff, 0x7f, 0x00, 0x5a) * 3:
        torch.full((size,), byte, dtype=torch.uint8, device="cuda")          # (freed at once, and the next to be handed out)
        r = moe.moe_layer(t["x"], w, 6, residual=t["residual"])
        for a, b in zip(r, want):
            assert torch.equal(a, b)
